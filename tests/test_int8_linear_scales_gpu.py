"""int8_linear with scales that are not finite: every element of their rows and channels, by value and sign."""
import math

import pytest
import torch

from block_reference import assert_close, int8_linear

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("tokens,k,n", [(1, 64, 40), (3, 2000, 9000), (20, 300, 64), (60, 1032, 7169), (130, 512, 140), (300, 1028, 770), (19, 301, 64), (150, 301, 90)])
def test_rows_and_channels(tde, tokens, k, n, biased, dtype):
    """Each of the kernels: rows of whole words for one token to many, and rows that begin anywhere."""
    g = torch.Generator().manual_seed(tokens + k + n)
    codes, weight = (torch.randint(-127, 128, shape, generator=g).to(torch.int8) for shape in ((tokens, k), (n, k)))
    scales, ws = torch.rand(tokens, generator=g) * 0.02 + 0.001, torch.rand(n, generator=g) * 0.002 + 0.0001
    bias = torch.randn(n, generator=g) if biased else None
    if tokens > 1:
        codes[0] = 0                        # a row whose sums are all 0
    weight[n // 2 - 1] = 0                  # and a channel
    want, bound = int8_linear(codes, scales, weight, ws, bias, dtype)
    total = codes.double() @ weight.double().t()
    bad_row, bad = tokens // 2 + 1, {n // 2: math.inf, n // 2 - 1: math.inf, 3: -math.inf, n - 1: math.nan}
    for channel, scale in bad.items():
        ws[channel] = scale
        # a sum times an infinite scale: infinite with the product's sign, NaN where the sum is 0
        want[:, channel] = torch.where(total[:, channel] == 0, math.nan, total[:, channel] * scale)
    if tokens > 2:
        scales[bad_row] = -math.inf
        want[bad_row] = torch.where(total[bad_row] == 0, math.nan, -total[bad_row] * ws.double().sign() * math.inf)
        scales[tokens - 1] = math.nan
        want[tokens - 1] = math.nan
    got = tde.int8_linear(*[None if x is None else x.cuda() for x in (codes, scales, weight, ws, bias)], dtype)
    assert_close(got, want, bound.nan_to_num(0.0))
