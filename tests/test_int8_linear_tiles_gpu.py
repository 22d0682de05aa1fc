"""int8_linear at sizes that take each of its kernels, odd in every dimension, against the product in doubles on the GPU.

What takes which kernel (256 units): 4 tokens and fewer dot products; up to 64 pieces of rows; beyond that tiles of 256 x 256, 256 x 128,
128 x 128, 64 x 128, 64 x 64 and pieces again by the rounds that they need; rows that do not begin on words registers."""
import pytest
import torch

from block_reference import U32, half_step, smallest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def on_gpu(shape, low, high, g):
    return torch.randint(low, high, shape, generator=g, device="cuda").to(torch.int8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("tokens,k,n", [
    (3, 8200, 8200), (4, 4104, 9001), (2, 33000, 1100),       # dot products: one and four channels a wavefront, streamed weights
    (15, 5128, 7170), (16, 1032, 500), (29, 4100, 8190), (32, 900, 300), (61, 5124, 7169), (64, 700, 1001),   # pieces, one block of channels and two
    (4001, 1028, 4090), (2500, 644, 6107),                     # 256 x 256
    (2000, 644, 3970), (1030, 520, 4090), (4090, 260, 1030),   # 256 x 128
    (1000, 516, 9000), (2050, 1028, 4100), (260, 1156, 7165),  # 128 x 128
    (1257, 1004, 1100), (129, 1284, 7000),                     # 64 x 128
    (701, 700, 700), (66, 516, 2000), (100, 2052, 1290),       # 64 x 64, pieces
    (5, 1013, 900), (31, 1025, 257), (33, 515, 300), (300, 259, 1025), (1500, 131, 2100), (2000, 517, 1411),   # rows that do not begin on words, tiles of 64 and 128
])
def test_every_tile(tde, tokens, k, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens + k + n)
    codes, weight = on_gpu((tokens, k), -127, 128, g), on_gpu((n, k), -128, 128, g)
    scales = torch.rand(tokens, generator=g, device="cuda") * 0.02 + 0.001
    weight_scales = torch.rand(n, generator=g, device="cuda") * 0.002 + 0.0001
    bias = torch.randn(n, generator=g, device="cuda") if n % 2 else None
    got = tde.int8_linear(codes, scales, weight, weight_scales, bias, dtype).double()
    y = torch.mm(codes.double(), weight.double().t().contiguous()) * scales.double()[:, None] * weight_scales.double()
    want = y if bias is None else y + bias.double()
    bound = y.abs() * 3.01 * U32 + want.abs() * (U32 + half_step(dtype)) * 1.01 + smallest(dtype)   # as in block_reference.int8_linear
    wrong = (got - want).abs() > bound
    assert not bool(wrong.any()), (int(wrong.sum()), wrong.nonzero()[0].tolist())
    # the same call again: integers add up to the same bits in every order
    assert torch.equal(got, tde.int8_linear(codes, scales, weight, weight_scales, bias, dtype).double())
