"""Values that are not finite in keys that rows do see: infinities arrive with their sign, both signs and NaN as NaN, in their channels alone."""
import pytest
import torch

from block_reference import Batch, assert_close, attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("new,lens,heads,kv_heads", [
    ([1, 1, 1], [700, 40, 3000], 4, 2),         # decode rows, split
    ([1] * 160, [70] * 160, 8, 8),              # whole
    ([2, 3], [90, 5], 4, 1),                    # a few rows each
    ([40, 7, 150], [90, 50, 333], 6, 2),        # chunks
], ids=["split", "whole", "few", "chunks"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_seen_values(tde, new, lens, heads, kv_heads, dim, dtype):
    batch = Batch(new, lens, page_size=16, seed=1, pad=2)
    q = randn((batch.tokens, heads, dim), dtype, 2)
    k, v = (randn((batch.pages, 16, kv_heads, dim), dtype, 3 + i) for i in (0, 1))
    inf, nan = float("inf"), float("nan")
    for b, n in enumerate(lens):
        first = n - new[b]        # keys that all rows see, in the first tiles and next to the call's own rows
        for at, channel, bad in ((0, 0, inf), (first, 1, -inf), (first // 2, 2, inf), (first // 3, 2, -inf), (first // 2, 3, nan), (first // 4, dim - 1, inf),
                                 (first // 2, dim - 1, inf)):
            v[batch.page_of(b, at), at % 16, :, channel] = bad
    got = tde.paged_attention(q.cuda(), k.cuda(), v.cuda(), *batch.on("cuda"))
    want, bound = attention(batch, q, k, v, dim ** -0.5)
    assert torch.isinf(want[..., :2]).any() and torch.isnan(want[..., 3]).any()
    assert_close(got, want, bound.nan_to_num(0.0))
