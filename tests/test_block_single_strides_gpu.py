"""Dimensions of one element, whose strides separate nothing and may be anything: one page, one slot, one head, one row, one sequence."""
import pytest
import torch

from block_reference import Batch

pytestmark = pytest.mark.gpu
ODD = [0, 1, 12345, (1 << 31) + 1, 1 << 42]


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def with_stride(t, d, stride):
    strides = list(t.stride())
    strides[d] = stride
    return t.as_strided(t.shape, strides)


@pytest.mark.parametrize("stride", ODD)
@pytest.mark.parametrize("page,kv_heads", [(64, 2), (1, 2), (16, 1)])
def test_any_stride(tde, stride, page, kv_heads):
    length = 40 if page > 1 else 1
    batch = Batch([1], [length], page_size=page, seed=1, extra_pages=0)
    args = batch.on("cuda")
    g = torch.Generator(device="cuda").manual_seed(page)
    k_cache, v_cache = (torch.randn((batch.pages, page, kv_heads, 64), generator=g, device="cuda").to(torch.bfloat16) for _ in (0, 1))
    rows = torch.randn((1, 8, 64), generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = rows.split([8 - 2 * kv_heads, kv_heads, kv_heads], dim=1)
    want_caches = k_cache.clone(), v_cache.clone()
    tde.append_kv(k, v, *want_caches, *args)
    want = tde.paged_attention(q, *want_caches, *args)
    odd = [k_cache, v_cache]
    for d in range(3):
        if k_cache.size(d) == 1:
            odd = [with_stride(x, d, stride) for x in odd]
    table, starts, lens = args
    table = with_stride(table, 0, stride)
    rows = [with_stride(x, 0, stride) for x in (q, k, v)]
    if kv_heads == 1:
        rows[1:] = [with_stride(x, 1, stride) for x in rows[1:]]
    tde.append_kv(*rows[1:], *odd, table, starts, lens)
    assert torch.equal(k_cache, want_caches[0]) and torch.equal(v_cache, want_caches[1])
    assert torch.equal(tde.paged_attention(rows[0], *odd, table, starts, lens), want)
    out = torch.zeros_like(want)
    tde.paged_attention_out(rows[0], *odd, table, starts, lens, with_stride(out, 0, stride))
    assert torch.equal(out, want)
