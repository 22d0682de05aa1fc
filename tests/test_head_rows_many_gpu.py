"""qk_norm_rope and append_kv with tokens enough for wavefronts that take 2, 3 and 5 rows of a token, streamed past the caches."""
import pytest
import torch

from block_reference import Batch, append, assert_close, norm_rope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def table(positions, rot):
    a = torch.rand((positions, rot // 2), generator=torch.Generator().manual_seed(rot), dtype=torch.float64) * 6.3
    return torch.cat([a.cos(), a.sin()], dim=1).float()


# rows a wavefront with and without values: 3 and 5, 2 and 2, 5 and 5, 2 and 2
SHAPES = [(4100, 20, 4, 128, 128), (5000, 3, 1, 64, 32), (2100, 24, 8, 256, 256), (4200, 5, 1, 96, 48)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot", SHAPES)
def test_norm_rope(tde, tokens, heads, kv_heads, dim, rot, interleaved, dtype):
    qkv = randn((tokens, heads + kv_heads, dim), dtype, dim)
    qg, kg, cs = randn((dim,), dtype, 1), randn((dim,), dtype, 2), table(90, rot)
    pos = torch.arange(tokens) * 7 % 90
    dev = qkv.cuda()
    q, k = tde.qk_norm_rope(dev[:, :heads], dev[:, heads:], qg.cuda(), kg.cuda(), 1e-6, pos.cuda(), cs.cuda(), interleaved)
    assert_close(q, *norm_rope(qkv[:, :heads], qg, 1e-6, cs[pos], interleaved, dtype), "q")
    assert_close(k, *norm_rope(qkv[:, heads:], kg, 1e-6, cs[pos], interleaved, dtype), "k")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("norm,rotate,interleaved", [(True, True, False), (False, True, True), ("keys", False, False), (False, False, False)])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot", SHAPES)
def test_append(tde, tokens, heads, kv_heads, dim, rot, norm, rotate, interleaved, dtype):
    # a sequence shorter than its rows, one with a page that does not exist, rows behind the last one
    new = [tokens - 1500, 30, 0, 900, 500]
    batch = Batch(new, [tokens, 11, 4, 900, 1700], page_size=24, pad=70, seed=dim)
    batch.table[4, 60] = batch.pages
    qkv = randn((batch.tokens, heads + 2 * kv_heads, dim), dtype, dim + 1)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    qg = randn((dim,), dtype, 3) if norm is True else None
    kg = randn((dim,), dtype, 4) if norm else None
    cs = table(tokens + 1, rot) if rotate else None
    k_cache, v_cache = (randn((batch.pages, 24, kv_heads, dim), dtype, i) for i in (5, 6))
    dev, gpu = qkv.cuda(), lambda x: None if x is None else x.cuda()
    k_dev, v_dev = k_cache.cuda(), v_cache.cuda()
    got = tde.append_kv(dev[:, heads:heads + kv_heads], dev[:, heads + kv_heads:], k_dev, v_dev, *batch.on("cuda"), cos_sin=gpu(cs), q=dev[:, :heads],
                        q_gamma=gpu(qg), k_gamma=gpu(kg), eps=1e-6, interleaved=interleaved)
    positions = torch.full((batch.tokens,), -1)
    for t, _, p in batch.rows():
        positions[t] = p
    rows = cs[positions.clamp(min=0)] if rotate else None
    k_want, k_bound = norm_rope(k, kg, 1e-6, rows, interleaved, dtype)
    keys, values, written, token_of = append(batch, k_want, v, k_cache, v_cache)
    bound = torch.zeros_like(keys)
    bound[written] = k_bound[token_of[written]]
    assert_close(k_dev, keys, bound, "keys")
    assert torch.equal(v_dev.cpu(), values)
    want, bound = norm_rope(q, qg, 1e-6, rows, interleaved, dtype)
    want[positions < 0], bound[positions < 0] = 0.0, 0.0
    assert_close(got, want, bound, "queries")
