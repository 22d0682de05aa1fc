"""q_starts that begin above 0, as a slice of a larger batch's has them: rows in front of the first sequence belong to none, like those
behind the last one."""
import pytest
import torch

from block_reference import Batch, append, assert_close, attention, norm_rope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def shifted(batch, front):
    """The same sequences behind `front` rows: the index arrays and the number of rows."""
    table, starts, lens = batch.on("cuda")
    return (table, starts + front, lens), batch.tokens + front


def remembered(rows, shape, dtype):
    """Leaves a freed block of that size full of sevens, which an output that nobody writes would show."""
    x = torch.full((rows,) + shape, 7.0, dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    del x


BATCHES = [
    ([1, 1, 1], [3, 700, 64]),             # decode rows, split
    ([1] * 300, [20] * 300),               # decode rows, whole
    ([40, 0, 7], [90, 5, 7]),              # chunks
    ([0, 0, 2], [4, 0, 2]),                # empty sequences first
    ([0], [9]),                            # no sequence has a row
]


@pytest.mark.parametrize("new,lens", BATCHES)
@pytest.mark.parametrize("front", [1, 5, 70])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 2, 64, torch.bfloat16), (8, 1, 128, torch.float16), (2, 2, 256, torch.bfloat16)])
def test_attention(tde, new, lens, front, heads, kv_heads, dim, dtype):
    batch = Batch(new, lens, page_size=16, pad=3, seed=1)
    args, tokens = shifted(batch, front)
    q = randn((tokens, heads, dim), dtype, 2)
    k, v = (randn((batch.pages, 16, kv_heads, dim), dtype, 3 + i) for i in (0, 1))
    want, bound = attention(batch, q[front:], k, v, dim ** -0.5)
    k, v, q_dev = k.cuda(), v.cuda(), q.cuda()
    remembered(tokens, (heads, dim), dtype)
    got = tde.paged_attention(q_dev, k, v, *args)
    assert_close(got[front:], want, bound)
    assert not got[:front].any()
    out = torch.full_like(q_dev, 5.0)
    tde.paged_attention_out(q_dev, k, v, *args, out)
    end = int(batch.starts[-1])
    assert_close(out[front:front + end], want[:end], bound[:end])
    assert bool((out[:front] == 5).all()) and bool((out[front + end:] == 5).all())


def test_attention_of_a_large_chunk(tde):
    """Rows enough for tiles of 128; the rows of no sequence are more than one tile."""
    new, front = [1400], 300
    batch = Batch(new, new, page_size=16, pad=130, seed=5)
    args, tokens = shifted(batch, front)
    q, k, v = (torch.randn(s, dtype=torch.bfloat16, device="cuda") for s in ((tokens, 64, 64), (batch.pages, 16, 8, 64), (batch.pages, 16, 8, 64)))
    alone = tde.paged_attention(q[front:].contiguous(), k, v, *batch.on("cuda"))
    remembered(tokens, (64, 64), torch.bfloat16)
    got = tde.paged_attention(q, k, v, *args)
    assert torch.equal(got[front:], alone) and not got[:front].any() and not got[-130:].any()
    out = torch.full_like(q, 5.0)
    tde.paged_attention_out(q, k, v, *args, out)
    assert torch.equal(out[front:-130], alone[:-130]) and bool((out[:front] == 5).all()) and bool((out[-130:] == 5).all())


def test_attention_without_sequences(tde):
    """One entry in q_starts, in the middle of the rows."""
    q = torch.ones((9, 4, 64), dtype=torch.bfloat16, device="cuda")
    k = torch.ones((3, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros((0, 4), dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    for at in (0, 4, 9):
        remembered(9, (4, 64), torch.bfloat16)
        assert not tde.paged_attention(q, k, k, table, torch.tensor([at], dtype=torch.int32, device="cuda"), lens).any()


@pytest.mark.parametrize("dim,rot,heads", [(64, 64, 4), (20, 12, 3)])
@pytest.mark.parametrize("front", [1, 70])
def test_append(tde, dim, rot, heads, front):
    dtype = torch.bfloat16
    batch = Batch([3, 0, 40], [10, 7, 41], page_size=16, pad=2, seed=6)
    args, tokens = shifted(batch, front)
    qkv = randn((tokens, heads + 4, dim), dtype, 7)
    q, k, v = qkv.split([heads, 2, 2], dim=1)
    a = torch.rand((50, rot // 2), generator=torch.Generator().manual_seed(8), dtype=torch.float64) * 6.3
    cs, gamma = torch.cat([a.cos(), a.sin()], dim=1).float(), randn((dim,), dtype, 9)
    k_cache, v_cache = (randn((batch.pages, 16, 2, dim), dtype, 10 + i) for i in (0, 1))
    dev, k_dev, v_dev = qkv.cuda(), k_cache.cuda(), v_cache.cuda()
    got = tde.append_kv(dev[:, heads:heads + 2], dev[:, heads + 2:], k_dev, v_dev, *args, cos_sin=cs.cuda(), q=dev[:, :heads], q_gamma=gamma.cuda(),
                        k_gamma=gamma.cuda(), eps=1e-6)
    positions = torch.full((batch.tokens,), -1)
    for t, _, p in batch.rows():
        positions[t] = p
    rows = cs[positions.clamp(min=0)]
    k_want, k_bound = norm_rope(k[front:], gamma, 1e-6, rows, False, dtype)
    keys, values, written, token_of = append(batch, k_want, v[front:], k_cache, v_cache)
    bound = torch.zeros_like(keys)
    bound[written] = k_bound[token_of[written]]
    assert_close(k_dev, keys, bound)
    assert torch.equal(v_dev.cpu(), values)
    want, bound = norm_rope(q[front:], gamma, 1e-6, rows, False, dtype)
    want[positions < 0], bound[positions < 0] = 0.0, 0.0
    assert_close(got[front:], want, bound)
    assert not got[:front].any()
