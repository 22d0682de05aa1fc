"""paged_attention where a call has rows enough for its largest tiles (128 rows: with 256 units from about 98 thousand rows of queries on,
a third of that with heads of more than 128 channels)."""
import pytest
import torch

from block_reference import Batch, assert_close, attention, attention_at_once

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def inputs(batch, heads, kv_heads, dim, dtype, seed):
    q = randn((batch.tokens, heads, dim), dtype, seed)
    return (q,) + tuple(randn((batch.pages, batch.page, kv_heads, dim), dtype, seed + i) for i in (1, 2))


# 64 heads that share 8: 1700 tokens are 109 thousand rows
CHUNKS = [([1700], [1700]), ([1000, 0, 1, 640, 130], [1000, 50, 900, 1337, 129]), ([40] * 44, [40 + 17 * i for i in range(44)])]


@pytest.mark.parametrize("new,lens", CHUNKS, ids=["one", "ragged", "many"])
@pytest.mark.parametrize("dim,page,dtype", [(128, 16, torch.bfloat16), (64, 24, torch.float16), (96, 7, torch.bfloat16), (40, 128, torch.float16), (256, 16, torch.bfloat16)],
                         ids=str)
def test_chunks(tde, new, lens, dim, page, dtype):
    batch = Batch(new, lens, page_size=page, seed=1, pad=5)
    q, k, v = inputs(batch, 64, 8, dim, dtype, dim)
    got = tde.paged_attention(q, k, v, *batch.on("cuda"))
    assert_close(got, *attention_at_once(batch, q, k, v, dim ** -0.5))
    assert torch.equal(got, tde.paged_attention(q, k, v, *batch.on("cuda")))


def test_the_two_references_agree(tde):
    batch = Batch([30, 0, 5], [40, 7, 3], page_size=8, seed=2, pad=3)
    batch.table[0, 4] = -1
    q, k, v = (x.cpu() for x in inputs(batch, 4, 2, 16, torch.float16, 3))
    v[batch.page_of(0, 20), 20 % 8, :, 2] = float("inf")
    (want, bound), (at_once, at_once_bound) = attention(batch, q, k, v, 0.25), attention_at_once(batch, q, k, v, 0.25)
    assert_close(at_once, want, want.nan_to_num(0.0, 0.0, 0.0).abs() * 1e-9 + 1e-12)
    shown = torch.isfinite(want)      # the others are compared for being the same, without a bound
    assert_close(at_once_bound[shown], bound[shown], bound[shown] * 1e-9)


@pytest.mark.parametrize("dim", [64, 128])
def test_hidden_values_and_lost_pages(tde, dim):
    batch = Batch([900, 800, 3], [950, 1100, 2], page_size=24, seed=4, pad=2)
    q, k, v = inputs(batch, 64, 8, dim, torch.bfloat16, 5)
    used = torch.zeros((batch.pages, 24), dtype=torch.bool)
    for b, n in enumerate(batch.lens):
        for j in range(n):
            used[batch.page_of(b, j), j % 24] = True
    k[~used.cuda()], v[~used.cuda()] = float("nan"), float("inf")
    for b, row, channel, bad in ((0, 899, 0, "nan"), (0, 500, 1, "inf"), (0, 400, 2, "-inf"), (0, 300, 1, "-inf"), (1, 799, dim - 1, "inf"), (1, 64, 7, "nan")):
        p = batch.lens[b] - batch.new[b] + row
        v[batch.page_of(b, p), p % 24, :, channel] = float(bad)
    batch.table[1, 30] = batch.pages      # keys 720 to 743: rows from position 720 on
    got = tde.paged_attention(q, k, v, *batch.on("cuda"))
    assert_close(got, *attention_at_once(batch, q, k, v, dim ** -0.5))


def test_strides_and_an_output_between_others(tde):
    batch = Batch([1700, 60], [1700, 100], page_size=16, seed=6, pad=4)
    both = randn((batch.pages, 2, batch.page, 8, 136), torch.bfloat16, 7)
    k, v = both[:, 0, ..., :128], both[:, 1, ..., 8:]
    q = randn((64, batch.tokens, 129), torch.bfloat16, 8).transpose(0, 1)[..., 1:]
    out = torch.full((batch.tokens, 65, 129), 7.0, dtype=torch.bfloat16, device="cuda")
    tde.paged_attention_out(q, k, v, *batch.on("cuda"), out[:, 1:, :128])
    want, bound = attention_at_once(batch, q, k, v, 128 ** -0.5)
    end = int(batch.starts[-1])
    assert_close(out[:end, 1:, :128], want[:end], bound[:end])
    assert bool((out[end:] == 7).all()) and bool((out[:, 0] == 7).all()) and bool((out[..., 128] == 7).all())


@pytest.mark.parametrize("new,lens", [([1, 1], [100, 16]), ([40, 3], [90, 7])])
def test_slots_far_apart(tde, new, lens):
    """Caches ordered by slot, where eight rows of a load lie 4.7 GB apart."""
    pages, dim = 5_200_000, 64
    k, v = (torch.zeros((8, pages, 1, dim), dtype=torch.bfloat16, device="cuda").transpose(0, 1) for _ in (0, 1))
    assert k.stride(1) * 2 * 7 > 2 ** 32
    batch = Batch(new, lens, page_size=8, seed=9)
    q, ks, vs = inputs(batch, 4, 1, dim, torch.bfloat16, 10)
    k[-batch.pages:], v[-batch.pages:] = ks, vs
    table, starts, lens_ = batch.on("cuda")
    table = torch.where(table >= 0, table + (pages - batch.pages), table)
    got = tde.paged_attention(q, k, v, table, starts, lens_)
    assert_close(got, *attention(batch, q.cpu(), ks.cpu(), vs.cpu(), dim ** -0.5))
    added = randn((batch.tokens, 1, dim), torch.bfloat16, 11)
    tde.append_kv(added, added, k, v, table, starts, lens_)
    for t, b, p in batch.rows():
        assert torch.equal(k[pages - batch.pages + batch.page_of(b, p), p % 8], added[t])
        assert torch.equal(v[pages - batch.pages + batch.page_of(b, p), p % 8], added[t])
