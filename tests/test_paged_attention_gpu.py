"""paged_attention against its definition in doubles, row by row: lengths, groups, pages, what rows do not see, splits, graphs."""
import pytest
import torch

from block_reference import Batch, assert_close, attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def run(tde, batch, heads, kv_heads, dim, dtype, seed=0, scale=None, spread=1.0):
    q = randn((batch.tokens, heads, dim), dtype, seed, spread)
    k, v = (randn((batch.pages, batch.page, kv_heads, dim), dtype, seed + i) for i in (1, 2))
    got = tde.paged_attention(q.cuda(), k.cuda(), v.cuda(), *batch.on("cuda"), scale)
    want, bound = attention(batch, q, k, v, dim ** -0.5 if scale is None else scale)
    assert_close(got, want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (1, 1, 8, 1), (4, 4, 64, 16), (8, 1, 128, 64), (6, 2, 40, 3), (10, 2, 80, 24), (7, 1, 96, 16), (16, 1, 128, 128), (5, 5, 128, 8), (12, 4, 192, 16),
    (8, 2, 256, 32), (34, 2, 64, 16), (3, 1, 256, 5),
])
def test_lengths_and_shapes(tde, heads, kv_heads, dim, page, dtype):
    decode = Batch(new=[1, 1, 1, 1, 1, 1, 1], lens=[1, 2, 31, 64, 65, 300, 1000], page_size=page, seed=1)
    run(tde, decode, heads, kv_heads, dim, dtype, seed=dim)
    # chunks; sequences without rows, without keys, shorter than their rows; rows behind the last sequence
    ragged = Batch(new=[5, 0, 17, 1, 3, 2, 70, 0], lens=[5, 9, 40, 513, 2, 0, 130, 0], page_size=page, pad=9, seed=2)
    run(tde, ragged, heads, kv_heads, dim, dtype, seed=dim + 9)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (2, 2), (3, 1)])
def test_long_chunks(tde, dim, heads, kv_heads):
    run(tde, Batch(new=[333], lens=[700], page_size=16, seed=3), heads, kv_heads, dim, torch.bfloat16, seed=4)
    run(tde, Batch(new=[129, 64, 250], lens=[129, 1024, 255], page_size=24, seed=5, pad=1), heads, kv_heads, dim, torch.float16, seed=6)


@pytest.mark.parametrize("seqs", [64, 65, 129, 300])
def test_many_sequences(tde, seqs):
    g = torch.Generator().manual_seed(seqs)
    new = torch.randint(0, 3, (seqs,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 40, (seqs,), generator=g))]
    run(tde, Batch(new, lens, page_size=8, seed=7, pad=5), 4, 2, 64, torch.bfloat16, seed=8)
    run(tde, Batch([1] * seqs, [x + 1 for x in lens], page_size=8, seed=9), 4, 2, 128, torch.bfloat16, seed=10)


@pytest.mark.parametrize("heads,kv_heads,dim,lens", [(8, 1, 128, [20000]), (2, 2, 64, [9000, 3, 700]), (4, 1, 256, [6000, 100]), (16, 2, 80, [5000])])
def test_one_token_behind_many(tde, heads, kv_heads, dim, lens):
    run(tde, Batch([1] * len(lens), lens, page_size=64, seed=11), heads, kv_heads, dim, torch.bfloat16, seed=12)
    run(tde, Batch([9] * len(lens), [n + 9 for n in lens], page_size=16, seed=11, pad=2), heads, kv_heads, dim, torch.float16, seed=13)


def test_scales_and_peaked_softmax(tde):
    batch = Batch(new=[1, 20, 80], lens=[200, 300, 80], page_size=16, seed=14)
    run(tde, batch, 4, 2, 128, torch.bfloat16, seed=15, scale=2.0)              # weights concentrate on few keys
    run(tde, batch, 4, 2, 128, torch.bfloat16, seed=16, scale=1e-3)             # nearly uniform
    run(tde, batch, 4, 2, 64, torch.float16, seed=17, scale=0.125, spread=8.0)


def strided(batch, kv_heads, dim, dtype, kind):
    if kind == "heads first":
        k = randn((batch.pages, kv_heads, batch.page, dim), dtype, 1).cuda().transpose(1, 2)
        v = randn((kv_heads, batch.pages, batch.page, dim), dtype, 2).cuda().permute(1, 2, 0, 3)
    else:
        both = randn((batch.pages, 2, batch.page, kv_heads, dim + 8), dtype, 3).cuda()
        k, v = both[:, 0, ..., :dim], both[:, 1, ..., :dim]
    return k, v


@pytest.mark.parametrize("kind", ["heads first", "together"])
def test_strides(tde, kind):
    for dim in (128, 72):
        batch = Batch(new=[3, 1, 90], lens=[100, 77, 95], page_size=16, seed=18)
        k, v = strided(batch, 2, dim, torch.bfloat16, kind)
        q = randn((4, batch.tokens, dim + 3), torch.bfloat16, 4).cuda().transpose(0, 1)[..., 1:1 + dim]   # rows that begin anywhere
        table, starts, lens = batch.on("cuda")
        wide = torch.zeros((table.size(0), table.size(1) + 3), dtype=torch.int32, device="cuda")
        wide[:, :-3] = table
        want, bound = attention(batch, q.cpu(), k.cpu(), v.cpu(), dim ** -0.5)
        assert_close(tde.paged_attention(q, k, v, wide[:, :-3], starts, lens), want, bound)
        out = torch.full((batch.tokens, 5, dim + 1), 7.0, dtype=torch.bfloat16, device="cuda")
        tde.paged_attention_out(q, k, v, table, starts, lens, out[:, 1:, :dim])
        assert_close(out[:, 1:, :dim], want, bound)
        assert bool((out[:, 0] == 7).all()) and bool((out[:, :, dim] == 7).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [1, 40, 700]), ([40, 7, 200], [40, 50, 333])])
def test_what_rows_do_not_see_does_not_reach_them(tde, dim, new, lens):
    """NaN and infinities behind the last key, in pages of no sequence, and in the call's later rows."""
    batch = Batch(new, lens, page_size=24, seed=19, pad=3)
    q = randn((batch.tokens, 6, dim), torch.bfloat16, 20)
    k, v = (randn((batch.pages, 24, 2, dim), torch.bfloat16, 21 + i) for i in (0, 1))
    used = torch.zeros((batch.pages, 24), dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            used[batch.page_of(b, j), j % 24] = True
    for x, bad in ((k, float("nan")), (v, float("inf"))):
        x[~used] = bad
    for b, (n, length) in enumerate(zip(new, lens)):
        if n > 3:   # values of later rows: one channel each of +inf, -inf, NaN, both infinities
            for row, channel, bad in ((n - 1, 0, float("nan")), (n - 2, 1, float("inf")), (n - 3, 2, float("-inf")), (n // 2, 3, float("inf")),
                                      (n // 2 + 1, 3, float("-inf")), (n // 2, dim - 1, float("-inf"))):
                p = length - n + row
                v[batch.page_of(b, p), p % 24, :, channel] = bad
            p = length - 1
            k[batch.page_of(b, p), p % 24, 0, 5] = float("nan")
    got = tde.paged_attention(q.cuda(), k.cuda(), v.cuda(), *batch.on("cuda"))
    want, bound = attention(batch, q, k, v, dim ** -0.5)
    assert_close(got, want, bound.nan_to_num(0.0))


@pytest.mark.parametrize("dim", [64, 256])
def test_keys_without_a_page_make_the_rows_that_see_them_nan(tde, dim):
    batch = Batch(new=[1, 1, 60, 1, 30, 1], lens=[100, 100, 100, 5, 64, 90], page_size=16, seed=23)
    batch.table[0, 3] = -1
    batch.table[1, 6] = batch.pages
    batch.table[2, 5] = 2 ** 31 - 1            # keys 80 to 95: rows from position 80 on
    batch.lens[3] = 16 * batch.table.size(1) + 1   # one key beyond the table
    batch.kv_lens[3] = batch.lens[3]
    batch.table[3] = batch.table[0, 0]
    batch.lens[5], batch.kv_lens[5] = 2 ** 31 - 1, 2 ** 31 - 1
    run(tde, batch, 4, 2, dim, torch.bfloat16, seed=24)


@pytest.mark.parametrize("new,lens", [([1, 1], [70, 3000]), ([40, 3], [50, 300]), ([2, 0], [0, 4])])
def test_rows_behind_the_last_sequence(tde, new, lens):
    batch = Batch(new, lens, page_size=16, seed=25, pad=21)
    q = randn((batch.tokens, 4, 64), torch.bfloat16, 26)
    k, v = (randn((batch.pages, 16, 2, 64), torch.bfloat16, 27 + i) for i in (0, 1))
    args = [x.cuda() for x in (q, k, v)] + batch.on("cuda")
    want, bound = attention(batch, q, k, v, 0.125)
    assert_close(tde.paged_attention(*args), want, bound)     # zeros among them
    out = torch.full_like(args[0], 5.0)
    tde.paged_attention_out(*args, out)
    end = int(batch.starts[-1])
    assert_close(out[:end], want[:end], bound[:end])
    assert bool((out[end:] == 5).all())


def test_starts_that_do_not_ascend_stay_in_bounds(tde):
    """What the rows get is unspecified; the call ends and what lies around the output stays."""
    batch = Batch(new=[5, 4, 3], lens=[50, 40, 30], page_size=16, seed=28)
    q = randn((batch.tokens, 4, 64), torch.bfloat16, 29).cuda()
    k, v = (randn((batch.pages, 16, 2, 64), torch.bfloat16, 30 + i).cuda() for i in (0, 1))
    table, _, lens = batch.on("cuda")
    for starts in ([0, 9, 2, 12], [7, -5, 100, 3], [12, 0, 0, 0], [-9, -9, -9, -9], [2 ** 31 - 1] * 4):
        starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        band = torch.full((batch.tokens + 2, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
        tde.paged_attention_out(q, k, v, table, starts, lens, band[1:-1])
        torch.cuda.synchronize()
        assert bool((band[0] == 3).all()) and bool((band[-1] == 3).all())
    # with keys that are split
    batch = Batch(new=[1, 1, 30], lens=[4000, 2000, 900], page_size=16, seed=28)
    q = randn((batch.tokens, 4, 64), torch.bfloat16, 29).cuda()
    k, v = (randn((batch.pages, 16, 2, 64), torch.bfloat16, 30 + i).cuda() for i in (0, 1))
    table, _, lens = batch.on("cuda")
    for starts in ([0, 30, 1, 32], [30, 2, 32, 5], [2, 32, 2, 32], [0, 32, 0, 32]):
        starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        band = torch.full((batch.tokens + 2, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
        tde.paged_attention_out(q, k, v, table, starts, lens, band[1:-1])
        torch.cuda.synchronize()
        assert bool((band[0] == 3).all()) and bool((band[-1] == 3).all())


def test_offsets_beyond_32_bits(tde):
    """A cache of 6 GB whose sequences lie at its end."""
    pages, page, heads, dim = 46000, 64, 8, 128
    k = torch.zeros((pages, page, heads, dim), dtype=torch.bfloat16, device="cuda")
    assert k.numel() * 2 > 5 << 30
    batch = Batch(new=[1, 40], lens=[100, 60], page_size=page, seed=31)
    q = randn((batch.tokens, 16, dim), torch.bfloat16, 32)
    ks, vs = (randn((batch.pages, page, heads, dim), torch.bfloat16, 33 + i) for i in (0, 1))
    v = torch.zeros_like(k)
    k[-batch.pages:], v[-batch.pages:] = ks.cuda(), vs.cuda()
    table, starts, lens = batch.on("cuda")
    got = tde.paged_attention(q.cuda(), k, v, torch.where(table >= 0, table + (pages - batch.pages), table), starts, lens)
    assert_close(got, *attention(batch, q, ks, vs, dim ** -0.5))
    # and appended there
    new = randn((batch.tokens, heads, dim), torch.bfloat16, 36).cuda()
    tde.append_kv(new, new, k, v, torch.where(table >= 0, table + (pages - batch.pages), table), starts, lens)
    for t, b, p in batch.rows():
        assert torch.equal(k[pages - batch.pages + batch.page_of(b, p), p % page], new[t])
    assert not k[: pages - batch.pages].any()


def test_nothing_to_do(tde):
    k = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    empty = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    starts, lens = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    for rows in (0, 3):
        q = torch.ones((rows, 4, 64), dtype=torch.bfloat16, device="cuda")
        out = tde.paged_attention(q, k, k, empty, starts, lens)
        assert out.shape == q.shape and not out.any()


def test_two_graphs_of_split_calls_and_another_stream(tde):
    """Both graphs hold a workspace of their own; lengths, tables and queries change between replays."""
    batch = Batch(new=[1, 1, 1], lens=[3000, 64, 1], page_size=16, seed=37)
    q = randn((3, 8, 128), torch.bfloat16, 38).cuda()
    k, v = (randn((batch.pages, 16, 1, 128), torch.bfloat16, 39 + i).cuda() for i in (0, 1))
    args = [q, k, v] + batch.on("cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = tde.paged_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, tde.paged_attention(*args))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(tde.paged_attention(*args))
        graphs.append(g)
    for replay in range(3):
        q.copy_(randn(q.shape, torch.bfloat16, 50 + replay))
        args[5].copy_(torch.tensor([3000 - 700 * replay, 64 - replay, 1], dtype=torch.int32))
        want = tde.paged_attention(*args)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, s in zip(graphs, streams):   # at once
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    batch.lens = args[5].tolist()
    assert_close(want, *attention(batch, q.cpu(), k.cpu(), v.cpu(), 128 ** -0.5))
