"""paged_attention_fp4 against the attention's definition in doubles over the numbers that its codes stand for."""
import math

import pytest
import torch

from block_reference import Batch, assert_close, attention, attention_at_once
from fp4_reference import as_read, random_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def held(batch, kv_heads, dim, seed, heads_first=True):
    """Codes and scales of keys and of values, on the CPU."""
    shape = (batch.pages, kv_heads, batch.page) if heads_first else (batch.pages, batch.page, kv_heads)
    parts = [x for i in (0, 1) for x in random_cache(shape, dim, seed + i)]
    return [x.transpose(1, 2) for x in parts] if heads_first else parts


def on_gpu(parts):
    """With their strides."""
    return [torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda").copy_(x) for x in parts]


def run(tde, batch, heads, kv_heads, dim, dtype, seed=0, scale=None, spread=1.0, heads_first=True, parts=None, reference=attention):
    q = randn((batch.tokens, heads, dim), dtype, seed, spread)
    parts = held(batch, kv_heads, dim, seed + 1, heads_first) if parts is None else parts
    got = tde.paged_attention_fp4(q.cuda(), *on_gpu(parts), *batch.on("cuda"), scale)
    k, v = as_read(*parts[:2], dtype), as_read(*parts[2:], dtype)
    if reference is attention_at_once:
        want, bound = reference(batch, q.cuda(), k.cuda(), v.cuda(), dim ** -0.5 if scale is None else scale)
    else:
        want, bound = reference(batch, q, k, v, dim ** -0.5 if scale is None else scale)
    assert_close(got, want, bound)


SHAPES = [(1, 1, 32, 1), (4, 4, 64, 16), (8, 1, 128, 64), (6, 2, 64, 3), (10, 2, 96, 24), (7, 1, 96, 16), (16, 1, 128, 128), (5, 5, 128, 8), (12, 4, 192, 16),
          (8, 2, 256, 32), (34, 2, 64, 16), (3, 1, 256, 5), (4, 2, 160, 16), (2, 2, 224, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_lengths_and_shapes(tde, heads, kv_heads, dim, page, dtype):
    decode = Batch(new=[1, 1, 1, 1, 1, 1, 1], lens=[1, 2, 31, 64, 65, 300, 1000], page_size=page, seed=1)
    run(tde, decode, heads, kv_heads, dim, dtype, seed=dim)
    # chunks; sequences without rows, without keys, shorter than their rows; rows behind the last sequence
    ragged = Batch(new=[5, 0, 17, 1, 3, 2, 70, 0], lens=[5, 9, 40, 513, 2, 0, 130, 0], page_size=page, pad=9, seed=2)
    run(tde, ragged, heads, kv_heads, dim, dtype, seed=dim + 9, heads_first=False)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (2, 2), (3, 1)])
def test_long_chunks(tde, dim, heads, kv_heads):
    run(tde, Batch(new=[333], lens=[700], page_size=16, seed=3), heads, kv_heads, dim, torch.bfloat16, seed=4)
    run(tde, Batch(new=[129, 64, 250], lens=[129, 1024, 255], page_size=24, seed=5, pad=1), heads, kv_heads, dim, torch.float16, seed=6)


@pytest.mark.parametrize("dim", [32, 128, 192, 256])
def test_calls_that_fill_the_units(tde, dim):
    """Enough rows for the largest tiles."""
    run(tde, Batch([1200, 300, 1100], [1500, 300, 3000], 16, seed=2, pad=5), 16, 8, dim, torch.bfloat16, seed=3, reference=attention_at_once)


@pytest.mark.parametrize("seqs", [64, 65, 129, 300])
def test_many_sequences(tde, seqs):
    g = torch.Generator().manual_seed(seqs)
    new = torch.randint(0, 3, (seqs,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 40, (seqs,), generator=g))]
    run(tde, Batch(new, lens, page_size=8, seed=7, pad=5), 4, 2, 64, torch.bfloat16, seed=8)
    run(tde, Batch([1] * seqs, [x + 1 for x in lens], page_size=8, seed=9), 4, 2, 128, torch.bfloat16, seed=10)


@pytest.mark.parametrize("heads,kv_heads,dim,lens", [(8, 1, 128, [20000]), (2, 2, 64, [9000, 3, 700]), (4, 1, 256, [6000, 100]), (16, 2, 96, [5000])])
def test_one_token_behind_many(tde, heads, kv_heads, dim, lens):
    run(tde, Batch([1] * len(lens), lens, page_size=64, seed=11), heads, kv_heads, dim, torch.bfloat16, seed=12)
    run(tde, Batch([9] * len(lens), [n + 9 for n in lens], page_size=16, seed=11, pad=2), heads, kv_heads, dim, torch.float16, seed=13)
    run(tde, Batch([1] * len(lens), lens, page_size=5, seed=11), heads, kv_heads, dim, torch.float16, seed=14, heads_first=False)


def test_scales_and_peaked_softmax(tde):
    batch = Batch(new=[1, 20, 80], lens=[200, 300, 80], page_size=16, seed=14)
    run(tde, batch, 4, 2, 128, torch.bfloat16, seed=15, scale=2.0)              # weights concentrate on few keys
    run(tde, batch, 4, 2, 128, torch.bfloat16, seed=16, scale=1e-3)             # nearly uniform
    run(tde, batch, 4, 2, 64, torch.float16, seed=17, scale=0.125, spread=8.0)
    decode = Batch(new=[1, 1, 2], lens=[200, 3000, 80], page_size=16, seed=14)
    run(tde, decode, 4, 2, 128, torch.bfloat16, seed=15, scale=2.0)
    run(tde, decode, 4, 2, 64, torch.float16, seed=15, scale=1e-3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("new", [[1, 1, 2], [40, 90, 7]], ids=["decode", "chunks"])
def test_every_scale_byte(tde, dtype, new):
    """Blocks of any size, from far below what T holds (fp16) to as large as scores of finite numbers allow."""
    batch = Batch(new=new, lens=[300, 90, 700], page_size=16, seed=3)
    parts = held(batch, 2, 64, 5)
    g = torch.Generator().manual_seed(1)
    lo, hi = (100, 131) if dtype == torch.float16 else (2, 131)
    for s in (parts[1], parts[3]):
        s.copy_(torch.randint(lo, hi + 1, s.shape, generator=g))
    run(tde, batch, 4, 2, 64, dtype, seed=6, scale=0.02, parts=parts)


@pytest.mark.parametrize("which", [1, 3], ids=["keys", "values"])
def test_blocks_beyond_fp16_are_nan(tde, which):
    """Blocks whose 6 fp16 does not hold are NaN for the rows that see them, and the largest that it holds are numbers."""
    for new in ([3], [90]):
        batch = Batch(new=new, lens=[150], page_size=16, seed=4)
        parts = held(batch, 1, 64, 7)
        j = 150 - new[0] + 1                                                       # the second new row's key
        parts[which][batch.page_of(0, j), j % 16, 0, 1] = 127 + 14
        parts[3][batch.page_of(0, 5), 5, 0, 0] = 127 + 13
        run(tde, batch, 2, 1, 64, torch.float16, seed=8, parts=parts)
        parts[which][batch.page_of(0, j), j % 16, 0, 1] = 127 + 13
        run(tde, batch, 2, 1, 64, torch.float16, seed=8, parts=parts, scale=1e-5)


@pytest.mark.parametrize("new,lens", [([2, 1, 3], [90, 2000, 40]), ([70, 150, 3], [90, 200, 40])], ids=["decode", "chunks"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_blocks_that_are_nan(tde, new, lens, dim):
    """A NaN block of values makes its 32 channels NaN for rows that see the key; one of keys all that such rows have; others see nothing of either.
    Neither do slots behind a sequence's last key reach anything."""
    batch = Batch(new=new, lens=lens, page_size=16, seed=5, pad=2)
    for which in (1, 3):
        parts = held(batch, 2, dim, 9)
        for b, (n, length) in enumerate(zip(new, lens)):
            j = length - n + n // 2
            parts[which][batch.page_of(b, j), j % 16, b % 2, dim // 64] = 255
            for s in range(length % 16, 16 if length % 16 else 0):                  # unused slots of the last page
                for i in (1, 3):
                    parts[i][batch.page_of(b, length - 1), s] = 255
        run(tde, batch, 4, 2, dim, torch.bfloat16, seed=10, parts=parts)
        run(tde, batch, 4, 2, dim, torch.float16, seed=11, parts=parts)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_behind_the_last_key_of_one_token(tde, dim):
    """A tile of 64 rows that all see the same keys, in a page whose other slots are NaN."""
    batch = Batch(new=[1, 1], lens=[67, 200], page_size=16, seed=6)
    parts = held(batch, 1, dim, 15)
    for b, length in enumerate(batch.lens):
        parts[1][batch.page_of(b, length - 1), length % 16:] = 255
        parts[3][batch.page_of(b, length - 1), length % 16:] = 255
    run(tde, batch, 64, 1, dim, torch.bfloat16, seed=16, parts=parts)
    run(tde, batch, 64, 1, dim, torch.float16, seed=16, parts=parts)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 1, 70, 9]], ids=["decode", "chunks"])
def test_pages_that_are_none(tde, new):
    batch = Batch(new=new, lens=[100, 700, 90, 64], page_size=16, seed=6)
    batch.table[1, 20], batch.table[2, 5], batch.table[3, 3] = -1, batch.pages, 0x7fffffff
    run(tde, batch, 4, 2, 128, torch.bfloat16, seed=12)
    run(tde, Batch(new=new, lens=[100, 700, 90, 64], page_size=16, seed=6, table_pages=5), 4, 2, 64, torch.float16, seed=13)


def test_rows_of_no_sequence(tde):
    """Rows in front of the first sequence and behind the last: zeros, or left as they were."""
    for new, lens in (([1, 1], [400, 30]), ([60, 9], [400, 30])):
        batch = Batch(new=new, lens=lens, page_size=16, seed=7, pad=6)
        parts = held(batch, 2, 64, 14)
        q = randn((batch.tokens + 4, 4, 64), torch.bfloat16, 15)
        table, starts, lengths = batch.on("cuda")
        starts = starts + 4
        got = tde.paged_attention_fp4(q.cuda(), *on_gpu(parts), table, starts, lengths)
        want, bound = attention(batch, q[4:], as_read(*parts[:2], torch.bfloat16), as_read(*parts[2:], torch.bfloat16), 64 ** -0.5)
        assert_close(got[4:], want, bound)
        assert not bool(got[:4].any()) and not bool(got[-6:].any())
        out = torch.full_like(got, 7.0)
        before = out._version
        tde.paged_attention_fp4_out(q.cuda(), *on_gpu(parts), table, starts, lengths, out)
        assert out._version > before
        assert torch.equal(out[4:-6], got[4:-6]) and bool((out[:4] == 7).all()) and bool((out[-6:] == 7).all())


def test_the_same_call_gives_the_same_bits(tde):
    batch = Batch(new=[1] * 5, lens=[3000, 100, 20000, 1, 64], page_size=64, seed=8)
    q, parts = randn((batch.tokens, 8, 128), torch.bfloat16, 1).cuda(), on_gpu(held(batch, 2, 128, 2))
    first = tde.paged_attention_fp4(q, *parts, *batch.on("cuda"))
    assert all(torch.equal(first, tde.paged_attention_fp4(q, *parts, *batch.on("cuda"))) for _ in range(3))


@pytest.mark.parametrize("lens,new", [([6000, 9000], 1), ([500, 700], 100)])
def test_captured_calls_follow_their_arrays(tde, lens, new):
    batch = Batch(new=[new] * len(lens), lens=lens, page_size=64, seed=9)
    q, parts = randn((batch.tokens, 8, 128), torch.bfloat16, 1).cuda(), on_gpu(held(batch, 2, 128, 2))
    table, starts, lengths = batch.on("cuda")
    graphs, outs = [], []
    for _ in (0, 1):                                                               # two graphs: each has a workspace of its own
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(tde.paged_attention_fp4(q, *parts, table, starts, lengths))
    for i in range(4):
        q.copy_(randn(q.shape, torch.bfloat16, 20 + i))
        lengths.sub_(3 * i)
        eager = tde.paged_attention_fp4(q, *parts, table, starts, lengths)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, eager) for o in outs)


def test_two_streams_at_once(tde):
    batch = Batch(new=[1] * 3, lens=[9000, 100, 5000], page_size=64, seed=10)
    q, parts = randn((batch.tokens, 8, 128), torch.bfloat16, 1).cuda(), on_gpu(held(batch, 1, 128, 2))
    where = batch.on("cuda")
    want = tde.paged_attention_fp4(q, *parts, *where)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(4)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(tde.paged_attention_fp4(q, *parts, *where))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_strided_rows_and_shared_caches(tde):
    batch = Batch(new=[1, 30], lens=[500, 90], page_size=16, seed=11)
    parts = held(batch, 2, 64, 3)
    parts[2:] = parts[:2]                                                          # one tensor may be keys and values: it is only read
    q = randn((batch.tokens, 9, 64), torch.bfloat16, 4)
    here = on_gpu(parts[:2])
    got = tde.paged_attention_fp4(q.cuda()[:, 2:6], *here, *here, *batch.on("cuda"))
    k = as_read(*parts[:2], torch.bfloat16)
    want, bound = attention(batch, q[:, 2:6].contiguous(), k, k, 64 ** -0.5)
    assert_close(got, want, bound)
    out = torch.zeros((batch.tokens, 4, 100), dtype=torch.bfloat16, device="cuda")
    tde.paged_attention_fp4_out(q.cuda()[:, 2:6], *here, *here, *batch.on("cuda"), out[..., 3:67])
    assert torch.equal(out[..., 3:67], got) and not bool(out[..., :3].any()) and not bool(out[..., 67:].any())
    # scales of any alignment beside their codes' rows
    rows = torch.zeros((batch.pages, 16, 2, 48), dtype=torch.uint8, device="cuda")
    rows[..., :32], rows[..., 35:37] = here[0], here[1]
    again = tde.paged_attention_fp4(q.cuda()[:, 2:6], rows[..., :32], rows[..., 35:37], rows[..., :32], rows[..., 35:37], *batch.on("cuda"))
    assert torch.equal(again, got)


def test_starts_that_do_not_ascend(tde):
    """What the rows get is unspecified; nothing outside the call's rows is touched, and the call ends."""
    batch = Batch(new=[1] * 40, lens=[300] * 40, page_size=16, seed=12)
    parts = on_gpu(held(batch, 2, 64, 3))
    table, _, lens = batch.on("cuda")
    q = randn((40, 4, 64), torch.bfloat16, 4).cuda()
    for starts in ([0, 40] * 20 + [0], list(range(40, -1, -1)), [0] + [1 << 30, -5] * 20, [7] * 41):
        whole = torch.full((60, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
        tde.paged_attention_fp4_out(q, *parts, table, torch.tensor(starts, dtype=torch.int32, device="cuda"), lens, whole[10:50])
        torch.cuda.synchronize()
        assert bool((whole[:10] == 3).all()) and bool((whole[50:] == 3).all())


def test_far_pages(tde):
    """Codes more than 4 GiB apart."""
    page_bytes, pages = 16 * 32, 9
    far = torch.zeros(9 * (1 << 29) + page_bytes, dtype=torch.uint8, device="cuda")
    k_cache = far.as_strided((pages, 16, 1, 32), (1 << 29, 32, 32, 1))
    batch = Batch(new=[1, 40], lens=[60, 75], page_size=16, seed=12, extra_pages=0)
    assert batch.pages == pages
    parts = held(batch, 1, 64, 6, heads_first=False)
    here = on_gpu(parts)
    k_cache.copy_(here[0])
    q = randn((batch.tokens, 2, 64), torch.bfloat16, 7)
    got = tde.paged_attention_fp4(q.cuda(), k_cache, here[1], here[2], here[3], *batch.on("cuda"))
    want, bound = attention(batch, q, as_read(*parts[:2], torch.bfloat16), as_read(*parts[2:], torch.bfloat16), 64 ** -0.5)
    assert_close(got, want, bound)


@pytest.mark.parametrize("which", range(4), ids=["k_cache", "k_scales", "v_cache", "v_scales"])
@pytest.mark.parametrize("new,lens", [([1, 2], [60, 75]), ([1, 150], [60, 275])], ids=["decode", "chunks"])
def test_slots_far_apart(tde, which, new, lens):
    """16 keys whose offsets from the first of them do not hold 32 bits."""
    slot = (1 << 28) + (1 << 24)
    batch = Batch(new=new, lens=lens, page_size=16, seed=14)
    parts = held(batch, 1, 64, 7, heads_first=False)
    here = on_gpu(parts)
    width = here[which].size(3)
    far = torch.zeros(15 * slot + batch.pages * width, dtype=torch.uint8, device="cuda")
    here[which] = far.as_strided((batch.pages, 16, 1, width), (width, slot, width, 1)).copy_(here[which])
    for dtype in (torch.bfloat16, torch.float16):
        q = randn((batch.tokens, 2, 64), dtype, 8)
        got = tde.paged_attention_fp4(q.cuda(), *here, *batch.on("cuda"))
        want, bound = attention(batch, q, as_read(*parts[:2], dtype), as_read(*parts[2:], dtype), 64 ** -0.5)
        assert_close(got, want, bound)


def test_nothing_to_do(tde):
    batch = Batch(new=[0, 0], lens=[5, 0], page_size=4)
    parts = on_gpu(held(batch, 2, 64, 1))
    q = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    assert tde.paged_attention_fp4(q, *parts, *batch.on("cuda")).shape == (0, 4, 64)
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    assert not bool(tde.paged_attention_fp4(q, *parts, *batch.on("cuda")).any())
    none = torch.zeros((0, 5), dtype=torch.int32, device="cuda")
    assert not bool(tde.paged_attention_fp4(q, *parts, none, torch.zeros(1, dtype=torch.int32, device="cuda"), none[:, 0].contiguous()).any())


def test_refusals(tde):
    batch = Batch(new=[3], lens=[5], page_size=4, seed=13)
    parts = on_gpu(held(batch, 2, 64, 1))
    q = randn((3, 4, 64), torch.bfloat16, 2).cuda()
    names = ("k_cache", "k_scales", "v_cache", "v_scales")

    def call(q=q, out=None, scale=None, **kw):
        c = dict(zip(names, parts))
        c.update(kw)
        if out is not None:
            return tde.paged_attention_fp4_out(q, *(c[n] for n in names), *batch.on("cuda"), out, scale)
        return tde.paged_attention_fp4(q, *(c[n] for n in names), *batch.on("cuda"), scale)

    call()
    moved = torch.zeros(parts[0].numel() + 16, dtype=torch.uint8, device="cuda")[1:1 + parts[0].numel()].view(batch.pages, 4, 2, 32)
    bytes_of_q = q.view(torch.uint8).view(-1)
    for kw, match in ((dict(q=q.float()), "dtype"), (dict(q=q.cpu()), "GPU"), (dict(q=q[:, :3]), "multiple"), (dict(q=q[..., :48]), "steps of 32"), (dict(q=q[0]), "q must"),
                      (dict(k_cache=parts[0].int()), "uint8"), (dict(k_cache=parts[0][..., :16]), "k_cache must be"), (dict(v_cache=parts[2][:, :, :1]), "v_cache must be"),
                      (dict(k_scales=parts[1][..., :1]), "k_scales must be"), (dict(v_scales=parts[3][:-1]), "differs"), (dict(v_scales=parts[3].cpu()), "GPU"),
                      (dict(v_cache=parts[2][:-1], v_scales=parts[3][:-1]), "differ in pages"), (dict(k_cache=moved), "align"),
                      (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=3e38), "scale"),
                      (dict(out=q), "overlaps q"), (dict(out=q[:, :2]), "shaped"), (dict(out=torch.zeros_like(q[:1]).expand(3, 4, 64)), "overlap"),
                      (dict(out=torch.zeros_like(q).float()), "dtype")):
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    scales = bytes_of_q[:batch.pages * 4 * 2 * 2].view(batch.pages, 4, 2, 2)
    with pytest.raises(RuntimeError, match="overlaps k_scales"):
        call(q=randn((3, 4, 64), torch.bfloat16, 3).cuda(), out=q, k_scales=scales)
