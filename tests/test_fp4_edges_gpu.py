"""The operators of a cache in 4 bits at the edges of what they take: calls that fill the device, scores far from zero, dimensions of one element, rows in
front, other streams, autograd and compiled graphs."""
import pytest
import torch

from block_reference import Batch, assert_close, attention, attention_at_once
from fp4_reference import as_read, decode, encode
from test_block_single_strides_gpu import ODD, with_stride
from test_fp4_cache_gpu import caches, cos_sin
from test_paged_attention_fp4_gpu import held, on_gpu, randn, run
from test_paged_attention_scores_gpu import CALLS, softmax_of, whole

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


# ---- calls of every size ----

@pytest.mark.parametrize("dim,seqs", [(64, 300), (96, 260), (128, 230), (256, 150)])
@pytest.mark.parametrize("page", [16, 8])
def test_tiles_alone_fill_the_device(tde, dim, seqs, page):
    g = torch.Generator().manual_seed(dim)
    new = torch.randint(0, 3, (seqs,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 90, (seqs,), generator=g))]
    lens[5], new[5], new[7], lens[7] = 1200, 2, 6, 700
    run(tde, Batch(new, lens, page, seed=dim, pad=7), 16, 8, dim, torch.bfloat16, seed=dim)
    batch = Batch([1] * seqs, [n + 1 for n in lens], page, seed=dim + 1)
    batch.table[9, 0] = -1
    run(tde, batch, 8, 8, dim, torch.float16, seed=dim + 1, heads_first=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim,page", [(96, 24), (128, 16), (128, 64), (256, 16)])
@pytest.mark.parametrize("new,lens", [([1650, 0, 130], [2000, 5, 130]), ([2300, 900, 1500], [2300, 1000, 3000]), ([1950, 100], [2200, 130])],
                         ids=["few", "many", "long"])
def test_largest_tiles(tde, new, lens, dim, page, dtype):
    """64 heads that share 8; a block of values that is NaN, a page that is none, garbage behind the last keys."""
    batch = Batch(new, lens, page, seed=2, pad=5)
    parts = held(batch, 8, dim, 3)
    parts[3][batch.page_of(0, 300), 300 % page, :, 1] = 255
    last = len(new) - 1
    parts[3][batch.page_of(last, lens[last] - 20), 5, 3, 0] = 255
    for b in (0, last):
        for i in (1, 3):
            parts[i][batch.page_of(b, lens[b] - 1), lens[b] % page or page:] = 255
    batch.table[last, (lens[last] - 1) // page] = -1                                 # (the last: the oracle wants a key in every sequence)
    run(tde, batch, 64, 8, dim, dtype, seed=4, parts=parts, reference=attention_at_once)


@pytest.mark.parametrize("heads,kv_heads,dim,page,new,seqs", [
    (8, 2, 64, 16, 6, 12), (8, 2, 64, 8, 8, 70), (16, 4, 128, 64, 8, 9), (16, 4, 96, 8, 7, 60), (12, 2, 256, 16, 14, 5), (12, 2, 192, 8, 10, 33), (24, 1, 128, 16, 1, 40)])
def test_a_few_tiles_each(tde, heads, kv_heads, dim, page, new, seqs):
    """More than one tile of 16 rows a sequence, on both sides of where larger tiles begin."""
    g = torch.Generator().manual_seed(seqs)
    lens = [new + int(x) for x in torch.randint(0, 400, (seqs,), generator=g)]
    lens[0] = 3000
    for more, dtype in ((0, torch.bfloat16), (new // 2, torch.float16), (3 * new, torch.bfloat16)):
        batch = Batch([new + more] * seqs, [n + more for n in lens], page, seed=seqs, pad=3)
        batch.table[2, 0] = -1
        run(tde, batch, heads, kv_heads, dim, dtype, seed=dim)
    uneven = torch.randint(0, 2 * new + 1, (seqs,), generator=g).tolist()
    run(tde, Batch(uneven, [n + m for n, m in zip(uneven, lens)], page, seed=seqs + 1, pad=20), heads, kv_heads, dim, torch.bfloat16, seed=dim + 1, heads_first=False)


def test_more_heads_than_the_device_holds_workgroups(tde):
    run(tde, Batch([1, 1], [70, 9], 8, seed=1), 1100, 1100, 32, torch.bfloat16, seed=2)
    run(tde, Batch([20], [33], 8, seed=3), 1100, 1100, 32, torch.bfloat16, seed=4)


def test_tiles_alone_with_starts_that_do_not_ascend(tde):
    batch = Batch(new=[1] * 300, lens=[40] * 300, page_size=16, seed=12)
    parts = on_gpu(held(batch, 8, 64, 3))
    table, _, lens = batch.on("cuda")
    q = randn((300, 8, 64), torch.bfloat16, 4).cuda()
    for starts in ([0, 300] * 150 + [0], list(range(300, -1, -1)), [0] + [1 << 30, -5] * 150, [7] * 301):
        whole_out = torch.full((320, 8, 64), 3.0, dtype=torch.bfloat16, device="cuda")
        tde.paged_attention_fp4_out(q, *parts, table, torch.tensor(starts, dtype=torch.int32, device="cuda"), lens, whole_out[10:310])
        torch.cuda.synchronize()
        assert bool((whole_out[:10] == 3).all()) and bool((whole_out[310:] == 3).all())


# ---- scores far from zero or from each other: keys are numbers that codes stand for, so that scores are exact in fp32 ----

def codes_of(batch, kv_heads, dim, rows):
    """Codes and scales that hold rows[b], [keys, kv_heads, dim] in doubles, and what they stand for."""
    made = [torch.zeros((batch.pages, batch.page, kv_heads, n), dtype=torch.uint8) for n in (dim // 2, dim // 32)]
    there = []
    for b, length in enumerate(batch.lens):
        j = torch.arange(length)
        pages = batch.table[b].long()[j // batch.page]
        parts = encode(rows[b].cpu(), 125)
        for to, part in zip(made, parts):
            to[pages, j % batch.page] = part
        there.append(decode(*parts).cuda())
    return [x.cuda() for x in made], there


def values_of(lens, kv_heads, dim, seed):
    """Random codes, between a sixteenth and six eighths."""
    sizes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda") / 8
    return [sizes[whole((n, kv_heads, dim), 0, 7, seed + b).long()] * (whole((n, kv_heads, dim), 0, 1, seed + 50 + b) * 2 - 1) for b, n in enumerate(lens)]


def check(tde, batch, q, keys, values, kv_heads, dtype, scale, weight_step=None):
    heads, dim = q.shape[1:]
    (k, keys), (v, values) = (codes_of(batch, kv_heads, dim, x) for x in (keys, values))
    starts = batch.starts.tolist()

    def scores(b, head):
        return q[starts[b]:starts[b + 1], head] @ keys[b][:, head * kv_heads // heads].t().contiguous() * scale

    got = tde.paged_attention_fp4(q.to(dtype), *k, *v, *batch.on("cuda"), scale)
    assert_close(got, *softmax_of(batch, scores, lambda b, h: values[b][:, h], heads, kv_heads, dim, dtype, weight_step))


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,octaves", [(torch.bfloat16, 0), (torch.bfloat16, 14), (torch.bfloat16, 40), (torch.float16, 0), (torch.float16, 11), (torch.float16, 13)], ids=str)
def test_large_scores(tde, call, dim, dtype, octaves):
    new, lens, heads, kv_heads = CALLS[call]
    batch = Batch(new, lens, page_size=16, seed=1)
    q = whole((batch.tokens, heads, dim), -3, 3, 2) * 2.0 ** octaves
    keys = [whole((n, kv_heads, dim), -3, 3, 3 + b) * 2.0 ** octaves for b, n in enumerate(lens)]
    check(tde, batch, q, keys, values_of(lens, kv_heads, dim, 1000), kv_heads, dtype, 2.0 ** -6)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("offset", [0, 768, 1 << 12, 1 << 15, -(1 << 12)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_scores_with_a_common_offset(tde, call, offset, dtype):
    """Scores that rise along the keys, all far from zero: maxima move and parts are joined there."""
    new, lens, heads, kv_heads = CALLS[call]
    batch, dim = Batch(new, lens, page_size=24, seed=4), 96
    q = whole((batch.tokens, heads, dim), -1, 1, 5)
    q[..., :64], q[..., 0], q[..., 32] = 0.0, 32.0, 32.0
    keys = [whole((n, kv_heads, dim), -1, 1, 6 + b) for b, n in enumerate(lens)]
    for x in keys:
        x[..., :64], x[..., 0], x[..., 32] = 0.0, offset / 8.0, (torch.arange(x.size(0), device="cuda") // 16)[:, None] / 32.0
    check(tde, batch, q, keys, values_of(lens, kv_heads, dim, 1000), kv_heads, dtype, 0.25)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("nats", [8.0, 16.0, 24.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_a_key_that_takes_nearly_all_weight(tde, call, nats, dtype):
    """One key far above all others, whose value is zero: what is left is the sum of the others' small weights."""
    new, lens, heads, kv_heads = CALLS[call]
    new, lens = ([1, 1], [20000, 130]) if call == "decode" else (new, lens)
    batch, dim = Batch(new, lens, page_size=16, seed=7), 64
    q = torch.zeros((batch.tokens, heads, dim), dtype=torch.float64, device="cuda")
    q[..., 0] = 1.0
    keys = [torch.zeros((n, kv_heads, dim), dtype=torch.float64, device="cuda") for n in lens]
    values = [x.abs() + 0.5 for x in values_of(lens, kv_heads, dim, 1000)]
    for b, x in enumerate(keys):
        x[..., 0] = whole(x.shape[:2], -8, 8, 2000 + b) / 64
        at = x.size(0) // 3 if b % 2 else 0
        x[at, :, 0], values[b][at] = nats, 0.0
    check(tde, batch, q, keys, values, kv_heads, dtype, 1.0)


@pytest.mark.parametrize("call", ["decode", "decode whole"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_decode_rows_are_off_by_their_own_rounding(tde, call, dim, dtype):
    """Weights are two numbers of T, each within a step: a step of a step of a weight is lost at most."""
    new, lens, heads, kv_heads = CALLS[call]
    batch = Batch(new, lens, page_size=16, seed=11)
    q = whole((batch.tokens, heads, dim), -3, 3, 12)
    keys = [whole((n, kv_heads, dim), -3, 3, 13 + b) for b, n in enumerate(lens)]
    check(tde, batch, q, keys, values_of(lens, kv_heads, dim, 1000), kv_heads, dtype, 2.0 ** -5, torch.finfo(dtype).eps ** 2)


# ---- layouts ----

@pytest.mark.parametrize("stride", ODD)
@pytest.mark.parametrize("page,kv_heads", [(64, 2), (1, 2), (16, 1)])
def test_dimensions_of_one_element_have_any_stride(tde, stride, page, kv_heads):
    batch = Batch([1], [40 if page > 1 else 1], page_size=page, seed=1, extra_pages=0)
    table, starts, lens = batch.on("cuda")
    cache = [x.contiguous().cuda() for x in caches(batch, kv_heads, 64, page)]
    rows = randn((1, 8, 64), torch.bfloat16, page).cuda()
    q, k, v = rows.split([8 - 2 * kv_heads, kv_heads, kv_heads], dim=1)
    want_cache = [x.clone() for x in cache]
    tde.append_kv_fp4(k, v, *want_cache, table, starts, lens)
    want = tde.paged_attention_fp4(q, *want_cache, table, starts, lens)
    odd = list(cache)
    for d in range(3):
        if cache[0].size(d) == 1:
            odd = [with_stride(x, d, stride) for x in odd]
    table = with_stride(table, 0, stride)
    rows = [with_stride(x, 0, stride) for x in (q, k, v)]
    if kv_heads == 1:
        rows[1:] = [with_stride(x, 1, stride) for x in rows[1:]]
    tde.append_kv_fp4(*rows[1:], *odd, table, starts, lens)
    assert all(torch.equal(a, b) for a, b in zip(cache, want_cache))
    assert torch.equal(tde.paged_attention_fp4(rows[0], *odd, table, starts, lens), want)
    out = torch.zeros_like(want)
    tde.paged_attention_fp4_out(rows[0], *odd, table, starts, lens, with_stride(out, 0, stride))
    assert torch.equal(out, want)
    assert torch.equal(tde.unpack_fp4(*odd[:2]), tde.unpack_fp4(*cache[:2]))
    free, count, new = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1, 2], [3], [1]))
    states = [[t.clone() for t in (lens, free, count)] for _ in (0, 1)]
    wide = torch.full((1, batch.table.size(1) + 2), -1, dtype=torch.int32, device="cuda")
    both = [wide.clone(), with_stride(wide.clone(), 0, stride)]
    got = [tde.update_pages(t, s[0], new, s[1], s[2], page, 3) for t, s in zip(both, states)]
    assert all(torch.equal(a, b) for a, b in zip([*got[0], both[0], *states[0]], [*got[1], both[1], *states[1]]))


@pytest.mark.parametrize("front", [1, 70])
@pytest.mark.parametrize("new,lens", [([3, 0, 40], [10, 7, 41]), ([1] * 300, [20] * 300)])
def test_rows_in_front(tde, new, lens, front):
    """q_starts that begin above 0: those rows are nobody's."""
    batch = Batch(new, lens, 16, seed=6, pad=3)
    table, starts, lengths = batch.on("cuda")
    starts, tokens = starts + front, batch.tokens + front
    rows, cs = randn((tokens, 8, 64), torch.bfloat16, 7).cuda(), cos_sin(50, 64).cuda()
    cache = [[x.contiguous().cuda() for x in caches(batch, 2, 64, 8)] for _ in (0, 1)]
    q, k, v = rows.split([4, 2, 2], dim=1)
    got = tde.append_kv_fp4(k, v, *cache[0], table, starts, lengths, cos_sin=cs, q=q)
    want = tde.append_kv_fp4(k[front:], v[front:], *cache[1], table, starts - front, lengths, cos_sin=cs, q=q[front:])
    assert not bool(got[:front].any()) and not bool(got[-3:].any()) and torch.equal(got[front:], want)
    assert all(torch.equal(a, b) for a, b in zip(*cache))
    got = tde.paged_attention_fp4(q, *cache[0], table, starts, lengths)
    want, bound = attention(batch, q[front:].cpu(), as_read(*[x.cpu() for x in cache[0][:2]], torch.bfloat16), as_read(*[x.cpu() for x in cache[0][2:]], torch.bfloat16), 64 ** -0.5)
    assert not bool(got[:front].any()) and not bool(got[-3:].any())
    assert_close(got[front:], want, bound)
    out = torch.full_like(got, 5.0)
    tde.paged_attention_fp4_out(q, *cache[0], table, starts, lengths, out)
    assert torch.equal(out[front:-3], got[front:-3]) and bool((out[:front] == 5).all()) and bool((out[-3:] == 5).all())


# ---- streams, autograd, compiled graphs ----

def a_step(seqs=3, page=16, dim=64):
    batch = Batch([1] * seqs, [40, 17, 1][:seqs], page, seed=8)
    cache = [x.contiguous().cuda() for x in caches(batch, 1, dim, 9)]
    qkv = randn((seqs, 6, dim), torch.bfloat16, 10).cuda()
    return batch, cache, qkv


def test_on_other_streams(tde):
    """Four streams, each with a server's state of its own, a few steps each."""
    def state():
        batch, cache, qkv = a_step()
        free = torch.arange(100, 120, dtype=torch.int32, device="cuda") % batch.pages
        wide = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
        wide[:, :batch.table.size(1)] = batch.table.cuda()
        return wide, batch.kv_lens.cuda(), free, torch.tensor([20], dtype=torch.int32, device="cuda"), cache, qkv

    def steps(table, lens, free, count, cache, qkv):
        new, outs = torch.ones(3, dtype=torch.int32, device="cuda"), []
        for _ in range(4):
            starts, positions, _ = tde.update_pages(table, lens, new, free, count, 16, 4)
            rows = torch.cat([qkv, qkv[:1]])
            q = tde.append_kv_fp4(rows[:, 4:5], rows[:, 5:], *cache, table, starts, lens, q=rows[:, :4])
            outs += [q, tde.paged_attention_fp4(q, *cache, table, starts, lens), tde.unpack_fp4(*cache[:2]), positions]
        return outs

    want = steps(*state())
    torch.cuda.synchronize()
    states, got = [state() for _ in range(4)], []
    torch.cuda.synchronize()
    for s in states:
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got.append(steps(*s))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for outs in got for a, b in zip(outs, want))


@pytest.mark.parametrize("queries", [False, True])
def test_changes_count_as_changes(tde, queries):
    batch, cache, qkv = a_step()
    before = [x._version for x in cache]
    tde.append_kv_fp4(qkv[:, 4:5], qkv[:, 5:], *cache, *batch.on("cuda"), q=qkv[:, :4] if queries else None)
    assert all(x._version > n for x, n in zip(cache, before))
    before, out = [x._version for x in cache], torch.zeros_like(qkv[:, :4])
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = (out * w).sum()
    tde.paged_attention_fp4_out(qkv[:, :4], *cache, *batch.on("cuda"), out)
    assert [x._version for x in cache] == before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_parameters_give_plain_tensors_and_inference_works(tde):
    batch, cache, qkv = a_step()
    gamma = torch.nn.Parameter(torch.ones(64, device="cuda", dtype=torch.bfloat16))
    rows = qkv.clone().requires_grad_()
    q = tde.append_kv_fp4(rows[:, 4:5], rows[:, 5:], *cache, *batch.on("cuda"), q=rows[:, :4], q_gamma=gamma, k_gamma=gamma)
    assert not q.requires_grad and not tde.paged_attention_fp4(rows[:, :4], *cache, *batch.on("cuda")).requires_grad
    with torch.inference_mode():
        cache = tde.fp4_cache(batch.pages, 16, 1, 64)
        table, starts, lens = batch.on("cuda")
        count, free = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
        starts, _, _ = tde.update_pages(table, lens, torch.zeros(3, dtype=torch.int32, device="cuda"), free, count, 16, 3, keep_lens=lens.clone())
        assert not bool(starts.any())
        tde.append_kv_fp4(qkv[:, 4:5], qkv[:, 5:], *cache, *batch.on("cuda"))
        out = torch.zeros_like(qkv[:, :4])
        tde.paged_attention_fp4_out(qkv[:, :4], *cache, *batch.on("cuda"), out)
        assert torch.equal(out, tde.paged_attention_fp4(qkv[:, :4], *cache, *batch.on("cuda")))


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_under_torch_compile(tde, backend):
    if backend == "inductor":
        pytest.importorskip("triton")
        import torch._inductor.config as inductor_config
        inductor_config.compile_threads = 1      # compile in this process: no pool of worker processes
    from torch._dynamo.exc import BackendCompilerFailed
    batch, cache, qkv = a_step()
    gamma, cs = torch.ones(64, dtype=torch.bfloat16, device="cuda"), cos_sin(64, 64).cuda()
    wide = torch.full((3, 6), -1, dtype=torch.int32)
    wide[:, :batch.table.size(1)] = batch.table
    free = torch.arange(2, dtype=torch.int32, device="cuda") + batch.pages - 2

    def step(rows, table, lens, free, count, k_cache, k_scales, v_cache, v_scales, out):
        starts, positions, slots = tde.update_pages(table, lens, torch.ones_like(lens), free, count, 16, 3)
        q = tde.append_kv_fp4(rows[:, 4:5] * 2, rows[:, 5:], k_cache, k_scales, v_cache, v_scales, table, starts, lens, cos_sin=cs, positions=positions, q=rows[:, :4],
                              q_gamma=gamma, k_gamma=gamma)
        tde.paged_attention_fp4_out(q, k_cache, k_scales, v_cache, v_scales, table, starts, lens, out)
        back = tde.unpack_fp4(k_cache, k_scales).float() + 1
        return tde.paged_attention_fp4(q, k_cache, k_scales, v_cache, v_scales, table, starts, lens).float() + 1, back, slots + 1

    results = []
    for f in (step, torch.compile(step, backend=backend, fullgraph=True)):
        args = [wide.cuda(), batch.kv_lens.cuda(), free.clone(), torch.tensor([2], dtype=torch.int32, device="cuda"), *(x.clone() for x in cache), torch.zeros_like(qkv[:, :4])]
        try:
            outs = f(qkv, *args)
        except BackendCompilerFailed as e:   # the code generator, not this library
            pytest.skip("torch.compile backend unavailable here: %s" % str(e)[:200])
        torch.cuda.synchronize()
        results.append([*outs, *args])
    for i, (got, want) in enumerate(zip(results[1], results[0])):
        assert torch.equal(got, want), i
    assert not torch.equal(results[0][7], cache[0]) and torch.equal(results[0][0], results[0][-1].float() + 1)
