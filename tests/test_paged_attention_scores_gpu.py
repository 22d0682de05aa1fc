"""paged_attention where a row's scores are far from zero or far from each other, with bounds that count roundings."""
import pytest
import torch

from block_reference import U32, Batch, assert_close, half_step, smallest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


# which kernel: one row split over many keys, rows whole, tiles of 64 and (with 64 heads that share 8) of 128 rows
CALLS = {
    "decode": ([1, 1], [3000, 130], 4, 2),
    "decode whole": ([1] * 300, [70] * 300, 4, 4),
    "chunk": ([150, 3], [900, 200], 4, 1),
    "large chunk": ([1700], [1700], 64, 8),
}


def softmax_of(batch, scores_of, values_of, heads, kv_heads, dim, dtype, weight_step=None):
    """From scores [rows, keys] that are exact in doubles and in fp32.  A weight enters twice, in numerator and sum, each time off

    - by half a step of T, an absolute one among T's subnormal numbers: 2^-36 of the largest weight in fp16, whose largest one is raised to 2^11 at
      least; in bf16 what lies below fp32's 2^-126 may be gone;
    - by what its exponent is off.  A score d below the row's largest (by way of maxima that lag by up to 12): three roundings of d, the
      scale's, the difference's, the product's.  Products of a maximum and the scale that are kept rounded, up to 1024 octaves, and raised: 2^-15 of an
      octave twice, 2 * 2^9 * log 2 units of 2^-24, in each of two maxima that meet, which they do twice (wavefronts, launches)."""
    out, bound = torch.zeros((batch.tokens, heads, dim), dtype=torch.float64), torch.zeros((batch.tokens, heads, dim), dtype=torch.float64)
    h, at = half_step(dtype), 0
    weight_step = h if weight_step is None else weight_step
    lost = 2.0 ** -36 if dtype == torch.float16 else 2.0 ** -126
    for b, (new, length) in enumerate(zip(batch.new, batch.lens)):
        sees = torch.arange(length, device="cuda")[None] <= torch.arange(length - new, length, device="cuda")[:, None]
        for head in range(heads):
            v = values_of(b, head * kv_heads // heads)
            s = torch.where(sees, scores_of(b, head), -torch.inf)
            w = torch.softmax(s, dim=-1)
            o, beyond = w @ v, sees.double() @ v.abs()
            counts = sees.sum(-1, keepdim=True)
            distance = (s.amax(-1, keepdim=True) - s).clamp(max=2000.0)
            wrong = w * (weight_step + (3 * (distance + 12) + 8 * 355 + counts + 16) * U32)
            out[at:at + new, head] = o.cpu()
            bound[at:at + new, head] = ((wrong @ v.abs() + wrong.sum(-1, keepdim=True) * o.abs()) * 1.02 + (h * o.abs() + smallest(dtype)) * 1.02
                                        + lost * (beyond + counts * o.abs()) * w.amax(-1, keepdim=True)).cpu()
        at += new
    return out, bound


def caches(batch, kv_heads, dim, dtype, keys, values):
    """Paged caches that hold keys[b] and values[b], [keys, kv_heads, dim]."""
    k, v = (torch.zeros((batch.pages, batch.page, kv_heads, dim), dtype=dtype, device="cuda") for _ in (0, 1))
    for b, length in enumerate(batch.lens):
        j = torch.arange(length)
        pages = batch.table[b].long()[j // batch.page]
        k[pages.cuda(), (j % batch.page).cuda()], v[pages.cuda(), (j % batch.page).cuda()] = keys[b].to(dtype), values[b].to(dtype)
    return k, v


def whole(shape, low, high, seed):
    return torch.randint(low, high + 1, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").double()


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,octaves", [(torch.bfloat16, 0), (torch.bfloat16, 4), (torch.bfloat16, 14), (torch.bfloat16, 40), (torch.float16, 0),
                                           (torch.float16, 4), (torch.float16, 11), (torch.float16, 14)], ids=str)
def test_large_scores(tde, call, dim, dtype, octaves):
    """Queries and keys of a few bits times 2^octaves: the scores are exact in fp32, whatever their size, and so is the largest one's weight."""
    new, lens, heads, kv_heads = CALLS[call]
    batch = Batch(new, lens, page_size=16, seed=1)
    q = whole((batch.tokens, heads, dim), -3, 3, 2) * 2.0 ** octaves
    keys = [whole((n, kv_heads, dim), -3, 3, 3 + b) * 2.0 ** octaves for b, n in enumerate(lens)]
    values = [whole((n, kv_heads, dim), -200, 200, 1000 + b) / 64 for b, n in enumerate(lens)]
    scale, starts = 2.0 ** -6, batch.starts.tolist()

    def scores(b, head):
        return q[starts[b]:starts[b + 1], head] @ keys[b][:, head * kv_heads // heads].t().contiguous() * scale

    k, v = caches(batch, kv_heads, dim, dtype, keys, values)
    got = tde.paged_attention(q.to(dtype), k, v, *batch.on("cuda"), scale)
    assert_close(got, *softmax_of(batch, scores, lambda b, h: values[b][:, h], heads, kv_heads, dim, dtype))


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("offset", [0, 600, 3000, 1 << 15, -3000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_scores_with_a_common_offset(tde, call, offset, dtype):
    """Scores that rise by a quarter every 16 keys, all far from zero: maxima move and parts are joined there."""
    new, lens, heads, kv_heads = CALLS[call]
    batch, dim = Batch(new, lens, page_size=24, seed=4), 64
    q = whole((batch.tokens, heads, dim), -1, 1, 5)
    q[..., :2] = 32.0
    keys = [whole((n, kv_heads, dim), -1, 1, 6 + b) for b, n in enumerate(lens)]
    for x in keys:
        x[..., 0] = offset / 32.0 * 4
        x[..., 1] = (torch.arange(x.size(0), device="cuda") // 16)[:, None] / 32.0
    values = [whole((n, kv_heads, dim), -200, 200, 1000 + b) / 64 for b, n in enumerate(lens)]
    scale, starts = 0.25, batch.starts.tolist()
    k, v = caches(batch, kv_heads, dim, dtype, keys, values)
    keys = [x.to(dtype).double() for x in keys]

    def scores(b, head):
        return q[starts[b]:starts[b + 1], head] @ keys[b][:, head * kv_heads // heads].t().contiguous() * scale

    got = tde.paged_attention(q.to(dtype), k, v, *batch.on("cuda"), scale)
    assert_close(got, *softmax_of(batch, scores, lambda b, h: values[b][:, h], heads, kv_heads, dim, dtype))


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("nats", [10.0, 17.375, 21.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_a_key_that_takes_nearly_all_weight(tde, call, nats, dtype):
    """One key far above all others, whose value is zero: what is left is the sum of the others' small weights."""
    new, lens, heads, kv_heads = CALLS[call]
    new, lens = ([1, 1], [20000, 130]) if call == "decode" else (new, lens)
    batch, dim = Batch(new, lens, page_size=16, seed=7), 64
    q = torch.zeros((batch.tokens, heads, dim), dtype=torch.float64, device="cuda")
    q[..., 0] = 1.0
    keys = [whole((n, kv_heads, dim), -5, 5, 8 + b) for b, n in enumerate(lens)]
    values = [1.0 + whole((n, kv_heads, dim), 0, 100, 1000 + b) / 128 for b, n in enumerate(lens)]
    for b, x in enumerate(keys):
        x[..., 0] = whole(x.shape[:2], -8, 8, 2000 + b) / 64
        at = x.size(0) // 3 if b % 2 else 0
        x[at, :, 0], values[b][at] = nats * 1.0, 0.0
    starts = batch.starts.tolist()
    k, v = caches(batch, kv_heads, dim, dtype, keys, values)

    def scores(b, head):
        return q[starts[b]:starts[b + 1], head] @ keys[b][:, head * kv_heads // heads].t().contiguous()

    got = tde.paged_attention(q.to(dtype), k, v, *batch.on("cuda"), 1.0)
    assert_close(got, *softmax_of(batch, scores, lambda b, h: values[b][:, h], heads, kv_heads, dim, dtype))


@pytest.mark.parametrize("call", ["decode", "decode whole"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_decode_rows_are_off_by_their_own_rounding(tde, call, dim, dtype):
    """With 16 rows a tile weights are two numbers of T, each within a step: a step of a step of a weight is lost at most."""
    new, lens, heads, kv_heads = CALLS[call]
    batch = Batch(new, lens, page_size=16, seed=11)
    q = whole((batch.tokens, heads, dim), -3, 3, 12)
    keys = [whole((n, kv_heads, dim), -3, 3, 13 + b) for b, n in enumerate(lens)]
    values = [whole((n, kv_heads, dim), -200, 200, 1000 + b) / 64 for b, n in enumerate(lens)]
    scale, starts = 2.0 ** -5, batch.starts.tolist()
    k, v = caches(batch, kv_heads, dim, dtype, keys, values)

    def scores(b, head):
        return q[starts[b]:starts[b + 1], head] @ keys[b][:, head * kv_heads // heads].t().contiguous() * scale

    got = tde.paged_attention(q.to(dtype), k, v, *batch.on("cuda"), scale)
    values = [x.to(dtype).double() for x in values]
    assert_close(got, *softmax_of(batch, scores, lambda b, h: values[b][:, h], heads, kv_heads, dim, dtype, torch.finfo(dtype).eps ** 2))
