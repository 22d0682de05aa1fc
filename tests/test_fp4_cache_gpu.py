"""append_kv_fp4 and unpack_fp4 against their definitions in doubles: every code of the caches, scales, queries, what is left alone."""
import math

import pytest
import torch

from block_reference import Batch, assert_close, norm_rope, half_step, smallest
from fp4_reference import decode, encode, most_exponent, random_cache

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def as_values(codes, scales, dtype):
    """What unpacking gives, rounded once."""
    return decode(codes, scales).to(dtype)


def same(got, want):
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0, 1.0, -1.0), want.nan_to_num(0.0, 1.0, -1.0)) and torch.equal(got.isinf(), want.isinf())


# ---- unpack_fp4 ----

@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_every_code_with_every_scale(tde, dtype):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(256, 16, 16)      # rows of 32 channels
    scales = torch.arange(256, dtype=torch.uint8)[:, None, None].expand(256, 16, 1)
    got = tde.unpack_fp4(codes.cuda(), scales.cuda(), dtype).cpu()
    want = as_values(codes, scales, dtype)
    assert got.dtype == dtype and got.shape == want.shape and same(got, want)
    assert torch.equal(torch.signbit(got[:255]), torch.signbit(want[:255]))            # zeros keep their sign
    assert got.isnan().sum() == 16 * 32


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 5, 2), (7, 16, 3), (300, 24, 1)])
def test_unpack_sizes_and_orders(tde, dim, shape):
    codes, scales = random_cache(shape, dim, dim)
    for dtype in DTYPES:
        assert torch.equal(tde.unpack_fp4(codes.cuda(), scales.cuda(), dtype).cpu(), as_values(codes, scales, dtype))
    # heads in front of slots, pages last, rows of a wider tensor, dimensions of two kinds, a dimension that is repeated
    want = as_values(codes, scales, torch.bfloat16)
    for order in ((0, 2, 1, 3), (2, 1, 0, 3), (1, 0, 2, 3)):
        back = [order.index(i) for i in range(4)]
        c, s = (x.permute(order).contiguous().cuda().permute(back) for x in (codes, scales))
        assert torch.equal(tde.unpack_fp4(c, s).cpu(), want)
        assert torch.equal(tde.unpack_fp4(c, scales.cuda()).cpu(), want)
    wide = torch.zeros((*shape, dim // 2 + 5), dtype=torch.uint8, device="cuda")
    wide[..., 3:3 + dim // 2] = codes.cuda()
    assert torch.equal(tde.unpack_fp4(wide[..., 3:3 + dim // 2], scales.cuda()).cpu(), want)
    assert torch.equal(tde.unpack_fp4(codes[:1].expand(4, *shape[1:], dim // 2).cuda(), scales[:1].cuda().expand(4, *shape[1:], dim // 32)).cpu(),
                       want[:1].expand(4, *shape[1:], dim))


def test_unpack_ranks(tde):
    codes, scales = random_cache((2, 3, 4, 5), 64, 1)
    assert torch.equal(tde.unpack_fp4(codes.cuda(), scales.cuda()).cpu(), as_values(codes, scales, torch.bfloat16))
    assert torch.equal(tde.unpack_fp4(codes[0, 0, 0, 0].cuda(), scales[0, 0, 0, 0].cuda()).cpu(), as_values(codes, scales, torch.bfloat16)[0, 0, 0, 0])
    assert tde.unpack_fp4(codes[:, :0].cuda(), scales[:, :0].cuda()).shape == (2, 0, 4, 5, 64)
    apart = codes.cuda().permute(3, 2, 1, 0, 4)
    with pytest.raises(RuntimeError, match="three dimensions"):
        tde.unpack_fp4(apart, scales.cuda().permute(3, 2, 1, 0, 4))


def test_unpack_refusals(tde):
    codes, scales = (x.cuda() for x in random_cache((2, 3), 64, 1))
    for c, s, kw, match in ((codes.cpu(), scales, {}, "GPU"), (codes, scales.cpu(), {}, "GPU"), (codes.int(), scales, {}, "uint8"), (codes, scales.int(), {}, "scales"),
                            (codes[..., :8], scales[..., :1], {}, "channels"), (codes, scales[..., :1], {}, "scales"), (codes, scales[:1], {}, "scales"),
                            (codes, scales, dict(out_dtype=torch.float64), "out_dtype"), (codes.repeat(1, 1, 9), scales.repeat(1, 1, 9), {}, "channels"),
                            (torch.stack([codes, codes], -1)[..., 0], scales, {}, "contiguous")):
        with pytest.raises(RuntimeError, match=match):
            tde.unpack_fp4(c, s, **kw)


# ---- append_kv_fp4 ----

def caches(batch, kv_heads, dim, seed, heads_first=False):
    shape = (batch.pages, kv_heads, batch.page) if heads_first else (batch.pages, batch.page, kv_heads)
    made = [x for i in (0, 1) for x in random_cache(shape, dim, seed + i)]
    return [x.transpose(1, 2) for x in made] if heads_first else made


def cos_sin(positions, rot):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    return torch.cat([a.cos(), a.sin()], 1).float()


def run(tde, batch, heads, kv_heads, dim, dtype, rot, interleaved, norm, seed=0, heads_first=False, positions=None, queries=True, spread=1.0, table_rows=None):
    g_q, g_k = ((randn((dim,), torch.float32, seed + i) * 0.2 + 1).to(dtype) if norm else None for i in (7, 8))
    q, k, v = (randn((batch.tokens, n, dim), dtype, seed + i, spread) for i, n in ((1, heads), (2, kv_heads), (3, kv_heads)))
    held = caches(batch, kv_heads, dim, seed + 20, heads_first)
    here = [x.cuda() for x in held]
    here = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in here] if heads_first else here
    longest = max([n for n in batch.lens] + [1])
    table = cos_sin(longest if table_rows is None else table_rows, rot) if rot else None
    at = torch.full((batch.tokens,), -1, dtype=torch.long)
    for t, _, p in batch.rows():
        at[t] = p
    where = at if positions is None else positions
    rows = None
    if rot:
        rows = torch.full((batch.tokens, rot), math.nan)
        known = (where >= 0) & (where < table.size(0))
        rows[known] = table[where[known]]
    kw = dict(cos_sin=None if table is None else table.cuda(), positions=None if positions is None else positions.cuda(), k_gamma=None if g_k is None else g_k.cuda(),
              eps=1e-6, interleaved=interleaved)
    if queries:
        kw.update(q=q.cuda(), q_gamma=None if g_q is None else g_q.cuda())
    got = tde.append_kv_fp4(k.cuda(), v.cuda(), *here, *batch.on("cuda"), **kw)
    if queries:
        want, bound = norm_rope(q, g_q, 1e-6, rows, interleaved, dtype)
        # A rotation adds two products, and one is rounded to fp32 before: a half step of its own among subnormal numbers, 2^-150, which norm_rope's bound,
        # relative but for the last rounding's half step, leaves out.  (Heads of 1e-38 in fp32 were off by up to 2^-149 in place of 2^-150.)
        bound = bound + smallest(torch.float32) * bool(rot)
        want[at < 0], bound[at < 0] = 0.0, 0.0
        assert_close(got, want, bound, "queries")
    else:
        assert got is None
    k_want, _ = norm_rope(k, g_k, 1e-6, rows, interleaved, dtype)
    k_new, v_new = encode(k_want, most_exponent(dtype)), encode(v.double(), most_exponent(dtype))
    for t, b, p in batch.rows():
        page = batch.page_of(b, p) if p >= 0 else None
        if page is not None:
            for i in (0, 1):
                held[i][page, p % batch.page], held[2 + i][page, p % batch.page] = k_new[i][t], v_new[i][t]
    for name, g, w in zip(("k_cache", "k_scales", "v_cache", "v_scales"), here, held):
        assert torch.equal(g.cpu(), w), name
    return here


RAGGED = dict(new=[5, 0, 17, 1, 3, 2, 40, 0], lens=[5, 9, 40, 513, 2, 0, 130, 0])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,page,rot,interleaved,norm", [
    (1, 1, 32, 1, 32, False, True), (8, 1, 128, 64, 128, False, True), (6, 2, 64, 3, 64, True, False), (15, 5, 96, 24, 96, False, True), (4, 4, 160, 16, 80, True, True),
    (12, 4, 192, 16, 96, False, False), (8, 2, 256, 32, 256, False, True), (7, 1, 224, 16, 0, False, True), (5, 5, 128, 8, 64, False, False), (3, 3, 64, 16, 20, False, True),
    (3, 3, 64, 16, 20, True, True), (2, 1, 96, 7, 2, False, False), (33, 11, 32, 5, 12, True, False),
])
def test_append(tde, heads, kv_heads, dim, page, rot, interleaved, norm, dtype):
    run(tde, Batch([1, 1, 1, 1, 1], [1, 2, 31, 64, 300], page, seed=1), heads, kv_heads, dim, dtype, rot, interleaved, norm, seed=dim)
    run(tde, Batch(page_size=page, pad=9, seed=2, **RAGGED), heads, kv_heads, dim, dtype, rot, interleaved, norm, seed=dim + 1, heads_first=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_large_and_small_numbers(tde, dtype):
    for spread in (1e-30, 1e-6, 1e-3, 3e4) if dtype == torch.float16 else (1e-38, 1e-30, 1e-3, 1e4, 1e37):
        run(tde, Batch([3, 9], [3, 20], 4, seed=3), 2, 1, 64, dtype, 0, False, False, spread=spread)
        run(tde, Batch([3, 9], [3, 20], 4, seed=3), 2, 1, 64, dtype, 64, False, False, spread=spread if spread < 1e4 else 1e3)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_borders_of_codes_and_scales(tde, dtype):
    """Numbers on the borders of two codes and next to them, blocks whose largest number is on the border of two scales and next to it."""
    steps = torch.tensor([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 6.5, 6.9375, 7, 7.0625, 7.9375], dtype=torch.float32)
    near = torch.cat([steps, steps * (1 + torch.finfo(dtype).eps), steps * (1 - torch.finfo(dtype).eps)]).to(dtype)
    g = torch.Generator().manual_seed(1)
    rows = near[torch.randint(0, len(near), (200, 1, 64), generator=g)] * torch.where(torch.rand((200, 1, 64), generator=g) < 0.5, -1.0, 1.0).to(dtype)
    top = near[torch.randint(len(near) // 2, len(near), (200, 1), generator=g)]
    rows[..., 5], rows[..., 40] = top, -top
    rows = (rows.float() * 2.0 ** torch.randint(-10, 11, (200, 1, 1), generator=g)).to(dtype)
    batch = Batch([200], [200], 16, seed=4)
    here = [x.cuda() for x in caches(batch, 1, 64, 5)]
    tde.append_kv_fp4(rows.cuda(), rows.cuda(), *here, *batch.on("cuda"))
    codes, scales = encode(rows.double(), most_exponent(dtype))
    for i in range(200):
        page, slot = batch.page_of(0, i), i % 16
        for c, s in ((here[0], here[1]), (here[2], here[3])):
            assert torch.equal(c[page, slot].cpu(), codes[i]) and torch.equal(s[page, slot].cpu(), scales[i]), i
    # a number is off by half a step of its code: a sixth of it or of the block's largest, nothing is cut off by more
    off = (decode(codes, scales) - rows.double()).abs()
    assert bool((off <= rows.double().abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1) / 6).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_zeros_infinities_and_nan(tde, dtype):
    batch = Batch([4], [4], 4, seed=5)
    k = randn((4, 2, 96), dtype, 1)
    k[0, 0, :32] = 0.0
    k[0, 0, 33] = -0.0
    k[1, 1, 40], k[2, 0, 95], k[3, 0, 0], k[3, 0, 64] = math.inf, -math.inf, math.nan, torch.finfo(dtype).max
    here = [x.cuda() for x in caches(batch, 2, 96, 6)]
    tde.append_kv_fp4(k.cuda(), k.cuda(), *here, *batch.on("cuda"))
    codes, scales = encode(k.double(), most_exponent(dtype))
    for t in range(4):
        page = batch.page_of(0, t)
        for c, s in ((here[0], here[1]), (here[2], here[3])):
            assert torch.equal(c[page, t].cpu(), codes[t]) and torch.equal(s[page, t].cpu(), scales[t])
    assert (scales == 255).sum() == 3
    values = tde.unpack_fp4(here[0], here[1], dtype).cpu()[batch.page_of(0, 0)]
    assert values[3, 0, :32].isnan().all() and torch.isfinite(values[3, 0, 64:]).all()


def test_positions(tde):
    batch = Batch(page_size=16, pad=3, seed=7, **RAGGED)
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.int64, torch.int32):
        positions = torch.randint(-2, 60, (batch.tokens,), generator=g)
        run(tde, batch, 4, 2, 64, torch.bfloat16, 64, False, True, positions=positions.to(dtype), table_rows=55)   # some lie outside: NaN there
    run(tde, batch, 4, 2, 128, torch.float16, 128, True, False, table_rows=100)


def test_without_queries_and_pages(tde):
    batch = Batch(page_size=16, pad=3, seed=8, **RAGGED)
    run(tde, batch, 4, 2, 64, torch.bfloat16, 64, False, True, queries=False)
    batch.table[2, 1], batch.table[3, 5], batch.table[6, 0] = -1, batch.pages, 0x7fffffff   # keys without a page change nothing
    run(tde, batch, 4, 2, 64, torch.bfloat16, 64, False, True)
    run(tde, Batch(page_size=16, seed=9, table_pages=3, **RAGGED), 4, 2, 64, torch.bfloat16, 64, False, True)
    run(tde, Batch([0, 0], [4, 0], 4, pad=5), 2, 1, 32, torch.bfloat16, 32, False, False)     # rows of no sequence alone
    run(tde, Batch([], [], 4, pad=5), 2, 1, 32, torch.bfloat16, 0, False, False)


def test_many_sequences_and_rows(tde):
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 5, (300,), generator=g).tolist()
    run(tde, Batch(new, [n + int(x) for n, x in zip(new, torch.randint(0, 40, (300,), generator=g))], 8, seed=2, pad=5), 3, 3, 32, torch.bfloat16, 32, False, True)
    run(tde, Batch([700, 900], [700, 1500], 64, seed=3), 4, 2, 64, torch.bfloat16, 64, False, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,rot,interleaved,norm,queries", [
    (8, 2, 128, 64, True, False, True), (15, 5, 96, 96, False, True, True), (7, 1, 256, 128, True, True, True), (3, 3, 64, 0, False, True, True),
    (1, 9, 32, 16, False, True, False), (33, 1, 64, 64, False, False, True), (2, 1, 96, 2, False, True, True)])
def test_many_rows(tde, heads, kv_heads, dim, rot, interleaved, norm, queries, dtype):
    run(tde, Batch([700, 1, 350], [700, 90, 500], 24, seed=4, pad=6), heads, kv_heads, dim, dtype, rot, interleaved, norm, seed=dim, queries=queries,
        heads_first=True)


def test_rows_of_one_projection_into_one_tensor(tde):
    """q, k and v as columns of one tensor, codes and scales as ranges of one allocation whose rows begin anywhere."""
    batch = Batch([3, 8], [9, 8], 4, seed=9)
    qkv = randn((batch.tokens, 2 + 2 * 2, 64), torch.bfloat16, 3).cuda()
    all_bytes = torch.zeros((batch.pages, 4, 2, 2 * (32 + 2) + 3), dtype=torch.uint8, device="cuda")
    k_cache, k_scales, v_cache, v_scales = all_bytes[..., 1:33], all_bytes[..., 33:35], all_bytes[..., 36:68], all_bytes[..., 68:70]
    tde.append_kv_fp4(qkv[:, 2:4], qkv[:, 4:], k_cache, k_scales, v_cache, v_scales, *batch.on("cuda"))
    for c, s, x in ((k_cache, k_scales, qkv[:, 2:4]), (v_cache, v_scales, qkv[:, 4:])):
        codes, scales = encode(x.cpu().double(), 125)
        for t, b, p in batch.rows():
            page = batch.page_of(b, p)
            assert torch.equal(c[page, p % 4].cpu(), codes[t]) and torch.equal(s[page, p % 4].cpu(), scales[t])
    assert int(all_bytes[..., 0].sum()) == int(all_bytes[..., 35].sum()) == int(all_bytes[..., 70].sum()) == 0


def test_a_captured_append_follows_its_arrays(tde):
    batch = Batch([4, 4], [4, 9], 4, seed=10, extra_pages=8)
    k, v = randn((8, 1, 64), torch.bfloat16, 1).cuda(), randn((8, 1, 64), torch.bfloat16, 2).cuda()
    here, eager = ([x.cuda() for x in caches(batch, 1, 64, 3)] for _ in (0, 1))
    table, starts, lens = batch.on("cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        tde.append_kv_fp4(k, v, *here, table, starts, lens)
    for i in range(3):
        k.copy_(randn((8, 1, 64), torch.bfloat16, 10 + i))
        lens.add_(-1)
        graph.replay()
        tde.append_kv_fp4(k, v, *eager, table, starts, lens)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(here, eager))


def test_append_refusals(tde):
    batch = Batch([3], [5], 4, seed=11)
    k, v, q = (randn((3, n, 64), torch.bfloat16, n).cuda() for n in (2, 2, 4))
    good = dict(zip(("k_cache", "k_scales", "v_cache", "v_scales"), (x.cuda() for x in caches(batch, 2, 64, 1))))

    def call(k=k, v=v, q=None, **kw):
        c = dict(good)
        rest = {n: kw.pop(n) for n in ("q_gamma", "k_gamma", "cos_sin", "positions") if n in kw}
        c.update(kw)
        tde.append_kv_fp4(k, v, c["k_cache"], c["k_scales"], c["v_cache"], c["v_scales"], *batch.on("cuda"), q=q, **rest)

    versions = [good[n]._version for n in good]
    call()
    assert all(good[n]._version > b for n, b in zip(good, versions))
    narrow = randn((3, 2, 48), torch.bfloat16, 1).cuda()
    shared = torch.zeros((batch.pages, 4, 2, 64), dtype=torch.uint8, device="cuda")
    in_k = k.view(torch.uint8).view(-1)[:batch.pages * 4 * 2 * 2].view(batch.pages, 4, 2, 2)
    for kw, match in ((dict(k=narrow, v=narrow), "steps of 32"), (dict(k=randn((3, 2, 288), torch.bfloat16, 1).cuda()), "steps of 32"), (dict(v=v[:, :1]), "shape"),
                      (dict(k_cache=good["k_cache"].int()), "uint8"), (dict(k_cache=good["k_cache"][..., :16]), "k_cache must be"), (dict(v_cache=good["v_cache"][:, :, :1]), "v_cache must be"),
                      (dict(k_scales=good["k_scales"][..., :1]), "k_scales must be"), (dict(v_scales=good["v_scales"][:-1]), "differs"), (dict(v_scales=good["v_scales"].cpu()), "GPU"),
                      (dict(k_scales=good["k_scales"][:, :3]), "differs"), (dict(v_cache=good["v_cache"][:-1], v_scales=good["v_scales"][:-1]), "differ in pages"),
                      (dict(k_cache=shared[..., :32], v_cache=shared[..., 31:63]), "overlaps v_cache"), (dict(k_cache=good["k_cache"][:1].expand(batch.pages, -1, -1, -1)), "overlap"),
                      (dict(v_scales=good["k_scales"]), "overlaps"), (dict(k_scales=in_k), "overlaps k"),
                      (dict(q_gamma=k[0, 0]), "without q"), (dict(q=q[:, :, :32]), "q and k differ"), (dict(q=q.float()), "dtype"), (dict(k=k.double(), v=v.double()), "dtype"),
                      (dict(cos_sin=torch.zeros((9, 66), device="cuda")), "rot_dim"), (dict(positions=torch.zeros(2, dtype=torch.int64, device="cuda")), "positions")):
        with pytest.raises(RuntimeError, match=match):
            call(**kw)


def test_fp4_cache(tde):
    parts = tde.fp4_cache(3, 16, 2, 96)
    assert [tuple(p.shape) for p in parts] == [(3, 16, 2, 48), (3, 16, 2, 3)] * 2 and all(p.is_cuda and p.dtype == torch.uint8 for p in parts)
    assert parts[0].stride() == (16 * 2 * 48, 48, 16 * 48, 1)
    with pytest.raises(RuntimeError, match="steps of 32"):
        tde.fp4_cache(3, 16, 2, 40)
