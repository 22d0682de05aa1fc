"""qk_norm_rope and append_kv against their definitions in doubles: head lengths, rotations, strides, positions, pages."""
import pytest
import torch

from block_reference import Batch, append, assert_close, norm_rope

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def table(positions, rot, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand((positions, rot // 2), generator=g, dtype=torch.float64) * 6.3
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def rows_at(cos_sin, positions):
    """The table's rows; NaN for positions outside."""
    rows = torch.full((len(positions), cos_sin.size(1)), float("nan"))
    for i, p in enumerate(positions):
        if 0 <= p < cos_sin.size(0):
            rows[i] = cos_sin[p]
    return rows


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot", [
    (1, 1, 1, 1, 0), (1, 1, 1, 2, 2), (3, 2, 1, 6, 4), (2, 3, 1, 7, 6), (5, 4, 2, 8, 8), (7, 3, 3, 16, 16), (4, 5, 1, 20, 12), (3, 2, 2, 33, 20), (9, 8, 1, 64, 64),
    (2, 6, 3, 64, 32), (3, 5, 5, 80, 80), (3, 10, 2, 80, 40), (4, 4, 4, 96, 48), (130, 8, 1, 128, 128), (3, 32, 8, 128, 64), (6, 4, 1, 192, 192),
    (5, 4, 2, 256, 256), (3, 2, 1, 256, 128), (2, 1, 1, 512, 256), (2, 2, 1, 1000, 500), (1, 1, 1, 1024, 1024), (700, 12, 4, 128, 128), (2100, 20, 4, 64, 64),
])
def test_norm_rope(tde, tokens, heads, kv_heads, dim, rot, interleaved, dtype):
    seed = tokens + heads + dim
    qkv = randn((tokens, heads + 2 * kv_heads, dim), dtype, seed)
    qg, kg = randn((dim,), dtype, seed + 1), randn((dim,), dtype, seed + 2)
    cs = table(50, rot, seed)
    pos = torch.randint(0, 50, (tokens,), generator=torch.Generator().manual_seed(seed))
    dev = qkv.cuda()
    eps = 1e-5
    for positions in (pos.cuda(), pos.to(torch.int32).cuda()):
        q, k = tde.qk_norm_rope(dev[:, :heads], dev[:, heads:heads + kv_heads], qg.cuda(), kg.cuda(), eps, positions, cs.cuda(), interleaved)
        assert q.is_contiguous() and k.is_contiguous()
        rows = rows_at(cs, pos.tolist())
        assert_close(q, *norm_rope(qkv[:, :heads], qg, eps, rows, interleaved, dtype), "q")
        assert_close(k, *norm_rope(qkv[:, heads:heads + kv_heads], kg, eps, rows, interleaved, dtype), "k")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (20, 12)])
def test_strides_positions_outside_and_values_that_are_not_finite(tde, dim, rot, interleaved):
    tokens, heads, kv_heads, dtype = 11, 4, 2, torch.bfloat16
    q = randn((heads, tokens, dim), dtype, 1)
    k = randn((tokens, kv_heads, dim + 3), dtype, 2)
    q[1, 3, 5], q[2, 4, 0], k[5, 1, dim - 1] = float("nan"), float("inf"), float("-inf")
    q[0, 6], k[7, 0] = 0.0, 0.0
    pos = torch.tensor([0, 1, 2, 9, 10, -1, 3, 4, 1 << 40, 5, 6])
    cs, qg, kg = table(10, rot), randn((dim,), dtype, 3), randn((dim,), dtype, 4)
    big = torch.zeros(10, rot + 5)
    big[:, :rot] = cs
    out = tde.qk_norm_rope(q.cuda().transpose(0, 1), k.cuda()[..., :dim], qg.cuda(), kg.cuda(), 1e-6, pos.cuda(), big.cuda()[:, :rot], interleaved)
    rows = rows_at(cs, pos.tolist())
    for got, x, gamma in ((out[0], q.transpose(0, 1), qg), (out[1], k[..., :dim], kg)):
        want, bound = norm_rope(x, gamma, 1e-6, rows, interleaved, dtype)
        assert_close(got, want, bound)


def test_other_streams_and_graphs(tde):
    tokens, heads, kv_heads, dim = 24, 8, 2, 128
    qkv = randn((tokens, heads + kv_heads, dim), torch.bfloat16, 5).cuda()
    g, cs, pos = torch.ones(dim, dtype=torch.bfloat16, device="cuda"), table(64, dim).cuda(), torch.arange(tokens, device="cuda")
    args = (qkv[:, :heads], qkv[:, heads:], g, g, 1e-6, pos, cs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tde.qk_norm_rope(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tde.qk_norm_rope(*args)
    for replay in range(3):
        qkv.copy_(randn(qkv.shape, torch.bfloat16, 60 + replay))
        pos.add_(1)
        want = tde.qk_norm_rope(*args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def caches_of(kind, batch, kv_heads, dim, dtype, seed):
    """Caches [pages, page_size, kv_heads, dim] in several layouts."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def make(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    if kind == "plain":
        return make(batch.pages, batch.page, kv_heads, dim), make(batch.pages, batch.page, kv_heads, dim)
    if kind == "heads first":
        return (make(batch.pages, kv_heads, batch.page, dim).transpose(1, 2), make(kv_heads, batch.pages, batch.page, dim).permute(1, 2, 0, 3))
    both = make(batch.pages, 2, batch.page, kv_heads, dim + 8)   # keys and values side by side, room behind each row
    return both[:, 0, ..., :dim], both[:, 1, ..., :dim]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["plain", "heads first", "together"])
@pytest.mark.parametrize("dim,rot,heads,kv_heads,page,norm,interleaved", [
    (128, 128, 8, 1, 16, True, False), (128, 64, 6, 2, 64, False, True), (80, 80, 5, 5, 3, True, False), (80, 40, 4, 2, 24, True, False),
    (20, 12, 3, 1, 1, True, True), (64, 0, 0, 2, 8, False, False), (256, 256, 4, 4, 7, True, False), (64, 64, 16, 8, 16, True, True),
])
def test_append(tde, kind, dim, rot, heads, kv_heads, page, norm, interleaved, dtype):
    # sequences without new rows, without keys, with fewer keys than rows, with a page that does not exist, beyond the table
    batch = Batch(new=[3, 0, 1, 5, 2, 1, 4], lens=[10, 7, 1, 2, 40, 33, 4], page_size=page, pad=3, seed=dim)
    batch.table[4, 39 // page] = batch.pages + 5          # sequence 4's last row
    batch.table[6, 0] = -1                                # sequence 6: its first page
    batch.kv_lens[5] = 10 ** 6                            # far beyond the table's row
    batch.lens[5] = 10 ** 6
    tokens = batch.tokens
    qkv = randn((tokens, heads + 2 * kv_heads, dim), dtype, 7)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    qg, kg = (randn((dim,), dtype, 8), randn((dim,), dtype, 9)) if norm else (None, None)
    cs = table(50, rot) if rot else None
    k_cache, v_cache = caches_of(kind, batch, kv_heads, dim, dtype, 10)
    before = k_cache.cpu().clone(), v_cache.cpu().clone()
    dev, gpu = qkv.cuda(), lambda x: None if x is None else x.cuda()
    got = tde.append_kv(dev[:, heads:heads + kv_heads], dev[:, heads + kv_heads:], k_cache, v_cache, *batch.on("cuda"), cos_sin=gpu(cs),
                        q=dev[:, :heads] if heads else None, q_gamma=gpu(qg) if heads else None, k_gamma=gpu(kg), eps=1e-6, interleaved=interleaved)
    positions = [-1] * tokens
    for t, b, p in batch.rows():
        positions[t] = p
    rows = rows_at(cs, positions) if rot else None
    k_want, k_bound = norm_rope(k, kg, 1e-6, rows, interleaved, dtype)
    keys, values, written, token_of = append(batch, k_want, v, *before)
    bound = torch.zeros_like(keys)
    bound[written] = k_bound[token_of[written]]
    assert_close(k_cache, keys, bound, "keys")
    assert torch.equal(v_cache.cpu(), values)
    if not heads:
        assert got is None
        return
    want, bound = norm_rope(q, qg, 1e-6, rows, interleaved, dtype)
    none = torch.tensor([p < 0 for p in positions])
    want[none], bound[none] = 0.0, 0.0
    assert_close(got, want, bound, "queries")


@pytest.mark.parametrize("seqs", [1, 63, 64, 65, 130, 4097])
def test_append_finds_every_sequence(tde, seqs):
    g = torch.Generator().manual_seed(seqs)
    new = torch.randint(0, 3, (seqs,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 5, (seqs,), generator=g))]
    batch = Batch(new, lens, page_size=4, pad=2, seed=1)
    k = randn((batch.tokens, 1, 16), torch.float32, 2)
    v = randn((batch.tokens, 1, 16), torch.float32, 3)
    k_cache, v_cache = caches_of("plain", batch, 1, 16, torch.float32, 4)
    before = k_cache.cpu().clone(), v_cache.cpu().clone()
    tde.append_kv(k.cuda(), v.cuda(), k_cache, v_cache, *batch.on("cuda"))
    keys, values, _, _ = append(batch, k.double(), v, *before)
    assert torch.equal(k_cache.cpu().double(), keys) and torch.equal(v_cache.cpu(), values)


def test_append_positions_of_its_own_and_empty_calls(tde):
    batch = Batch([2, 3], [2, 9], page_size=4)
    k, v = randn((5, 2, 64), torch.bfloat16, 1), randn((5, 2, 64), torch.bfloat16, 2)
    cs, pos = table(200, 64), torch.tensor([7, 199, 0, 3, 100], dtype=torch.int32)
    k_cache, v_cache = caches_of("plain", batch, 2, 64, torch.bfloat16, 3)
    before = k_cache.cpu().clone(), v_cache.cpu().clone()
    tde.append_kv(k.cuda(), v.cuda(), k_cache, v_cache, *batch.on("cuda"), cos_sin=cs.cuda(), positions=pos.cuda())
    want, k_bound = norm_rope(k, None, 0.0, rows_at(cs, pos.tolist()), False, torch.bfloat16)
    keys, values, written, token_of = append(batch, want, v, *before)
    bound = torch.zeros_like(keys)
    bound[written] = k_bound[token_of[written]]
    assert_close(k_cache, keys, bound)
    assert torch.equal(v_cache.cpu(), values)
    # no rows; rows and no sequences
    before = k_cache.clone()
    none = Batch([], [], page_size=4)
    empty = torch.zeros((0, 1), dtype=torch.int32, device="cuda")
    for rows in (0, 3):
        q = tde.append_kv(k[:rows].cuda(), v[:rows].cuda(), k_cache, v_cache, empty, none.starts.cuda(), none.kv_lens.cuda(), q=k[:rows].cuda())
        assert q.shape == (rows, 2, 64) and not q.any()
    assert torch.equal(k_cache, before)
