"""The attention block as a rank runs it: fused norm with int8 codes -> int8_linear -> append_kv (norm, rotation) -> paged_attention ->
the next int8_linear, over a prefill chunk and decode steps; every operator against its definition on the inputs that it was given.
And what the operators refuse."""
import pytest
import torch

from block_reference import Batch, assert_close, append, attention, int8_linear, norm_rope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def table(positions, rot):
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def test_prefill_and_decode_steps(tde):
    torch.manual_seed(3)
    hidden, heads, kv_heads, dim, page, ranks, dtype, eps = 512, 8, 2, 64, 16, 4, torch.bfloat16, 1e-6
    width = (heads + 2 * kv_heads) * dim
    lens, steps = [37, 5, 80], [None, 1, 1, 1]
    final = [n + 3 for n in lens]
    whole = Batch(final, final, page, seed=4)     # the table's pages for the whole run
    k_cache = torch.randn(whole.pages, page, kv_heads, dim).to(dtype).cuda()
    v_cache = torch.randn(whole.pages, page, kv_heads, dim).to(dtype).cuda()
    w_qkv = torch.randint(-127, 128, (width, hidden)).to(torch.int8)
    w_out = torch.randint(-127, 128, (hidden, heads * dim)).to(torch.int8)
    u_qkv, u_out = torch.rand(width) * 1e-4 + 1e-4, torch.rand(hidden) * 1e-4 + 1e-4
    gamma, qg, kg = (torch.rand(n) + 0.5 for n in (hidden, dim, dim))
    gamma, qg, kg = gamma.to(dtype), qg.to(dtype), kg.to(dtype)
    cs = table(200, dim)
    done = [0, 0, 0]
    for step, new in enumerate(steps):
        rows = lens if new is None else [new] * 3
        done = [d + n for d, n in zip(done, rows)]
        batch = Batch(rows, done, page, extra_pages=0)
        batch.table, batch.pages = whole.table, whole.pages
        tokens = batch.tokens
        partials = [torch.randn(tokens, hidden).to(dtype).cuda() for _ in range(ranks)]
        out = tde.reduce_rms(partials, torch.randn(tokens, hidden).to(dtype).cuda(), gamma.cuda(), eps, tde.QUANT_INT8_TOKEN)
        qkv = tde.int8_linear(out["q"], out["scale"], w_qkv.cuda(), u_qkv.cuda(), None, dtype)
        assert_close(qkv, *int8_linear(out["q"].cpu(), out["scale"].cpu(), w_qkv, u_qkv, None, dtype), "qkv %d" % step)
        q, k, v = qkv.view(tokens, -1, dim).split([heads, kv_heads, kv_heads], dim=1)
        before = k_cache.cpu().clone(), v_cache.cpu().clone()
        args = batch.on("cuda")
        turned = tde.append_kv(k, v, k_cache, v_cache, *args, cos_sin=cs.cuda(), q=q, q_gamma=qg.cuda(), k_gamma=kg.cuda(), eps=eps)
        positions = [p for _, _, p in batch.rows()]
        assert_close(turned, *norm_rope(q.cpu(), qg, eps, cs[positions], False, dtype), "queries %d" % step)
        k_want, k_bound = norm_rope(k.cpu(), kg, eps, cs[positions], False, dtype)
        keys, values, written, token_of = append(batch, k_want, v.cpu(), *before)
        bound = torch.zeros_like(keys)
        bound[written] = k_bound[token_of[written]]
        assert_close(k_cache, keys, bound, "keys %d" % step)
        assert torch.equal(v_cache.cpu(), values)
        # the same rows without a cache
        alone = tde.qk_norm_rope(q, k, qg.cuda(), kg.cuda(), eps, torch.tensor(positions).cuda(), cs.cuda())
        assert torch.equal(alone[0], turned)
        o = tde.paged_attention(turned, k_cache, v_cache, *args)
        assert_close(o, *attention(batch, turned.cpu(), k_cache.cpu(), v_cache.cpu(), dim ** -0.5), "attention %d" % step)
        codes = torch.randint(-127, 128, (tokens, heads * dim)).to(torch.int8)
        scale = o.view(tokens, -1).float().abs().amax(-1) / 127
        codes = (o.view(tokens, -1).float() / scale[:, None]).round().to(torch.int8)
        partial = tde.int8_linear(codes, scale, w_out.cuda(), u_out.cuda(), None, dtype)     # the next stage's partial
        assert_close(partial, *int8_linear(codes.cpu(), scale.cpu(), w_out, u_out, None, dtype), "partial %d" % step)


def test_decode_step_in_one_graph(tde):
    """Captured once for a fixed number of rows; replays see other lengths, tokens and rows behind the last sequence."""
    torch.manual_seed(5)
    heads, kv_heads, dim, page, seqs, dtype = 4, 1, 128, 16, 6, torch.bfloat16
    batch = Batch([1] * seqs, [600] * seqs, page, seed=6)
    k_cache = torch.randn(batch.pages, page, kv_heads, dim).to(dtype).cuda()
    v_cache = torch.randn(batch.pages, page, kv_heads, dim).to(dtype).cuda()
    codes = torch.randint(-127, 128, (seqs, 256)).to(torch.int8).cuda()
    scales, w = torch.rand(seqs).cuda() * 0.01, torch.randint(-127, 128, ((heads + 2) * dim, 256)).to(torch.int8).cuda()
    u, cs = torch.rand((heads + 2) * dim).cuda() * 1e-2, table(700, dim).cuda()
    g = torch.ones(dim, dtype=dtype).cuda()
    page_table, starts, lens = batch.on("cuda")

    def step():
        qkv = tde.int8_linear(codes, scales, w, u, None, dtype).view(seqs, -1, dim)
        q, k, v = qkv.split([heads, 1, 1], dim=1)
        q = tde.append_kv(k, v, k_cache, v_cache, page_table, starts, lens, cos_sin=cs, q=q, q_gamma=g, k_gamma=g)
        return tde.paged_attention(q, k_cache, v_cache, page_table, starts, lens)

    lens.fill_(500)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for replay, live in enumerate((6, 4, 5, 1)):
        starts.copy_(torch.clamp(torch.arange(seqs + 1), max=live))
        lens.copy_(torch.tensor([501 + 7 * replay + 3 * i if i < live else 0 for i in range(seqs)]))
        codes.copy_(torch.randint(-127, 128, codes.shape))
        saved = k_cache.clone(), v_cache.clone()
        graph.replay()
        torch.cuda.synchronize()
        got, k_after, v_after = out.clone(), k_cache.clone(), v_cache.clone()
        k_cache.copy_(saved[0])
        v_cache.copy_(saved[1])
        want = step()
        assert torch.equal(got, want) and torch.equal(k_after, k_cache) and torch.equal(v_after, v_cache)
        assert not got[live:].any()


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_under_torch_compile(tde, backend):
    """A decode step with other operators around, traced through the operators' fake kernels: outputs and changed caches as without."""
    if backend == "inductor":
        pytest.importorskip("triton")
        import torch._inductor.config as inductor_config
        inductor_config.compile_threads = 1      # compile in this process: no pool of worker processes
    from torch._dynamo.exc import BackendCompilerFailed
    torch.manual_seed(7)
    heads, dim, page, seqs, dtype = 4, 64, 16, 3, torch.bfloat16
    batch = Batch([1] * seqs, [40, 17, 1], page, seed=8)
    caches = [torch.randn(batch.pages, page, 1, dim).to(dtype).cuda() for _ in (0, 1)]
    codes, scales = torch.randint(-127, 128, (seqs, 96)).to(torch.int8).cuda(), torch.rand(seqs).cuda() * 0.01
    w, u = torch.randint(-127, 128, ((heads + 2) * dim, 96)).to(torch.int8).cuda(), torch.rand((heads + 2) * dim).cuda() * 1e-2
    g, cs = torch.ones(dim, dtype=dtype).cuda(), table(64, dim).cuda()
    page_table, starts, lens = batch.on("cuda")

    def step(codes, k_cache, v_cache, out):
        qkv = tde.int8_linear(codes, scales, w, u).view(seqs, -1, dim)
        q, k, v = qkv.split([heads, 1, 1], dim=1)
        first, _ = tde.qk_norm_rope(q, k, g, g, 1e-6, lens - 1, cs)
        tde.append_kv(k, v * 2, k_cache, v_cache, page_table, starts, lens)
        q = tde.append_kv(k, v, k_cache, v_cache, page_table, starts, lens, cos_sin=cs, q=q, q_gamma=g, k_gamma=g)
        tde.paged_attention_out(q, k_cache, v_cache, page_table, starts, lens, out)
        return tde.paged_attention(q, k_cache, v_cache, page_table, starts, lens).float() + 1, first

    results = []
    for f in (step, torch.compile(step, backend=backend, fullgraph=True)):
        k_cache, v_cache, out = caches[0].clone(), caches[1].clone(), torch.zeros((seqs, heads, dim), dtype=dtype, device="cuda")
        try:
            y, first = f(codes, k_cache, v_cache, out)
        except BackendCompilerFailed as e:   # the code generator, not this library
            pytest.skip("torch.compile backend unavailable here: %s" % str(e)[:200])
        torch.cuda.synchronize()
        results.append((y, first, k_cache, v_cache, out))
    for got, want in zip(results[1], results[0]):
        assert torch.equal(got, want)
    assert not torch.equal(results[0][2], caches[0]) and torch.equal(results[0][0], results[0][4].float() + 1)


def test_parameters_give_plain_tensors(tde):
    """A gamma that requires a gradient: the operators have none, and their outputs do not pretend to."""
    qkv = torch.randn(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    g = torch.nn.Parameter(torch.ones(64, device="cuda", dtype=torch.bfloat16))
    q, k = tde.qk_norm_rope(qkv[:, :2], qkv[:, 2:], g, g, 1e-6, torch.arange(3, device="cuda"), torch.ones(4, 64, device="cuda"))
    assert not q.requires_grad and q.grad_fn is None and not k.requires_grad


def good_linear():
    return dict(codes=torch.zeros((2, 3, 64), dtype=torch.int8, device="cuda"), scales=torch.ones((2, 3), device="cuda"),
                weight=torch.zeros((8, 64), dtype=torch.int8, device="cuda"), weight_scales=torch.ones(8, device="cuda"))


@pytest.mark.parametrize("change", [
    dict(codes=lambda t: t.to(torch.uint8)), dict(codes=lambda t: t.transpose(0, 1)), dict(codes=lambda t: t[..., ::2]), dict(scales=lambda t: t[:1]),
    dict(scales=lambda t: t.double()), dict(weight=lambda t: t.t()), dict(weight=lambda t: t[:, :32].contiguous()), dict(weight=lambda t: t.cpu()),
    dict(weight=lambda t: t.float()), dict(weight_scales=lambda t: t[:4]), dict(weight_scales=lambda t: t.half()), dict(bias=lambda t: torch.ones(7, device="cuda")),
    dict(bias=lambda t: torch.ones(8, device="cuda").half()), dict(out_dtype=lambda t: torch.float64), dict(out_dtype=lambda t: torch.int8),
    dict(codes=lambda t: torch.zeros((1, 131072), dtype=torch.int8, device="cuda"), weight=lambda t: torch.zeros((1, 131072), dtype=torch.int8, device="cuda"),
         scales=lambda t: t[0, :1], weight_scales=lambda t: t[:1]),
])
def test_int8_linear_refuses(tde, change):
    kw = good_linear()
    tde.int8_linear(**kw)
    for name, f in change.items():
        kw[name] = f(kw.get(name))
    with pytest.raises(RuntimeError):
        tde.int8_linear(**kw)


def good_heads():
    z = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    g = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    return dict(q=z, k=z[:, :2], q_gamma=g, k_gamma=g, eps=1e-6, positions=torch.zeros(3, dtype=torch.long, device="cuda"), cos_sin=torch.zeros((5, 64), device="cuda"))


@pytest.mark.parametrize("change", [
    dict(q=lambda t: t.double()), dict(q=lambda t: t.half()), dict(q=lambda t: t[:2]), dict(q=lambda t: t[..., :32]), dict(q=lambda t: t[0]), dict(q=lambda t: t.cpu()),
    dict(k=lambda t: t.transpose(1, 2)), dict(q=lambda t: torch.zeros((3, 4, 128), dtype=torch.bfloat16, device="cuda")[..., ::2]), dict(q_gamma=lambda t: t.float()),
    dict(k_gamma=lambda t: t[:32]), dict(eps=lambda t: -1.0), dict(eps=lambda t: float("nan")), dict(positions=lambda t: t[:2]), dict(positions=lambda t: t.float()),
    dict(cos_sin=lambda t: t.double()), dict(cos_sin=lambda t: t[:, :63]), dict(cos_sin=lambda t: torch.zeros((5, 66), device="cuda")), dict(cos_sin=lambda t: t.t()),
])
def test_heads_refuse(tde, change):
    kw = good_heads()
    tde.qk_norm_rope(**kw)
    for name, f in change.items():
        kw[name] = f(kw[name])
    with pytest.raises(RuntimeError):
        tde.qk_norm_rope(**kw)


def good_batch():
    z = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    return dict(k=z, v=z, k_cache=cache, v_cache=cache.clone(), page_table=torch.zeros((2, 2), dtype=torch.int32, device="cuda"),
                q_starts=torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda"), kv_lens=torch.tensor([2, 1], dtype=torch.int32, device="cuda"))


BATCHES = [
    dict(k_cache=lambda t: t.half()), dict(v_cache=lambda t: t[:, :8]), dict(v_cache=lambda t: t[:3]), dict(k_cache=lambda t: t[..., :32]), dict(k_cache=lambda t: t[0]),
    dict(k_cache=lambda t: t.transpose(2, 3)), dict(v_cache=lambda t: t.cpu()), dict(page_table=lambda t: t.long()), dict(page_table=lambda t: t.t()),
    dict(page_table=lambda t: t[0]), dict(q_starts=lambda t: t[:2]), dict(q_starts=lambda t: t.long()), dict(kv_lens=lambda t: t[:1]), dict(kv_lens=lambda t: t.float()),
    dict(k_cache=lambda t: t[:, :0], v_cache=lambda t: t[:, :0]),
]


@pytest.mark.parametrize("change", BATCHES + [dict(v=lambda t: t[:2]), dict(v=lambda t: t.float()), dict(k=lambda t: t.double(), v=lambda t: t.double())])
def test_append_refuses(tde, change):
    kw = good_batch()
    kw["page_table"] = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    if "page_table" in change and change["page_table"](kw["page_table"]).shape == (2, 2) and change["page_table"](kw["page_table"]).dtype == torch.int32:
        kw["page_table"] = torch.tensor([[0, 1, 0], [2, 3, 0]], dtype=torch.int32, device="cuda")
    tde.append_kv(**kw)
    for name, f in change.items():
        kw[name] = f(kw[name])
    with pytest.raises(RuntimeError):
        tde.append_kv(**kw)


@pytest.mark.parametrize("change", BATCHES + [
    dict(q=lambda t: t.float(), k_cache=lambda t: t.float(), v_cache=lambda t: t.float()), dict(q=lambda t: t[:, :3]), dict(q=lambda t: t[0]), dict(scale=lambda t: 0.0),
    dict(scale=lambda t: -1.0), dict(scale=lambda t: float("inf")), dict(q=lambda t: torch.zeros((3, 4, 264), dtype=t.dtype, device="cuda")),
    dict(k_cache=lambda t: torch.zeros(t.numel() + 4, dtype=t.dtype, device="cuda")[4:].view(t.shape)),      # not on 16 bytes
    dict(k_cache=lambda t: torch.zeros((4, 16, 2, 68), dtype=t.dtype, device="cuda")[..., :64]),             # rows not on 16 bytes
])
def test_attention_refuses(tde, change):
    kw = good_batch()
    del kw["k"], kw["v"]
    kw["q"], kw["scale"] = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda"), None
    if "page_table" in change:
        kw["page_table"] = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    tde.paged_attention(**kw)
    for name, f in change.items():
        kw[name] = f(kw[name])
    with pytest.raises(RuntimeError):
        tde.paged_attention(**kw)
