"""A server's steps over a cache in 4 bits: update_pages, append_kv_fp4, paged_attention_fp4 one behind the other, eager and replayed from a graph, against
the same state on the CPU in doubles."""
import pytest
import torch

from block_reference import Batch, assert_close, attention, norm_rope
from fp4_reference import Pages, as_read, encode, most_exponent

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def ints(x):
    return torch.as_tensor(x, dtype=torch.int32)


class Server:
    """What stays on the GPU between steps, and a step."""

    def __init__(self, tde, seqs, width, pages, page, heads, kv_heads, dim, dtype, tokens):
        self.tde, self.page, self.tokens, self.heads, self.kv_heads = tde, page, tokens, heads, kv_heads
        g = torch.Generator().manual_seed(dim)
        self.cache = tde.fp4_cache(pages, page, kv_heads, dim)
        self.table, self.lens = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda"), torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.free, self.count = torch.randperm(pages, generator=g).to(torch.int32).cuda(), ints([pages]).cuda()
        self.new, self.keep = ints([0] * seqs).cuda(), ints([0] * seqs).cuda()
        self.qkv = torch.zeros((tokens, heads + 2 * kv_heads, dim), dtype=dtype, device="cuda")
        self.gammas = [(torch.randn((dim,), generator=g) * 0.2 + 1).to(dtype).cuda() for _ in (0, 1)]
        angles = torch.arange(width * page).double()[:, None] * 100.0 ** (-torch.arange(0, dim, 2).double() / dim)
        self.cos_sin = torch.cat([angles.cos(), angles.sin()], 1).float().cuda()

    def step(self):
        starts, positions, slots = self.tde.update_pages(self.table, self.lens, self.new, self.free, self.count, self.page, self.tokens, keep_lens=self.keep)
        q, k, v = self.qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        q = self.tde.append_kv_fp4(k, v, *self.cache, self.table, starts, self.lens, cos_sin=self.cos_sin, positions=positions, q=q, q_gamma=self.gammas[0],
                                   k_gamma=self.gammas[1])
        return starts, positions, slots, q, self.tde.paged_attention_fp4(q, *self.cache, self.table, starts, self.lens)

    def state(self):
        return [self.table, self.lens, self.free, self.count, *self.cache]


class Host:
    """The same on the CPU."""

    def __init__(self, server):
        self.pages = Pages(server.table.cpu(), server.lens.cpu(), server.free.cpu(), int(server.count))
        self.cache = [x.cpu() for x in server.cache]
        self.gammas, self.cos_sin = [x.cpu() for x in server.gammas], server.cos_sin.cpu()

    def check(self, server, new, keep, qkv, got):
        tokens, page, dtype = server.tokens, server.page, qkv.dtype
        want = self.pages.step(new, page, tokens, keep)
        for name, g, w in zip(("q_starts", "positions", "slots"), got, want):
            assert torch.equal(g.cpu().long(), w), name
        starts, positions, slots = want
        for name, g, w in zip(("table", "lens", "free"), server.state(), (self.pages.table, self.pages.lens, self.pages.free)):
            assert torch.equal(g.cpu().long(), w), name
        assert int(server.count) == self.pages.count
        batch = Batch.__new__(Batch)
        batch.new, batch.lens, batch.page, batch.pad = (starts[1:] - starts[:-1]).tolist(), self.pages.lens.tolist(), page, tokens - int(starts[-1])
        batch.pages, batch.table, batch.tokens = self.cache[0].size(0), self.pages.table, tokens
        q, k, v = qkv.split([server.heads, server.kv_heads, server.kv_heads], dim=1)
        rows = torch.full((tokens, self.cos_sin.size(1)), float("nan"))
        rows[positions >= 0] = self.cos_sin[positions[positions >= 0]]
        q_want, q_bound = norm_rope(q, self.gammas[0], 1e-6, rows, False, dtype)
        q_want[positions < 0], q_bound[positions < 0] = 0.0, 0.0
        assert_close(got[3], q_want, q_bound, "queries")
        k_want, _ = norm_rope(k, self.gammas[1], 1e-6, rows, False, dtype)
        filled = slots >= 0
        for i, x in ((0, k_want), (2, v.double())):
            for part, bytes_ in zip(self.cache[i:i + 2], encode(x[filled], most_exponent(dtype))):
                part[slots[filled] // page, slots[filled] % page] = bytes_
        for name, g, w in zip(("k_cache", "k_scales", "v_cache", "v_scales"), server.cache, self.cache):
            assert torch.equal(g.cpu(), w), name
        held = server.tde.unpack_fp4(*server.cache[:2], out_dtype=dtype).flatten(0, 1)[slots[filled].cuda()]
        assert torch.equal(held.cpu().double(), as_read(*self.cache[:2], dtype).flatten(0, 1)[slots[filled]])
        out, bound = attention(batch, got[3].cpu(), as_read(*self.cache[:2], dtype), as_read(*self.cache[2:], dtype), qkv.size(2) ** -0.5)
        assert_close(got[4], out, bound, "attention")


# (rows of a sequence at most; how many sequences end) of each step: prompts, tokens one at a time, drafts some of which are dropped, others' prompts
STEPS = [(40, 0.0), (1, 0.0), (1, 0.0), (4, 0.0), (4, 0.0), (30, 0.5), (1, 0.0), (3, 0.3), (1, 1.0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,page,tokens", [(8, 2, 64, 16, 150), (4, 1, 128, 24, 90), (3, 3, 96, 4, 200), (6, 2, 256, 8, 70)])
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "captured"])
def test_steps_of_a_server(tde, heads, kv_heads, dim, page, tokens, dtype, captured):
    seqs, width = 6, -(-100 // page)
    args = (tde, seqs, width, seqs * width * 2 // 3, page, heads, kv_heads, dim, dtype, tokens)
    server = Server(*args)
    host, eager, graph = Host(server), Server(*args), None
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = server.step()
    g = torch.Generator().manual_seed(page)
    for most, gone in STEPS:
        new = torch.randint(1, most + 1, (seqs,), generator=g)
        keep = (host.pages.lens - torch.randint(0, 3, (seqs,), generator=g)).clamp(min=0)
        keep[torch.rand(seqs, generator=g) < gone] = 0
        qkv = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=g).to(dtype)
        for one in (server, eager) if captured else (server,):
            one.new.copy_(new)
            one.keep.copy_(keep)
            one.qkv.copy_(qkv)
        if captured:
            graph.replay()
        else:
            got = server.step()
        torch.cuda.synchronize()
        host.check(server, new, keep, qkv, got)
        if captured:
            for i, (a, b) in enumerate(zip([*got, *server.state()], [*eager.step(), *eager.state()])):
                assert torch.equal(a, b), i
