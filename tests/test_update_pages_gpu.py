"""update_pages against the moves of one page at a time: every array whole, after every step."""
import pytest
import torch

from fp4_reference import Pages

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def ints(x):
    return torch.as_tensor(x, dtype=torch.int32)


class Both:
    """The same state on the GPU and as lists."""

    def __init__(self, seqs, width, pages, seed=0, room=None):
        g = torch.Generator().manual_seed(seed)
        room = pages if room is None else room
        free = torch.full((room,), -5, dtype=torch.int32)
        free[:min(room, pages)] = torch.randperm(pages, generator=g).to(torch.int32)[:room]
        count = min(room, pages)
        table, lens = torch.full((seqs, width), -9, dtype=torch.int32), torch.zeros(seqs, dtype=torch.int32)
        self.here = Pages(table, lens, free, count)
        self.table, self.lens, self.free, self.count = table.cuda(), lens.cuda(), free.cuda(), ints([count]).cuda()

    def step(self, tde, new, page, tokens, keep=None):
        want = self.here.step(new, page, tokens, keep)
        got = tde.update_pages(self.table, self.lens, ints(new).cuda(), self.free, self.count, page, tokens, keep_lens=None if keep is None else ints(keep).cuda())
        self.check(got, want)
        return got

    def check(self, got, want):
        for name, g, w in zip(("q_starts", "positions", "slots"), got, want):
            assert torch.equal(g.cpu().long(), w), name
        assert got[0].dtype == got[1].dtype == torch.int32 and got[2].dtype == torch.int64
        for name, g, w in (("table", self.table, self.here.table), ("lens", self.lens, self.here.lens), ("free", self.free, self.here.free)):
            assert torch.equal(g.cpu().long(), w), name
        assert int(self.count) == self.here.count


@pytest.mark.parametrize("seqs,page,width,most", [(1, 1, 9, 3), (3, 4, 5, 9), (64, 16, 8, 40), (65, 5, 9, 30), (256, 16, 4, 20), (257, 8, 6, 20), (1024, 16, 3, 9),
                                                  (1025, 16, 3, 9), (2500, 3, 4, 6)])
@pytest.mark.parametrize("spare", [1.0, 0.4])
def test_steps(tde, seqs, page, width, most, spare):
    """Sequences grow, shrink, end and begin; with too few pages, some wait."""
    g = torch.Generator().manual_seed(seqs)
    both = Both(seqs, width, max(1, int(seqs * width * spare)), seed=seqs)
    for i in range(6):
        new = torch.randint(0, most + 1, (seqs,), generator=g)
        lens = both.here.lens
        keep = (torch.rand(seqs, generator=g) * (lens + 2)).long()
        keep[torch.rand(seqs, generator=g) < 0.3] = 0
        rows = int(new.sum())
        tokens = [rows, rows + 7, max(1, rows // 2), 5000, rows, 0][i]
        both.step(tde, new, page, tokens, None if i % 3 == 0 else keep)


def test_one_token_a_step_until_pages_run_out(tde):
    both = Both(5, 4, 9, seed=3)
    for _ in range(14):
        both.step(tde, [1] * 5, 3, 5)
    assert int(both.count) == 0
    starts = both.step(tde, [1] * 5, 3, 5, keep=[0, 99, 0, 1, 99])[0]    # two sequences end, one goes back to its first token
    assert int(starts[-1]) == 5


def test_what_is_dropped_and_added_again_is_the_same(tde):
    """The first page that went back is the first that comes, so a step that is undone and done again finds its pages."""
    both = Both(40, 30, 1000, seed=4)
    g = torch.Generator().manual_seed(1)
    both.step(tde, torch.randint(1, 200, (40,), generator=g), 8, 8000)
    lens, table, free = both.lens.clone(), both.table.clone(), both.free[:int(both.count)].clone()
    keep = (torch.rand(40, generator=g) * lens.cpu()).int()
    starts = both.step(tde, lens.cpu() - keep, 8, 8000, keep=keep)[0]
    assert torch.equal(lens, both.lens) and torch.equal(table, both.table) and torch.equal(free, both.free[:int(both.count)])
    assert int(starts[-1]) == int((lens.cpu() - keep).sum())


def test_long_sequences_move_many_pages(tde):
    both = Both(6, 2000, 9000, seed=5)
    both.step(tde, [30000, 5, 0, 31999, 32000, 32001], 16, 94004)          # the last asks for more than its row holds
    assert int(both.lens[5]) == 0
    both.step(tde, [1, 31000, 31000, 0, 9, 32000], 16, 94016, keep=[17, 0, 0, 31999, 0, 0])
    both.step(tde, [0] * 6, 16, 3, keep=[0] * 6)
    assert int(both.count) == 9000


def test_rows_beyond_the_batch_wait(tde):
    both = Both(6, 10, 100, seed=6)
    starts = both.step(tde, [3, 4, 5, 1, 0, 2], 4, 8)[0]   # 3 + 4 fit; the third does not, nor does what comes behind it
    assert starts.tolist() == [0, 3, 7, 7, 7, 7, 7]
    starts = both.step(tde, [0, 0, 5, 1, 0, 2], 4, 8)[0]
    assert starts.tolist() == [0, 0, 0, 5, 6, 6, 8]


def test_without_pages_those_that_need_none_go_on(tde):
    both = Both(4, 10, 3, seed=7)
    both.step(tde, [3, 4, 1, 0], 4, 8)
    starts = both.step(tde, [1, 1, 2, 1], 4, 8)[0]
    assert starts.tolist() == [0, 1, 1, 3, 3]
    assert int(both.count) == 0


def test_odd_arrays(tde):
    """Lengths below zero and beyond the table, counts below zero and beyond the stack, tables without columns or rows: nothing is touched out of place."""
    both = Both(4, 3, 5, seed=8, room=7)
    for lens, count, new, keep in (([-3, 100, 5, 0x7fffffff], 5, [2, 1, 0, 1], None), ([-3, 100, 5, 7], -4, [2, 1, 0, 1], [1, 2, 3, -1]),
                                   ([9, 9, 9, 9], 100, [-5, 0x7fffffff, 0, 1], [0, 0, 0, 0]), ([2, 0x7fffffff, 1, 0], 2, [1, 0x7fffffff, 0x7fffffff, 1], [2, 0x7ffffffe, 5, 6])):
        both.here.lens, both.here.count = torch.tensor(lens), count
        both.lens.copy_(ints(lens))
        both.count.fill_(count)
        both.here.table.copy_(torch.arange(12).view(4, 3))
        both.table.copy_(both.here.table)
        both.step(tde, new, 4, 9, keep)
    none = Both(0, 3, 2)
    assert none.step(tde, [], 4, 3)[0].tolist() == [0]
    narrow = Both(3, 0, 2)
    narrow.step(tde, [0, 1, 0], 4, 3)
    assert [t.numel() for t in Both(3, 2, 6).step(tde, [0, 0, 0], 4, 0)] == [4, 0, 0]


def test_strided_table(tde):
    both = Both(5, 4, 20, seed=9)
    wide = torch.full((5, 11), 77, dtype=torch.int32, device="cuda")
    wide[:, 3:7] = both.table
    both.table = wide[:, 3:7]
    both.step(tde, [3, 9, 1, 16, 2], 4, 40)
    both.step(tde, [3, 0, 1, 0, 2], 4, 40, keep=[1, 0, 1, 3, 2])
    assert bool((wide[:, :3] == 77).all()) and bool((wide[:, 7:] == 77).all())


def test_a_captured_step_follows_its_arrays(tde):
    both = Both(9, 12, 60, seed=10)
    new, keep = ints([0] * 9).cuda(), ints([0] * 9).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = tde.update_pages(both.table, both.lens, new, both.free, both.count, 4, 50, keep_lens=keep)
    g = torch.Generator().manual_seed(2)
    for _ in range(5):
        n = torch.randint(0, 9, (9,), generator=g)
        k = (torch.rand(9, generator=g) * (both.here.lens + 1)).long()
        new.copy_(n)
        keep.copy_(k)
        graph.replay()
        torch.cuda.synchronize()
        both.check(got, both.here.step(n, 4, 50, k))


def test_versions_rise(tde):
    both = Both(2, 3, 5)
    before = [t._version for t in (both.table, both.lens, both.free, both.count)]
    both.step(tde, [1, 2], 4, 3)
    assert all(t._version > b for t, b in zip((both.table, both.lens, both.free, both.count), before))


def test_refusals(tde):
    def call(**kw):
        base = dict(table=torch.zeros((2, 3), dtype=torch.int32, device="cuda"), lens=ints([0, 0]).cuda(), new=ints([1, 1]).cuda(), free=ints(range(6)).cuda(),
                    count=ints([6]).cuda(), page=4, tokens=2, keep=None)
        base.update(kw)
        return tde.update_pages(base["table"], base["lens"], base["new"], base["free"], base["count"], base["page"], base["tokens"], keep_lens=base["keep"])

    call()
    both = torch.zeros(40, dtype=torch.int32, device="cuda")
    for kw, match in ((dict(table=torch.zeros((2, 3), device="cuda")), "page_table"), (dict(table=torch.zeros(6, dtype=torch.int32, device="cuda")), "page_table"),
                      (dict(table=torch.zeros((3, 2), dtype=torch.int32, device="cuda").t()), "page_table"),
                      (dict(table=torch.zeros((1, 3), dtype=torch.int32, device="cuda").expand(2, 3)), "page_table overlap"),
                      (dict(lens=ints([0]).cuda()), "kv_lens"), (dict(new=ints([0, 1])), "GPU"), (dict(new=torch.zeros(2, dtype=torch.int64, device="cuda")), "new_tokens"),
                      (dict(keep=ints([0, 1, 2]).cuda()), "keep_lens"), (dict(count=ints([1, 2]).cuda()), "free_count"), (dict(free=torch.zeros((2, 2), dtype=torch.int32, device="cuda")), "free_pages"),
                      (dict(page=0), "page"), (dict(page=1 << 31), "page"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "update_pages"),
                      (dict(lens=both[:2], new=both[1:3]), "overlaps new_tokens"), (dict(table=both[:6].view(2, 3), free=both[5:20]), "overlaps"),
                      (dict(lens=both[:2], keep=both[:2]), "overlaps keep_lens"), (dict(free=both[:6], count=both[5:6]), "overlaps")):
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
