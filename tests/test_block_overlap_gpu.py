"""append_kv and paged_attention_out refuse tensors to write that overlap themselves or what the call reads; slices beside each other are fine."""
import pytest
import torch

from block_reference import Batch

pytestmark = pytest.mark.gpu
ROWS, HEADS, DIM = 6, 4, 64


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def randn(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape))).to(torch.bfloat16).cuda()


def setup():
    batch = Batch([4, 2], [20, 9], page_size=8, seed=1)
    return batch, batch.on("cuda")


def cache_pairs(batch):
    """Keys and values apart, in one tensor in different ways, and with the heads in front."""
    p = batch.pages
    side = randn(p, 2, 8, 2, DIM)
    pages = randn(2 * p, 8, 2, DIM)
    heads = randn(p, 8, 4, DIM)
    channels = randn(p, 8, 2, 2 * DIM)
    front = randn(p, 2, 8, DIM)
    return {
        "apart": (randn(p, 8, 2, DIM), randn(p, 8, 2, DIM)), "side by side": (side[:, 0], side[:, 1]), "pages in turn": (pages[::2], pages[1::2]),
        "pages": (pages[:p], pages[p:]), "heads": (heads[:, :, :2], heads[:, :, 2:]), "heads in turn": (heads[:, :, ::2], heads[:, :, 1::2]),
        "channels": (channels[..., :DIM], channels[..., DIM:]), "heads in front": (front.transpose(1, 2), randn(p, 2, 8, DIM).transpose(1, 2)),
    }


@pytest.mark.parametrize("kind", ["apart", "side by side", "pages in turn", "pages", "heads", "heads in turn", "channels", "heads in front"])
def test_caches_beside_each_other(tde, kind):
    batch, args = setup()
    k_cache, v_cache = cache_pairs(batch)[kind]
    qkv = randn(ROWS, HEADS + 4, DIM)
    q, k, v = qkv.split([HEADS, 2, 2], dim=1)
    plain = k_cache.clone(memory_format=torch.contiguous_format), v_cache.clone(memory_format=torch.contiguous_format)
    tde.append_kv(k, v, *plain, *args)
    tde.append_kv(k, v, k_cache, v_cache, *args)
    assert torch.equal(k_cache, plain[0]) and torch.equal(v_cache, plain[1])
    want = tde.paged_attention(q, *plain, *args)
    room = randn(ROWS, 2 * HEADS, DIM)
    room[:, ::2] = q
    out = room[:, 1::2]                 # the queries' heads between the output's
    tde.paged_attention_out(room[:, ::2], k_cache, v_cache, *args, out)
    assert torch.equal(out, want) and torch.equal(room[:, ::2], q)
    wide = randn(HEADS, ROWS, 2 * DIM)
    wide[..., :DIM] = q.transpose(0, 1)
    tde.paged_attention_out(wide[..., :DIM].transpose(0, 1), k_cache, v_cache, *args, wide[..., DIM:].transpose(0, 1))
    assert torch.equal(wide[..., DIM:].transpose(0, 1), want)


def test_what_is_only_read_may_overlap(tde):
    batch, args = setup()
    cache = randn(batch.pages, 8, 1, DIM)
    q = randn(ROWS, 1, DIM).expand(ROWS, HEADS, DIM)
    both = cache.expand(batch.pages, 8, 2, DIM)
    got = tde.paged_attention(q, both, both, *args)
    assert torch.equal(got, tde.paged_attention(q.contiguous(), both.contiguous(), both.contiguous(), *args))
    one = randn(ROWS, 1, DIM).expand(ROWS, 2, DIM)
    caches = [torch.zeros((batch.pages, 8, 2, DIM), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    tde.append_kv(one, one, *caches, *args)
    assert torch.equal(*caches)


def refused(tde, call, message):
    with pytest.raises(RuntimeError, match=message):
        call()


def test_append_refuses(tde):
    batch, args = setup()
    p = batch.pages
    k, v = randn(ROWS, 2, DIM), randn(ROWS, 2, DIM)
    cache, other = randn(p, 8, 2, DIM), randn(p + 1, 8, 2, DIM)
    before = other.clone()
    refused(tde, lambda: tde.append_kv(k, v, cache, cache, *args), "k_cache overlaps v_cache")
    refused(tde, lambda: tde.append_kv(k, v, other[:p], other[1:], *args), "k_cache overlaps v_cache")
    refused(tde, lambda: tde.append_kv(k, v, other[:p, :, :1].expand(p, 8, 2, DIM), cache, *args), "elements of k_cache overlap")
    refused(tde, lambda: tde.append_kv(k, v, cache, other[:1].expand(p, 8, 2, DIM), *args), "elements of v_cache overlap")
    rows = other.view(-1, 2, DIM)[3:3 + ROWS]
    refused(tde, lambda: tde.append_kv(rows, v, other[:p], cache, *args), "k_cache overlaps k")
    refused(tde, lambda: tde.append_kv(k, rows, other[:p], cache, *args), "k_cache overlaps v")
    refused(tde, lambda: tde.append_kv(k, rows, cache, other[:p], *args), "v_cache overlaps v")
    refused(tde, lambda: tde.append_kv(k, v, cache, other[:p], *args, q=rows), "v_cache overlaps q")
    torch.cuda.synchronize()
    assert torch.equal(other, before)


def test_attention_refuses(tde):
    batch, args = setup()
    k_cache, v_cache = randn(batch.pages, 8, 2, DIM), randn(batch.pages, 8, 2, DIM)
    room = randn(ROWS + 1, 2 * HEADS, DIM)
    q, before = room[:ROWS, :HEADS], room.clone()

    def call(out, name="out"):
        return lambda: tde.paged_attention_out(q, k_cache, v_cache, *args, out)

    refused(tde, call(q), "out overlaps q")
    refused(tde, call(room[1:, :HEADS]), "out overlaps q")
    refused(tde, call(room[:ROWS, 2:2 + HEADS]), "out overlaps q")
    refused(tde, call(room[:ROWS, ::2]), "out overlaps q")
    refused(tde, call(room[:1, HEADS:].expand(ROWS, HEADS, DIM)), "elements of out overlap")
    refused(tde, call(room[:ROWS, HEADS:HEADS + 1].expand(ROWS, HEADS, DIM)), "elements of out overlap")
    refused(tde, call(room.view(-1).as_strided((ROWS, HEADS, DIM), (DIM, DIM, 1), HEADS * DIM)), "elements of out overlap")
    refused(tde, call(k_cache.view(-1)[:ROWS * HEADS * DIM].view(ROWS, HEADS, DIM)), "out overlaps k_cache")
    refused(tde, call(v_cache.view(-1)[-ROWS * HEADS * DIM:].view(ROWS, HEADS, DIM)), "out overlaps v_cache")
    torch.cuda.synchronize()
    assert torch.equal(room, before)
