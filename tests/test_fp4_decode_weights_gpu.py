"""paged_attention_fp4 of at most 16 rows a sequence keeps weights as two numbers of T whatever pages and slots are like."""
import types

import pytest
import torch

import test_fp4_edges_gpu as edges
from block_reference import Batch, assert_close
from test_paged_attention_scores_gpu import CALLS, softmax_of, whole

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


@pytest.mark.parametrize("call", ["decode", "decode whole"])
@pytest.mark.parametrize("page", [1, 5, 12, 17])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_pages_that_8_does_not_divide(tde, call, page, dim, dtype):
    """A step of a step of a weight is lost at most."""
    new, lens, heads, kv_heads = CALLS[call]
    batch = Batch(new, lens, page_size=page, seed=11)
    q = whole((batch.tokens, heads, dim), -3, 3, 12)
    keys = [whole((n, kv_heads, dim), -3, 3, 13 + b) for b, n in enumerate(lens)]
    edges.check(tde, batch, q, keys, edges.values_of(lens, kv_heads, dim, 1000), kv_heads, dtype, 2.0 ** -5, torch.finfo(dtype).eps ** 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_slots_far_apart(tde, dtype):
    slot, dim, kv_heads, lens = 1 << 27, 128, 2, [300, 40]
    batch = Batch([1, 3], lens, page_size=16, seed=3)
    q = whole((batch.tokens, 4, dim), -3, 3, 12)
    keys, values = [whole((n, kv_heads, dim), -3, 3, 13 + b) for b, n in enumerate(lens)], edges.values_of(lens, kv_heads, dim, 1000)
    (k, keys), (v, values) = (edges.codes_of(batch, kv_heads, dim, x) for x in (keys, values))
    far = torch.zeros(15 * slot + batch.pages * kv_heads * 4, dtype=torch.uint8, device="cuda")
    v[1] = far.as_strided((batch.pages, 16, kv_heads, 4), (kv_heads * 4, slot, 4, 1)).copy_(v[1])
    starts, scale = batch.starts.tolist(), 2.0 ** -5
    got = tde.paged_attention_fp4(q.to(dtype), *k, *v, *batch.on("cuda"), scale)

    def scores(b, head):
        return q[starts[b]:starts[b + 1], head] @ keys[b][:, head // 2].t().contiguous() * scale

    assert_close(got, *softmax_of(batch, scores, lambda b, h: values[b][:, h], 4, kv_heads, dim, dtype, torch.finfo(dtype).eps ** 2))


@pytest.mark.parametrize("dim,seqs", [(256, 270), (64, 800)])
def test_calls_that_fill_the_units(tde, dim, seqs):
    """As many rows as larger tiles begin at: 128 heads that share 8.  The last four sequences are compared."""
    lens, dtype, scale = [20 + b % 7 for b in range(seqs)], torch.bfloat16, 2.0 ** -5
    batch = Batch([1] * seqs, lens, page_size=12, seed=5)
    q = whole((seqs, 128, dim), -3, 3, 12)
    keys = [whole((n, 8, dim), -3, 3, 13 + b) for b, n in enumerate(lens)]
    (k, keys), (v, values) = (edges.codes_of(batch, 8, dim, x) for x in (keys, edges.values_of(lens, 8, dim, 5000)))
    got = tde.paged_attention_fp4(q.to(dtype), *k, *v, *batch.on("cuda"), scale)
    last = types.SimpleNamespace(tokens=4, new=[1] * 4, lens=lens[-4:])

    def scores(b, head):
        return q[seqs - 4 + b, head:head + 1] @ keys[seqs - 4 + b][:, head // 16].t().contiguous() * scale

    assert_close(got[-4:], *softmax_of(last, scores, lambda b, h: values[seqs - 4 + b][:, h], 128, 8, dim, dtype, torch.finfo(dtype).eps ** 2))
