"""Codes that bf16 holds as infinities (scales of 2^126 and 2^127): they arrive with their sign in rows that see them, and nowhere else."""
import math

import pytest
import torch

from block_reference import Batch, assert_close, attention
from fp4_reference import as_read
from test_paged_attention_fp4_gpu import held, on_gpu, randn

pytestmark = pytest.mark.gpu
CALLS = {
    "split": ([1, 1, 1], [700, 40, 3000], 4, 2),
    "whole": ([1] * 160, [70] * 160, 8, 8),
    "few": ([2, 3], [90, 5], 4, 1),
    "drafts": ([9, 12, 7], [90, 300, 33], 4, 2),
    "chunks": ([40, 7, 150], [90, 50, 333], 6, 2),
}


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def compare(tde, batch, heads, dim, parts):
    q = randn((batch.tokens, heads, dim), torch.bfloat16, 2)
    got = tde.paged_attention_fp4(q.cuda(), *on_gpu(parts), *batch.on("cuda"))
    want, bound = attention(batch, q, as_read(*parts[:2], torch.bfloat16), as_read(*parts[2:], torch.bfloat16), dim ** -0.5)
    assert_close(got, want, bound.nan_to_num(0.0))
    return want


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("page", [16, 8, 12])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_seen_values(tde, call, page, dim):
    new, lens, heads, kv_heads = CALLS[call]
    batch = Batch(new, lens, page_size=page, seed=1, pad=2)
    parts = held(batch, kv_heads, dim, 3)

    def put(b, key, channel, code, scale):
        """A block of zeros but for one code."""
        at = (batch.page_of(b, key), key % page)
        if not bool((parts[3][at][:, channel // 32] >= 253).all()):
            parts[2][at][:, channel // 32 * 16:channel // 32 * 16 + 16] = 0
        parts[3][at][:, channel // 32] = scale
        parts[2][at][:, channel // 2] |= code << (channel % 2 * 4)

    for b, n in enumerate(lens):
        first = n - new[b]    # keys that all rows see
        for key, channel, code, scale in ((0, 0, 7, 254), (first, 1, 15, 253), (first // 2, 2, 6, 253), (first // 3, 2, 12, 254), (first // 4, dim - 1, 4, 254),
                                          (first // 2, dim - 1, 7, 253)):
            put(b, key, channel, code, scale)
        if new[b] > 3:        # and some that later rows see
            put(b, n - 2, 33, 7, 254)
            put(b, n - 3, 34, 15, 254)
    want = compare(tde, batch, heads, dim, parts)
    assert bool((want == math.inf).any()) and bool((want == -math.inf).any())


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("page", [16, 24, 12])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_what_rows_do_not_see_does_not_reach_them(tde, call, page, dim):
    """Any codes with the largest scales behind the last key, in pages of no sequence, and in the call's later rows."""
    new, lens, heads, kv_heads = CALLS[call]
    batch = Batch(new, lens, page_size=page, seed=4, pad=2)
    parts = held(batch, kv_heads, dim, 5)
    used = torch.zeros((batch.pages, page), dtype=torch.bool)
    for b, n in enumerate(lens):
        used[[batch.page_of(b, j) for j in range(n)], [j % page for j in range(n)]] = True
    for i in (1, 3):
        parts[i][~used] = torch.randint(252, 256, parts[i][~used].shape, generator=torch.Generator().manual_seed(i)).to(torch.uint8)
    for b, (n, length) in enumerate(zip(new, lens)):
        if n > 1:
            at = (batch.page_of(b, length - 1), (length - 1) % page)
            parts[2][at][:, :16], parts[3][at][:, 0] = 0x70, 254
    compare(tde, batch, heads, dim, parts)
