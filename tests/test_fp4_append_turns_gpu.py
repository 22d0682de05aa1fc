"""append_kv_fp4 of many rows of several heads: a wavefront takes as many rows as it holds several times, and kinds change from one time to the next."""
import pytest
import torch

from block_reference import Batch
from test_fp4_cache_gpu import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


# Groups of rows (of 2048 / dim heads of one kind) of queries, keys, values, and how often a wavefront takes four of them: with 2060 tokens 3 + 2 + 2 and twice, 5 + 3 + 3
# and three times, 5 + 1 + 1 and twice, 0 + 4 + 4 and twice (keys, then values), 3 + 1 + 1 and twice, 0 + 2 + 2 + ... ; with 1400 10 + 2 + 2, two wavefronts twice.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot,interleaved,norm,queries", [
    (2060, 20, 10, 64, 64, False, True, True), (2060, 9, 5, 256, 256, False, True, True), (2060, 17, 4, 128, 64, True, False, True), (2060, 1, 13, 96, 96, False, False, False),
    (2060, 33, 3, 32, 32, True, True, True), (2060, 1, 9, 192, 96, False, True, True), (1400, 40, 8, 128, 128, False, True, True), (4200, 2, 9, 128, 0, False, True, True)])
def test_several_turns(tde, tokens, heads, kv_heads, dim, rot, interleaved, norm, queries, dtype):
    first = tokens // 2 + 17
    batch = Batch([first, 1, tokens - first - 7], [first, 90, tokens], 24, seed=4, pad=6)
    run(tde, batch, heads, kv_heads, dim, dtype, rot, interleaved, norm, seed=dim, queries=queries, heads_first=True)
