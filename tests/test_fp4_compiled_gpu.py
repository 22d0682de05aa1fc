"""The operators over a cache in 4 bits in a graph that is traced whole and run without a code generator: shapes, changed arguments and results are theirs."""
import pytest
import torch

from test_fp4_cache_gpu import cos_sin
from test_fp4_edges_gpu import a_step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_step(tde, backend):
    batch, cache, qkv = a_step()
    gamma, cs = torch.ones(64, dtype=torch.bfloat16, device="cuda"), cos_sin(64, 64).cuda()
    wide = torch.full((3, 6), -1, dtype=torch.int32)
    wide[:, :batch.table.size(1)] = batch.table
    free = torch.arange(2, dtype=torch.int32, device="cuda") + batch.pages - 2

    def step(rows, table, lens, free, count, k_cache, k_scales, v_cache, v_scales, out):
        starts, positions, slots = tde.update_pages(table, lens, torch.ones_like(lens), free, count, 16, 3)
        q = tde.append_kv_fp4(rows[:, 4:5] * 2, rows[:, 5:], k_cache, k_scales, v_cache, v_scales, table, starts, lens, cos_sin=cs, positions=positions, q=rows[:, :4],
                              q_gamma=gamma, k_gamma=gamma)
        tde.append_kv_fp4(rows[:, 4:5], rows[:, 5:], k_cache, k_scales, v_cache, v_scales, table, starts, lens)
        tde.paged_attention_fp4_out(q, k_cache, k_scales, v_cache, v_scales, table, starts, lens, out)
        back = tde.unpack_fp4(k_cache, k_scales).float() + 1
        return tde.paged_attention_fp4(q, k_cache, k_scales, v_cache, v_scales, table, starts, lens).float() + 1, back, slots + 1

    results = []
    for f in (step, torch.compile(step, backend=backend, fullgraph=True)):
        args = [wide.cuda(), batch.kv_lens.cuda(), free.clone(), torch.tensor([2], dtype=torch.int32, device="cuda"), *(x.clone() for x in cache), torch.zeros_like(qkv[:, :4])]
        outs = f(qkv, *args)
        torch.cuda.synchronize()
        results.append([*outs, *args])
    for i, (got, want) in enumerate(zip(results[1], results[0])):
        assert torch.equal(got, want), i
    assert not torch.equal(results[0][7], cache[0]) and torch.equal(results[0][0], results[0][-1].float() + 1)
