"""Arguments just beyond what the attention block's operators take."""
import ctypes
import math

import pytest
import torch

from torch_dist_ext_amd import _capi
from test_block_abi_host import attention


def test_scales():
    """A scale whose product with log2(e) is no fp32 number would make every weight NaN."""
    lib, n = _capi.load(), ctypes.c_int64()
    for scale, status in ((2e38, _capi.OK), (2.4e38, _capi.EINVAL), (3e38, _capi.EINVAL), (1e-45, _capi.OK), (1e-46, _capi.EINVAL), (math.inf, _capi.EINVAL)):
        assert lib.tde_paged_attention_workspace(ctypes.byref(attention(scale=scale)), ctypes.byref(n)) == status, scale


@pytest.mark.gpu
def test_scales_on_tensors(cuda_device):
    import torch_dist_ext_amd as tde
    cache = torch.randn((2, 4, 1, 64), device="cuda").to(torch.bfloat16)
    q = torch.randn((1, 1, 64), device="cuda").to(torch.bfloat16)
    table, starts, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0, 1]], [0, 1], [5]))
    out = tde.paged_attention(q, cache, cache, table, starts, lens, 1e38)
    top = (cache.view(8, 64)[:5].double() @ q.view(64).double()).argmax()
    assert torch.equal(out.view(64), cache.view(8, 64)[top])        # all weight on one key
    with pytest.raises(RuntimeError, match="scale"):
        tde.paged_attention(q, cache, cache, table, starts, lens, 2.4e38)


@pytest.mark.gpu
def test_head_counts(cuda_device):
    """Heads are counted in 32 bits: a tensor expanded beyond them is not one of its first few."""
    import torch_dist_ext_amd as tde
    many = torch.zeros((1, 1, 1), dtype=torch.bfloat16, device="cuda").expand(1, (1 << 32) + 4, 1)
    k = torch.zeros((1, 1, 1), dtype=torch.bfloat16, device="cuda")
    k_cache, v_cache = (torch.zeros((2, 4, 1, 1), dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
    table, starts, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0, 1]], [0, 1], [5]))
    with pytest.raises(RuntimeError, match="heads"):
        tde.append_kv(k, k, k_cache, v_cache, table, starts, lens, q=many)
