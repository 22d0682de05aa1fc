"""What autograd sees of the tensors that append_kv and paged_attention_out change."""
import pytest
import torch

from block_reference import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def setup():
    batch = Batch([2, 1], [5, 9], page_size=4, seed=1)
    k_cache, v_cache = (torch.randn((batch.pages, 4, 1, 64), dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
    rows = torch.randn((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    return batch.on("cuda"), k_cache, v_cache, rows


@pytest.mark.parametrize("queries", [False, True])
def test_append_counts_as_a_change(tde, queries):
    args, k_cache, v_cache, rows = setup()
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = (k_cache * w).sum() + (v_cache * w).sum()
    before = k_cache._version, v_cache._version
    tde.append_kv(rows[:, 1:2], rows[:, 2:3], k_cache, v_cache, *args, q=rows[:, :1] if queries else None)
    assert k_cache._version > before[0] and v_cache._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_attention_into_an_output_counts_as_a_change(tde):
    args, k_cache, v_cache, rows = setup()
    out = torch.zeros_like(rows)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = (out * w).sum()
    before = out._version, k_cache._version
    tde.paged_attention_out(rows, k_cache, v_cache, *args, out)
    assert out._version > before[0] and k_cache._version == before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors_have_no_count(tde):
    with torch.inference_mode():
        args, k_cache, v_cache, rows = setup()
        out = torch.zeros_like(rows)
        tde.append_kv(rows[:, 1:2], rows[:, 2:3], k_cache, v_cache, *args)
        tde.paged_attention_out(rows, k_cache, v_cache, *args, out)
        assert torch.equal(out, tde.paged_attention(rows, k_cache, v_cache, *args))
