"""update_pages over a table as wide as it takes: 2^31 - 1 pages of a token."""
import pytest
import torch

pytestmark = pytest.mark.gpu
MOST = 0x7fffffff


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("tokens", [8, 600, 5000], ids=["one launch", "more threads", "maps apart"])
def test_a_length_ends_at_2_to_the_31st(cuda_device, tokens):
    import torch_dist_ext_amd as tde
    table = torch.empty((1, MOST), dtype=torch.int32, device="cuda")
    table[0, -4:] = -9
    lens, free, count = ints(MOST - 1), ints(5, 6, 7, 8, 9, 10, 11, -3), ints(7)
    # more tokens than a length holds: as one whose row of the table does not reach
    for new in (2, 5, MOST):
        starts, positions, slots = tde.update_pages(table, lens, ints(new), free, count, 1, tokens)
        assert starts.tolist() == [0, 0] and int(lens) == MOST - 1 and int(count) == 7
        assert table[0, -4:].tolist() == [-9] * 4 and bool((positions == -1).all()) and bool((slots == -1).all())
    starts, positions, slots = tde.update_pages(table, lens, ints(1), free, count, 1, tokens)
    assert starts.tolist() == [0, 1] and int(lens) == MOST and int(count) == 6
    assert table[0, -4:].tolist() == [-9, -9, -9, 11]
    assert positions[:2].tolist() == [MOST - 1, -1] and slots[:2].tolist() == [11, -1]
    # and back
    starts, _, slots = tde.update_pages(table, lens, ints(2), free, count, 1, tokens, keep_lens=ints(MOST - 2))
    assert starts.tolist() == [0, 2] and int(lens) == MOST and int(count) == 6 and free[:6].tolist() == [5, 6, 7, 8, 9, 10]
    assert table[0, -4:].tolist() == [-9, -9, -9, 11] and slots[:2].tolist() == [-9, 11]
