"""VoxelCache's bookkeeping: what its calls take for numbers of rows and samples."""
import pytest
import torch

import trispconv.pytorch as spconv


def _cache():
    return spconv.VoxelCache(samples=3, positions=40, kv_heads=2, dim=8, pages=8, page_rows=8, device="cpu")


@pytest.mark.parametrize("rows", [[2.5, 0, 0], torch.tensor([2.5, 0.0, 0.0]), [1, float("nan"), 0],
                                  torch.tensor([0.0, -0.5, 0.0])])
def test_rows_that_are_not_whole_are_refused(rows):
    c = _cache()
    c.extend([4, 0, 9])
    with pytest.raises(ValueError):
        c.extend(rows)
    assert c.rows() == [4, 0, 9] == c.lengths.tolist() and c.free_pages() == 5


def test_whole_rows_of_any_type_count_as_integers():
    c = _cache()
    c.extend(torch.tensor([4.0, 0.0, 9.0]))
    c.extend([1.0, torch.tensor(2), True])
    assert c.rows() == [5, 2, 10] == c.lengths.tolist() and c.free_pages() == 4
    assert all(type(n) is int for n in c.rows())
    c.extend([9, 0, 0])
    assert c.rows() == [14, 2, 10] and c.free_pages() == 3
