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


def test_samples_and_rows_as_tensors():
    """Elements of tensors name samples and rows as integers do: the same twice is
    found, and nothing of the keeper changes with a tensor later."""
    c = _cache()
    c.extend([16, 0, 0])
    with pytest.raises(ValueError):
        c.share(0, torch.tensor([1, 1]), 8)
    assert c.rows() == [16, 0, 0] and c.free_pages() == 6
    rows = torch.tensor([8, 8])
    c.share(torch.tensor(0), torch.tensor([1, 2]), rows[0])
    rows += 5
    assert c.rows() == [16, 8, 8] and all(type(n) is int for n in c.rows())
    c.extend([0, 1, 0])
    c.drop(torch.tensor([0, 2]))
    assert c.rows() == [0, 9, 0] == c.lengths.tolist() and c.free_pages() == 6
    for bad in ((0.5, [1], 8), (1, [0.0], 8), (1, [0], 8.0)):
        with pytest.raises(TypeError):
            c.share(*bad)
    assert c.rows() == [0, 9, 0] and c.free_pages() == 6
