"""SerialOrder's key has 15 bits for the sample (any device: torch's own sort)."""
import pytest
import torch

import trispconv.pytorch as spconv


def _tensor(batch_size, samples):
    idx = torch.tensor([[b, 0, 0, i] for i, b in enumerate(samples)], dtype=torch.int32)
    return spconv.SparseConvTensor(torch.arange(float(len(idx)))[:, None], idx, [4, 4, 8], batch_size)


def test_as_many_samples_as_the_key_holds():
    y = spconv.SerialOrder("o")(_tensor(32767, [32766, 0, 5]))
    assert y.features.flatten().tolist() == [1.0, 2.0, 0.0]
    offsets = y.indice_dict["o"].offsets
    assert offsets.shape == (32768,)
    assert [int(offsets[i]) for i in (0, 1, 5, 6, 32766, 32767)] == [0, 1, 1, 2, 2, 3]


def test_more_samples_are_refused():
    with pytest.raises(ValueError, match="32767 samples"):
        spconv.SerialOrder("o")(_tensor(32768, [0, 32767]))
