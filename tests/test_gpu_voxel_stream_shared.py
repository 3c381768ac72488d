"""Samples that share pages, through blocks whose windows end inside what is
shared, behind it and before it, against copies of the same rows."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu
from test_gpu_voxel_block import _input
from test_gpu_voxel_stream import _blocks, _cache, _step

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.float16, 2 ** -8)])
@pytest.mark.parametrize("window,sinks", [((200, 0), 3), ((20, 0), 0), ((20, 0), 5), ((90, 4), 100), ((0, 0), 1)])
@pytest.mark.parametrize("steps", [[(1, 1, 1), (1, 2, 30), (0, 1, 2)], [(150, 3, 70), (1, 1, 1)]])
def test_sharing_in_a_window(steps, window, sinks, dtype, tol):
    """Tolerances relative to the largest feature: f32 sums in another order (some
    hundred terms of 2^-24 each), and in 16 bits a rounding or two of the features
    (2^-11 each) that falls the other way."""
    blocks = [m.to(DEV).to(dtype) for m in _blocks(window=window, sinks=sinks)]
    scene = _input((160, 0, 0), dtype=dtype, seed=1)
    shared, copies = _cache(dtype=dtype), _cache(dtype=dtype)
    _step(blocks, scene, shared)
    shared.share(0, [1, 2], 160)
    idx = scene.indices.repeat(3, 1)
    idx[:, 0] = torch.arange(3, device=DEV).repeat_interleave(160)
    _step(blocks, spconv.SparseConvTensor(scene.features.repeat(3, 1), idx, scene.spatial_shape, 3), copies)
    for i, rows in enumerate(steps):
        x = _input(rows, dtype=dtype, seed=20 + i)
        a, b = _step(blocks, x, shared), _step(blocks, x, copies)
        assert shared._tables()[1].shape == (10,) and copies._tables()[1] is None
        err = (a.features - b.features).abs().max() / b.features.abs().max()
        assert float(err) <= tol, (i, float(err))
    assert shared.rows() == copies.rows()
