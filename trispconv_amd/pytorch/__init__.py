"""MI355X backend of the ``trispconv.pytorch`` API (same names, same behaviour).

Export list of trispconv/pytorch/__init__.py:13-21, then the operators and
modules of transformer blocks over the voxels.
"""
from .cache import VoxelCache, cache_attention, norm_rotate_append
from .compat import ConvAlgo
from .modules import (SparseConv3d, SparseConvolution, SparseInverseConv3d, SparseModule,
                      SparseSequential, SubMConv3d)
from .sequence import (SerialOrder, VoxelBlock, VoxelOrder, linear_act, norm_rotate_heads,
                       window_attention)
from .tensor import SparseConvTensor

__all__ = [
    "SparseConvTensor",
    "SparseConvolution",
    "SubMConv3d",
    "SparseConv3d",
    "SparseInverseConv3d",
    "SparseSequential",
    "SparseModule",
    "ConvAlgo",
    "linear_act",
    "norm_rotate_heads",
    "window_attention",
    "VoxelOrder",
    "SerialOrder",
    "VoxelBlock",
    "norm_rotate_append",
    "cache_attention",
    "VoxelCache",
]
