"""``trispconv.pytorch`` served by ``trispconv_amd.pytorch``.

The submodules (cache, indices, functional, weight, modules, sequence, tensor, compat)
are the same module objects under both names, so ``from trispconv.pytorch.indices
import generate_subm_indice_pairs`` and friends work as with the reference.
"""
import sys as _sys

import trispconv_amd.pytorch as _impl
from trispconv_amd.pytorch import (cache, compat, functional, indices, modules,  # noqa: F401
                                   sequence, tensor, weight)
from trispconv_amd.pytorch import *  # noqa: F401,F403

for _name in ("cache", "compat", "functional", "indices", "modules", "sequence", "tensor", "weight"):
    _sys.modules[f"{__name__}.{_name}"] = getattr(_impl, _name)

__all__ = list(_impl.__all__)
