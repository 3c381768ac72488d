"""Transformer blocks over the active voxels: operators and modules.

The rows of a sparse tensor, sample after sample in some order, are packed
sequences.  Three operators run a block over them in hand-written HIP kernels
(no counterpart in the reference; inference, as everything here: their
results carry no gradient):

``linear_act``         act(x W^T + bias) + residual
``norm_rotate_heads``  RMS norm of every query and key head and its rotation
                       by the row's position, in one pass
``window_attention``   attention in a sliding window whose first keys stay
                       visible

``SerialOrder`` puts a tensor's rows into a serial order and ``VoxelBlock``
is the block: both are SparseModules for a SparseSequential.
"""
from __future__ import annotations

from typing import TYPE_CHECKING, NamedTuple, Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _lib as L
from .functional import compute_dtype
from .modules import SparseModule, _plain
from .tensor import SparseConvTensor

if TYPE_CHECKING:
    from .cache import VoxelCache

__all__ = ["linear_act", "norm_rotate_heads", "window_attention", "VoxelOrder", "SerialOrder",
           "VoxelBlock"]

_ACTS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_MOST = 2 ** 31 - 1


def _same(t: torch.Tensor, like: torch.Tensor, what: str, name: str) -> None:
    if t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise ValueError(f"{what}: {name} is {t.dtype} on {t.device}, expected {like.dtype} on "
                         f"{like.device}")


def _rows_of(t: torch.Tensor) -> Tuple[torch.Tensor, Tuple[int, ...]]:
    """``t`` with its last dimension contiguous (any strides before it), and its strides."""
    strides = t.stride()
    if strides[-1] != 1 and t.shape[-1] > 1:
        t = t.contiguous()
        strides = t.stride()
    return t, strides


def _matrix(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """``t`` as the product kernels read it, and its row stride: rows
    contiguous, less than 2^21 elements apart."""
    row, column = t.stride()
    if (column != 1 and t.shape[1] > 1) or row >= 1 << 21:
        if t.shape[0] <= 1 and (column == 1 or t.shape[1] <= 1):
            return t, 0  # one row: its stride means nothing
        t = t.clone(memory_format=torch.contiguous_format)
        row = t.stride(0)
    return t, row


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               activation: Optional[str] = None,
               residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x @ weight.T + bias) + residual, in one launch.

    x (N, C_in), weight (C_out, C_in) as ``nn.Linear`` holds it, bias (C_out),
    residual (N, C_out).  activation: None, "relu", "gelu" (x Phi(x)),
    "gelu_tanh" or "silu".  x, weight and residual share one dtype (float32,
    float16 or bfloat16) and may have any row stride; the bias may have
    another.  The sums, the bias, the activation and the residual are float32,
    rounded once to x's dtype.
    """
    what = "linear_act"
    if not x.is_cuda:
        L.require_gpu(x, what)
    code = L.dtype_code(x.dtype)
    act = _ACTS.get(activation)
    if act is None:
        raise ValueError(f"{what}: unknown activation {activation!r}; one of "
                         f"{sorted(a for a in _ACTS if a)}")
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]:
        raise ValueError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)} are not "
                         "(N, C_in) and (C_out, C_in)")
    _same(weight, x, what, "weight")
    (n, c_in), c_out = x.shape, weight.shape[0]
    (x, x_stride), (weight, w_stride) = _matrix(x), _matrix(weight)
    b_ptr = r_ptr = None
    b_code = r_stride = 0
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != c_out or bias.get_device() != x.get_device():
            raise ValueError(f"{what}: bias must have {c_out} entries on {x.device}")
        bias = bias.contiguous()
        b_ptr, b_code = bias.data_ptr(), L.dtype_code(bias.dtype)
    if residual is not None:
        if residual.shape != (n, c_out):
            raise ValueError(f"{what}: residual {tuple(residual.shape)}, expected {(n, c_out)}")
        _same(residual, x, what, "residual")
        residual, (r_stride, _) = _rows_of(residual)
        r_ptr = residual.data_ptr()
    out = x.new_empty((n, c_out))
    rc = L.lib().tsc_linear_act(x.data_ptr(), x_stride, weight.data_ptr(), w_stride, b_ptr, b_code,
                                r_ptr, r_stride, code, n, c_in, c_out, act, out.data_ptr(),
                                L.stream_of(x))
    if rc:
        L.check(rc, what)
    return out


def _position_rows(positions: torch.Tensor, q: torch.Tensor, n: int,
                   what: str) -> Tuple[torch.Tensor, int, int, bool]:
    """Checked positions of q's n rows, their axes, their row stride and whether
    they are float32."""
    dtype, shape = positions.dtype, positions.shape
    in_f32 = dtype is torch.float32
    if len(shape) != 2 or shape[0] != n or positions.get_device() != q.get_device() or \
            not (in_f32 or dtype is torch.int32):
        raise ValueError(f"{what}: positions must be ({n}, axes) int32 or float32 on {q.device}")
    positions, (row, _) = _rows_of(positions)
    return positions, shape[1], row, in_f32


def _head_gains(q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                q: torch.Tensor, hq: int, hk: int, dim: int, what: str):
    """Checked gains, and their arguments of a C entry: two pointers, the
    dtype's code and whether each has a gain per head."""
    qg_ptr = kg_ptr = None
    qg_heads = kg_heads = g_code = 0
    if q_weight is not None or k_weight is not None:
        device = q.get_device()
        g_dtype = (k_weight if q_weight is None else q_weight).dtype
        g_code = L.dtype_code(g_dtype)
        for w, h, name in ((q_weight, hq, "q_weight"), (k_weight, hk, "k_weight")):
            if w is not None and (w.shape not in ((dim,), (h, dim)) or w.get_device() != device
                                  or w.dtype is not g_dtype):
                raise ValueError(f"{what}: {name} must be ({dim},) or ({h}, {dim}) {g_dtype} on "
                                 f"{q.device}")
        if q_weight is not None:
            q_weight = q_weight.contiguous()
            qg_ptr, qg_heads = q_weight.data_ptr(), q_weight.dim() - 1
        if k_weight is not None:
            k_weight = k_weight.contiguous()
            kg_ptr, kg_heads = k_weight.data_ptr(), k_weight.dim() - 1
    return q_weight, k_weight, (qg_ptr, kg_ptr, g_code, qg_heads, kg_heads)


def norm_rotate_heads(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                      q_weight: Optional[torch.Tensor] = None,
                      k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                      base: float = 10000.0,
                      interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of q and k and its rotation by the row's position.

    q (N, Hq, D) and k (N, Hk, D) of one dtype, D even and at most 256, with
    any row and head strides (views of a packed projection); positions (N, A),
    A from 1 to 4 axes, int32 or float32, for instance ``x.indices[:, 1:]``.
    A head y is first y / sqrt(mean(y^2) + eps) * weight (weight (D,) or
    (H, D), None for 1).  Then its D/2 pairs turn: each axis has
    F = (D/2) // A of them, pair i of axis a by positions[:, a] * base^(-i/F)
    radians; left over pairs stay.  A pair is (y[j], y[j + D/2]), or
    (y[2j], y[2j+1]) with ``interleaved``.  Returns new contiguous tensors.
    """
    what = "norm_rotate_heads"
    if not q.is_cuda:
        L.require_gpu(q, what)
    code = L.dtype_code(q.dtype)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)} are not (N, Hq, D) "
                         "and (N, Hk, D)")
    _same(k, q, what, "k")
    n, hq, dim = q.shape
    hk = k.shape[1]
    positions, axes, p_row, in_f32 = _position_rows(positions, q, n, what)
    q_weight, k_weight, gains = _head_gains(q_weight, k_weight, q, hq, hk, dim, what)
    (q, (q_row, q_head, _)), (k, (k_row, k_head, _)) = _rows_of(q), _rows_of(k)
    q_out, k_out = q.new_empty(n, hq, dim), q.new_empty(n, hk, dim)
    rc = L.lib().tsc_norm_rotate_heads(
        q.data_ptr(), q_row, q_head, k.data_ptr(), k_row, k_head, positions.data_ptr(), p_row,
        in_f32, axes, *gains, eps, base, interleaved, code, n, hq, hk, dim,
        q_out.data_ptr(), k_out.data_ptr(), L.stream_of(q))
    if rc:
        L.check(rc, what)
    return q_out, k_out


def _limit(v: Optional[int], what: str) -> int:
    if v is None:
        return -1
    if v < 0:
        raise ValueError(f"{what}: a window side must not be negative (None: no limit), got {v}")
    return min(int(v), _MOST)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                     offsets_k: Optional[torch.Tensor] = None,
                     window: Tuple[Optional[int], Optional[int]] = (None, None), sinks: int = 0,
                     scale: Optional[float] = None) -> torch.Tensor:
    """Attention of packed samples in a sliding window with sinks.

    q (Nq, Hq, D), k and v (Nk, Hk, D) of one dtype, Hq a multiple of Hk
    (query heads h*G .. h*G+G-1 share key head h), D at most 256, any row and
    head strides.  offsets: int32 (B + 1,) on the GPU, sample b's queries are
    rows offsets[b] to offsets[b+1]; offsets_k the same for the keys (None:
    the queries').  A sample's queries are the last of its positions: query i
    of Lq stands at p = i + Lk - Lq, so a streaming step passes its new rows
    as q and everything kept as k and v.  It sees the keys j with
    p - left <= j <= p + right (window = (left, right), None for no limit)
    and, up to p + right, the sample's first ``sinks`` keys.  scale defaults
    to D^-0.5.  A query that sees no key gives zeros, as rows outside every
    sample do (before offsets[0], from offsets[-1] on); what lies at keys a
    query does not see (NaN, infinities) does not reach it.  Scores, maxima and
    sums are float32; for float16 and bfloat16 the softmax weights are rounded
    to that type for the product with v.
    """
    what = "window_attention"
    if not q.is_cuda:
        L.require_gpu(q, what)
    code = L.dtype_code(q.dtype)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} are "
                         "not (Nq, Hq, D), (Nk, Hk, D), (Nk, Hk, D)")
    _same(k, q, what, "k")
    _same(v, q, what, "v")
    n_q, hq, dim = q.shape
    n_k, hk, _ = k.shape
    if offsets_k is None:
        offsets_k = offsets
        if n_q != n_k:
            raise ValueError(f"{what}: {n_q} queries and {n_k} keys need offsets_k")
    if offsets.shape != offsets_k.shape or offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ValueError(f"{what}: offsets must be (B + 1,) for queries and keys, got "
                         f"{tuple(offsets.shape)} and {tuple(offsets_k.shape)}")
    for t in (offsets, offsets_k):
        if t.dtype is not torch.int32 or t.get_device() != q.get_device():
            raise ValueError(f"{what}: offsets must be int32 on {q.device}, got {t.dtype} on "
                             f"{t.device}")
    left, right = window
    left, right = _limit(left, what), _limit(right, what)
    if sinks < 0:
        raise ValueError(f"{what}: sinks must not be negative, got {sinks}")
    (q, (q_row, q_head, _)), (k, (k_row, k_head, _)) = _rows_of(q), _rows_of(k)
    v, (v_row, v_head, _) = _rows_of(v)
    offsets, offsets_k = offsets.contiguous(), offsets_k.contiguous()
    if offsets.shape[0] == 1:  # no samples
        return q.new_zeros((n_q, hq, dim))
    out = q.new_empty((n_q, hq, dim))
    lib, samples, sinks = L.lib(), offsets.shape[0] - 1, min(sinks, _MOST)
    nbytes = lib.tsc_window_attention_workspace_bytes(samples, n_q, n_k, hq, hk, dim, left, right,
                                                      sinks, code)
    ws = None
    if nbytes > 0:
        ws = offsets.new_empty(-(-nbytes // 4))
    rc = lib.tsc_window_attention(
        q.data_ptr(), q_row, q_head, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head,
        offsets.data_ptr(), offsets_k.data_ptr(), samples, n_q, n_k, hq, hk, dim, left, right,
        sinks, max(dim, 1) ** -0.5 if scale is None else scale, code,
        None if ws is None else ws.data_ptr(), nbytes, out.data_ptr(), L.stream_of(q))
    if rc:
        L.check(rc, what)
    return out


# ----------------------------------------------------------------- modules
class VoxelOrder(NamedTuple):
    """Rows in serial order: sample b's are offsets[b] to offsets[b+1] (int32
    on the GPU); ``rows`` are the rows they had before, ``indices`` the
    coordinate tensor in that order."""
    offsets: torch.Tensor
    rows: torch.Tensor
    indices: torch.Tensor


def _spread(v: torch.Tensor) -> torch.Tensor:
    """Bits 0..15 of ``v`` at every third place."""
    for shift, mask in ((16, 0xFF0000FF), (8, 0xF00F00F00F), (4, 0xC30C30C30C3),
                        (2, 0x249249249249)):
        v = (v | (v << shift)) & mask
    return v


class SerialOrder(SparseModule):
    """Puts the rows into Z-order, sample after sample, so that rows near in
    the sequence are near in space and a window over the sequence is a
    neighbourhood.

    The output has its own ``indice_dict``: row numbers that layers before it
    stored do not hold for the new rows.  It keeps the order there under
    ``order_key`` for the VoxelBlocks behind it."""

    def __init__(self, order_key: str):
        super().__init__()
        self.order_key = order_key

    def forward(self, x: SparseConvTensor) -> SparseConvTensor:
        if max(x.spatial_shape) > 1 << 16:
            raise ValueError(f"SerialOrder: {list(x.spatial_shape)} has an axis over 65536 cells")
        if x.batch_size > (1 << 15) - 1:  # with 48 bits of a cell a key fills 63
            raise ValueError(f"SerialOrder: over 32767 samples ({x.batch_size})")
        b, zc, yc, xc = (c.long() for c in x.indices.unbind(1))
        key = (b << 48) | (_spread(zc) << 2) | (_spread(yc) << 1) | _spread(xc)
        key, rows = torch.sort(key, stable=True)
        edges = torch.arange(x.batch_size + 1, device=key.device) << 48
        offsets = torch.searchsorted(key, edges).to(torch.int32)
        indices = x.indices[rows]
        order = VoxelOrder(offsets, rows, indices)
        return SparseConvTensor(x.features[rows], indices, x.spatial_shape, x.batch_size,
                                indice_dict={self.order_key: order})


_ACT_MODULES = {None: lambda v: v, "none": lambda v: v, "relu": F.relu, "gelu": F.gelu,
                "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"), "silu": F.silu}


def _project(m: nn.Module, x: torch.Tensor, activation: Optional[str] = None,
             residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(m(x)) + residual: one launch where ``m`` is an nn.Linear as it is;
    a subclass, a module in its place or one with hooks runs by itself."""
    if type(m) is nn.Linear and _plain(m):
        return linear_act(x, m.weight, m.bias, activation, residual)
    v = _ACT_MODULES[activation](m(x))
    return v if residual is None else v + residual


class VoxelBlock(SparseModule):
    """A transformer block over the voxels of each sample, in the order that a
    SerialOrder with the same ``order_key`` left them:

        x + proj(attention(norm(x))),  then  x + down(act(up(norm(x))))

    Queries and keys are normalised per head and rotated by the voxel's
    (z, y, x); the attention sees ``window`` rows on either side and the first
    ``sinks`` of the sample.  kv_heads (default: heads) shares key heads.

    With a VoxelCache, as ``block(x, cache, layer)``, the tensor's voxels are the
    new ones of a stream: they go behind what their samples keep in that layer
    of the cache (which ``cache.extend`` has made room for), and the attention
    runs over all of it."""

    def __init__(self, channels: int, heads: int, order_key: str, kv_heads: Optional[int] = None,
                 window: Tuple[Optional[int], Optional[int]] = (None, None), sinks: int = 0,
                 hidden: Optional[int] = None, activation: str = "gelu", base: float = 100.0,
                 eps: float = 1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if channels % heads or heads % kv_heads:
            raise ValueError(f"VoxelBlock: {channels} channels, {heads} heads, {kv_heads} key "
                             "heads do not divide evenly")
        self.heads, self.kv_heads, self.dim = heads, kv_heads, channels // heads
        self.order_key, self.window, self.sinks = order_key, window, sinks
        self.activation, self.base, self.eps = activation, base, eps
        hidden = 4 * channels if hidden is None else hidden
        self.norm1, self.norm2 = nn.LayerNorm(channels), nn.LayerNorm(channels)
        self.qkv = nn.Linear(channels, (heads + 2 * kv_heads) * self.dim)
        self.q_gain = nn.Parameter(torch.ones(self.dim))
        self.k_gain = nn.Parameter(torch.ones(self.dim))
        self.proj = nn.Linear(channels, channels)
        self.up, self.down = nn.Linear(channels, hidden), nn.Linear(hidden, channels)

    def _computes_in(self, dtype: torch.dtype) -> bool:
        """Whether the kernels take ``dtype`` and the layers' weights have it."""
        if compute_dtype(dtype, dtype) is not dtype:
            return False
        layers = self._modules
        for name in ("norm1", "qkv", "proj", "norm2", "up", "down"):
            w = layers[name]._parameters.get("weight")
            if w is not None and w.dtype is not dtype:
                return False
        return True

    def forward(self, x: SparseConvTensor, cache: Optional["VoxelCache"] = None,
                layer: int = 0) -> SparseConvTensor:
        order = x.indice_dict.get(self.order_key)
        if not isinstance(order, VoxelOrder):
            raise KeyError(f"order_key '{self.order_key}' not found in indice_dict. "
                           "A SerialOrder with that key must run before VoxelBlock.")
        if x.indices is not order.indices:
            raise ValueError(f"VoxelBlock: the rows are not those that SerialOrder "
                             f"'{self.order_key}' ordered (a layer since then changed the "
                             "coordinates); run a SerialOrder on them first")
        if cache is not None and cache.samples != x.batch_size:
            raise ValueError(f"VoxelBlock: {x.batch_size} samples, the cache has {cache.samples}")
        f = x.features
        if not self._computes_in(f.dtype):
            # on f32 copies, as the convolutions do
            wide = {n: p.float() for n, p in self.named_parameters() if p.is_floating_point()}
            y = torch.func.functional_call(self, wide, (x.replace_feature(f.float()), cache, layer))
            return x.replace_feature(y.features.to(f.dtype))
        with torch.no_grad():
            hq, hk = self.heads, self.kv_heads
            qkv = _project(self.qkv, self.norm1(f))
            qkv = qkv.reshape(f.shape[0], hq + 2 * hk, self.dim)
            q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
            coords = x.indices[:, 1:]
            if cache is None:
                q, k = norm_rotate_heads(q, k, coords, self.q_gain, self.k_gain, self.eps, self.base)
                a = window_attention(q, k, v, order.offsets, window=self.window, sinks=self.sinks)
            else:
                q = cache.append(layer, q, k, v, coords, order.offsets, self.q_gain, self.k_gain,
                                 self.eps, self.base)
                a = cache.attend(layer, q, order.offsets, self.window, self.sinks)
            f = _project(self.proj, a.view(f.shape), residual=f)
            h = _project(self.up, self.norm2(f), self.activation)
            f = _project(self.down, h, residual=f)
        return x.replace_feature(f)
