"""Streams of voxels: keys and values kept in pages from step to step.

A stream brings a sample's voxels in steps (sweeps of a scan, what a generator
has drawn so far); the blocks' attention sees the new rows and everything the
sample keeps.  Two operators work on pages of rows (no counterpart in the
reference; inference, as everything here):

``norm_rotate_append``  norm_rotate_heads, with the keys and the values written
                        to the pages of their samples
``cache_attention``     window_attention over those pages; pages that all
                        samples begin with are read once for all

``VoxelCache`` holds the pages of a network's blocks, hands them out and shares
them; a VoxelBlock called with one streams.
"""
from __future__ import annotations

from operator import index
from typing import Callable, List, Optional, Sequence, Tuple, Union

import torch

from .. import _lib as L
from .sequence import _head_gains, _limit, _MOST, _position_rows, _rows_of, _same

__all__ = ["norm_rotate_append", "cache_attention", "VoxelCache"]


def _launch(device: int, call: Callable, *args) -> int:
    """``call`` with ``device`` as the current one, as launches on its streams need."""
    if torch.cuda.current_device() == device:
        return call(*args)
    with torch.cuda.device(device):
        return call(*args)


def _check_pages(what: str, like: torch.Tensor, dim: int, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, table: torch.Tensor, offsets: torch.Tensor,
                 lengths: torch.Tensor):
    """Pages and tables beside ``like`` (..., dim), whose device they have to be
    on: the pages' shape and strides, and the table's shape.  A call of few rows
    takes the host longer than the GPU, so each attribute is asked for once (appending
    one row of four samples: 13.5 us, asked for wherever it is used 16.7)."""
    shape, samples_entries = k_pages.shape, table.shape
    if len(shape) != 4 or v_pages.shape != shape or shape[3] != dim:
        raise ValueError(f"{what}: pages {tuple(shape)} and {tuple(v_pages.shape)} are not "
                         f"(pages, rows, heads, {dim})")
    dtype, device = like.dtype, like.get_device()
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if t.dtype is not dtype or t.get_device() != device:
            _same(t, like, what, name)
    k_strides, v_strides = k_pages.stride(), v_pages.stride()
    if dim > 1 and (k_strides[3] != 1 or v_strides[3] != 1):
        raise ValueError(f"{what}: the values of a head must lie one behind the other in the pages")
    if len(samples_entries) != 2 or lengths.shape != samples_entries[:1] or \
            offsets.shape != (samples_entries[0] + 1,):
        raise ValueError(f"{what}: table {tuple(table.shape)}, offsets {tuple(offsets.shape)} and "
                         f"lengths {tuple(lengths.shape)} are not (B, pages), (B + 1,) and (B,)")
    for t in (table, offsets, lengths):
        if t.dtype is not torch.int32 or t.get_device() != device:
            raise ValueError(f"{what}: table, offsets and lengths must be int32 on {like.device}, "
                             f"got {t.dtype} on {t.device}")
    return shape, k_strides[:3], v_strides[:3], samples_entries


def norm_rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                       k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                       offsets: torch.Tensor, lengths: torch.Tensor,
                       q_weight: Optional[torch.Tensor] = None,
                       k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                       base: float = 10000.0, interleaved: bool = False) -> torch.Tensor:
    """norm_rotate_heads whose keys, and the values beside them, go to pages.

    q (N, Hq, D), k and v (N, Hk, D) and the arguments of the norm and the
    rotation as in ``norm_rotate_heads``; returns the queries as it does.
    k_pages and v_pages (P, R, Hk, D), R rows a page, any strides with D
    contiguous, are written in place: sample b's new rows are rows offsets[b]
    to offsets[b+1], the last of its lengths[b] positions, and position t is row
    t % R of page table[b, t // R].  offsets (B + 1,), lengths (B,) and table
    (B, pages) are int32 on the GPU.  Nothing else in the pages is written; a row
    of no sample, or one whose position or page there is not, is written nowhere
    (with a length over the table's room those that are past it).
    No row of a page may be that of two new rows, and no input may lie in the pages.
    """
    what = "norm_rotate_append"
    if not q.is_cuda:
        L.require_gpu(q, what)
    code = L.dtype_code(q.dtype)
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 3 or len(k_shape) != 3 or k_shape != v.shape or \
            q_shape[0] != k_shape[0] or q_shape[2] != k_shape[2]:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} are "
                         "not (N, Hq, D), (N, Hk, D), (N, Hk, D)")
    _same(k, q, what, "k")
    _same(v, q, what, "v")
    n, hq, dim = q_shape
    hk = k_shape[1]
    (pages, rows, heads, _), k_at, v_at, (samples, entries) = \
        _check_pages(what, q, dim, k_pages, v_pages, table, offsets, lengths)
    if heads != hk:
        raise ValueError(f"{what}: {hk} key heads, the pages have {heads}")
    for at, name in ((k_at, "k_pages"), (v_at, "v_pages")):
        if 0 in at and any(s == 0 and e > 1 for s, e in zip(at, (pages, rows, heads))):
            raise ValueError(f"{what}: {name} is expanded: its rows share memory")
    positions, axes, p_row, in_f32 = _position_rows(positions, q, n, what)
    q_weight, k_weight, gains = _head_gains(q_weight, k_weight, q, hq, hk, dim, what)
    (q, (q_row, q_head, _)), (k, (k_row, k_head, _)) = _rows_of(q), _rows_of(k)
    (v, (v_row, v_head, _)), (table, (t_row, _)) = _rows_of(v), _rows_of(table)
    offsets, lengths = offsets.contiguous(), lengths.contiguous()
    q_out = q.new_empty(n, hq, dim)
    rc = _launch(
        q.get_device(), L.lib().tsc_norm_rotate_append, q.data_ptr(), q_row, q_head, k.data_ptr(),
        k_row, k_head, v.data_ptr(), v_row, v_head, positions.data_ptr(), p_row, in_f32,
        axes, *gains, eps, base, interleaved, code, n, hq, hk, dim, k_pages.data_ptr(), *k_at,
        v_pages.data_ptr(), *v_at, pages, rows, table.data_ptr(), t_row, entries,
        offsets.data_ptr(), lengths.data_ptr(), samples, q_out.data_ptr(), L.stream_of(q))
    if rc:
        L.check(rc, what)
    return q_out


def cache_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    table: torch.Tensor, offsets: torch.Tensor, lengths: torch.Tensor,
                    prefix: Optional[torch.Tensor] = None,
                    window: Tuple[Optional[int], Optional[int]] = (None, None), sinks: int = 0,
                    scale: Optional[float] = None) -> torch.Tensor:
    """window_attention of new rows over what their samples keep in pages.

    q (Nq, Hq, D), the pages, table, offsets and lengths as in
    ``norm_rotate_append``, Hq a multiple of the pages' heads, D at most 256:
    query i of a sample's Lq stands at p = i + lengths[b] - Lq and sees of its
    positions what ``window_attention`` with the same window, sinks and scale
    would let it see.  Which pages a table names beyond a sample's length, and
    what they hold, means nothing.  prefix (int32 on the GPU, page numbers):
    every sample's first positions lie in these pages; they are then read once
    for the queries of all samples, and the table's entries for them not at all.
    A query that sees no key gives zeros, as rows outside every sample do.  Lengths
    over the table's room, and negative ones, are cut before anything else.

    Scores, maxima and sums are float32.  For float16 and bfloat16 the softmax
    weights are rounded to that type for the product with the values where a
    sample has over 64 rows (queries times Hq / heads) in the mean, and for a
    prefix of over 64 such rows in all; with fewer they go into it as two values
    of the type.  The same step may therefore differ in its last bits with and
    without ``prefix``.
    """
    what = "cache_attention"
    if not q.is_cuda:
        L.require_gpu(q, what)
    code = L.dtype_code(q.dtype)
    q_shape = q.shape
    if len(q_shape) != 3:
        raise ValueError(f"{what}: q {tuple(q_shape)} is not (Nq, Hq, D)")
    n_q, hq, dim = q_shape
    (pages, rows, hk, _), k_at, v_at, (samples, entries) = \
        _check_pages(what, q, dim, k_pages, v_pages, table, offsets, lengths)
    p_ptr, p_pages = None, 0
    if prefix is not None:
        if prefix.dim() != 1 or prefix.dtype is not torch.int32 or \
                prefix.get_device() != q.get_device() or prefix.shape[0] > entries:
            raise ValueError(f"{what}: prefix must be up to {entries} page numbers, int32 on "
                             f"{q.device}, got {tuple(prefix.shape)} {prefix.dtype} on "
                             f"{prefix.device}")
        prefix = prefix.contiguous()
        p_ptr, p_pages = prefix.data_ptr(), prefix.shape[0]
    left, right = window
    left, right = _limit(left, what), _limit(right, what)
    if sinks < 0:
        raise ValueError(f"{what}: sinks must not be negative, got {sinks}")
    (q, (q_row, q_head, _)), (table, (t_row, _)) = _rows_of(q), _rows_of(table)
    offsets, lengths = offsets.contiguous(), lengths.contiguous()
    if samples == 0:
        return q.new_zeros((n_q, hq, dim))
    out = q.new_empty(n_q, hq, dim)
    lib, sinks = L.lib(), min(sinks, _MOST)
    nbytes = lib.tsc_cache_attention_workspace_bytes(samples, n_q, entries * rows, p_pages * rows,
                                                     hq, hk, dim, left, right, sinks, code)
    ws = None
    if nbytes > 0:
        ws = offsets.new_empty(-(-nbytes // 4))
    rc = _launch(
        q.get_device(), lib.tsc_cache_attention, q.data_ptr(), q_row, q_head, k_pages.data_ptr(),
        *k_at, v_pages.data_ptr(), *v_at, pages, rows, table.data_ptr(), t_row, entries,
        offsets.data_ptr(), lengths.data_ptr(), samples, p_ptr, p_pages, n_q, hq, hk, dim, left,
        right, sinks, max(dim, 1) ** -0.5 if scale is None else scale, code,
        None if ws is None else ws.data_ptr(), nbytes, out.data_ptr(), L.stream_of(q))
    if rc:
        L.check(rc, what)
    return out


class VoxelCache:
    """What the samples of a stream keep: pages of ``page_rows`` rows for the keys
    and the values of every layer, and which of them each sample has.

    ``positions`` is the most rows that one sample may keep, ``pages`` how many
    there are for all samples (default: enough for all to keep that many).  Every
    layer has pages of its own under the same numbers: ``k[layer]`` and
    ``v[layer]`` (pages, page_rows, kv_heads, dim).  ``lengths`` (samples,) and
    ``table`` (samples, pages of a sample) are int32 on the device and keep their
    memory, so that a captured step finds there what later steps have changed.

    A step takes room for its new rows (``extend``), then runs the blocks with
    the cache: ``block(x, cache, layer)``.
    """

    def __init__(self, samples: int, positions: int, kv_heads: int, dim: int, layers: int = 1,
                 pages: Optional[int] = None, page_rows: int = 64,
                 dtype: torch.dtype = torch.float32,
                 device: Union[str, torch.device] = "cuda"):
        if min(samples, kv_heads, dim, layers) < 1 or positions < 0 or \
                not 1 <= page_rows <= 1 << 20:
            raise ValueError("VoxelCache: samples, kv_heads, dim and layers must be 1 or more, "
                             "page_rows 1 to 2^20")
        L.dtype_code(dtype)
        self.samples, self.positions, self.page_rows = samples, positions, page_rows
        entries = max(1, -(-positions // page_rows))
        pages = samples * entries if pages is None else pages
        if pages < 0:
            raise ValueError(f"VoxelCache: {pages} pages")
        # the rows of a head lie together in a page
        shape = (layers, pages, kv_heads, page_rows, dim)
        self.k, self.v = (list(torch.empty(shape, dtype=dtype, device=device).transpose(2, 3))
                          for _ in range(2))
        self.table = torch.zeros(samples, entries, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(samples, dtype=torch.int32, device=device)
        self._entries = torch.zeros(samples, entries, dtype=torch.int32)
        self._kept = [0] * samples
        self._pages: List[List[int]] = [[] for _ in range(samples)]
        self._users = [0] * pages
        self._free = list(range(pages - 1, -1, -1))
        self._used = 0           # the longest row of the table
        self._first = None       # a sample that keeps something
        self._common = 0         # pages that all those begin with

    def _give(self, b: int, pages: List[int]) -> None:
        """Appends pages to sample b's."""
        at = len(self._pages[b])
        self._entries[b, at:at + len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self._pages[b] = self._pages[b] + pages

    def _publish(self, pages: bool, samples: bool) -> None:
        """The host's state to the device; whether a sample's pages have changed, and
        whether they can begin differently now (new pages at an end cannot)."""
        if pages:
            self.table.copy_(self._entries)
            self._used = max(len(p) for p in self._pages)
        if samples:
            held = [b for b, p in enumerate(self._pages) if p]
            self._first, self._common = (held[0] if held else None), 0
            if len(held) > 1:
                first, *others = (self._pages[b] for b in held)
                n = min(len(p) for p in (first, *others))
                for p in others:
                    n = next((i for i in range(n) if p[i] != first[i]), n)
                self._common = n
        kept = torch.tensor(self._kept, dtype=torch.int32)
        if self.lengths.is_cuda:
            self.lengths.copy_(kept.pin_memory(), non_blocking=True)
        else:
            self.lengths.copy_(kept)

    def _capturing(self) -> bool:
        return self.table.is_cuda and torch.cuda.is_current_stream_capturing()

    def _check_steps(self) -> None:
        if self._capturing():
            raise RuntimeError("VoxelCache: rows are given and dropped between the replays of a "
                               "captured step, not in it")

    def _check_samples(self, samples: Sequence[int]) -> List[int]:
        samples = [index(b) for b in samples]
        if any(not 0 <= b < self.samples for b in samples):
            raise ValueError(f"VoxelCache: samples {samples}, there are {self.samples}")
        return samples

    def rows(self) -> List[int]:
        """The rows that each sample keeps."""
        return list(self._kept)

    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, rows: Union[Sequence[int], torch.Tensor]) -> None:
        """Room for ``rows[b]`` new rows behind what sample b keeps, for instance
        ``order.offsets.diff()``.  A ValueError leaves everything as it was."""
        self._check_steps()
        rows = rows.tolist() if isinstance(rows, torch.Tensor) else list(rows)
        new_rows = [int(n) for n in rows]
        if len(rows) != self.samples or any(n < 0 or n != r for n, r in zip(new_rows, rows)):
            raise ValueError(f"VoxelCache: {rows} new rows for {self.samples} samples")
        kept = [a + b for a, b in zip(self._kept, new_rows)]
        if max(kept) > self.positions:
            raise ValueError(f"VoxelCache: {max(kept)} rows of a sample, it has room for "
                             f"{self.positions}")
        need = [-(-n // self.page_rows) - len(p) for n, p in zip(kept, self._pages)]
        if sum(need) > len(self._free):
            raise ValueError(f"VoxelCache: {sum(need)} pages are needed, {len(self._free)} are free")
        new = any(n and not p for n, p in zip(need, self._pages))
        for b, n in enumerate(need):
            if n:
                pages = [self._free.pop() for _ in range(n)]
                for page in pages:
                    self._users[page] = 1
                self._give(b, pages)
        self._kept = kept
        self._publish(sum(need) > 0, new)

    def share(self, source: int, targets: Sequence[int], rows: int) -> None:
        """Lets samples that keep nothing begin with the first ``rows`` rows of
        ``source``, in the same pages: whole pages, so a multiple of page_rows.

        Pages that all samples share are read once for all of them.  With over 64
        rows of queries and heads that share a key head they are read whole, though
        a window sees less of them: one row each of 64 samples behind 32,768 shared
        ones takes 45 us, from unshared pages 160; in a window of 4096 45, unshared 31
        (16 heads on 4 of 64, bf16)."""
        self._check_steps()
        source, *targets = self._check_samples([source, *targets])
        rows = index(rows)
        if rows % self.page_rows or not 0 <= rows <= self._kept[source]:
            raise ValueError(f"VoxelCache: {rows} rows of sample {source}, which keeps "
                             f"{self._kept[source]}, are not whole pages of {self.page_rows}")
        if len(set(targets)) < len(targets) or any(self._kept[b] for b in targets):
            raise ValueError(f"VoxelCache: samples {targets} must be different and keep nothing")
        pages = self._pages[source][:rows // self.page_rows]
        for page in pages:
            self._users[page] += len(targets)
        for b in targets:
            self._give(b, pages)
            self._kept[b] = rows
        self._publish(True, True)

    def drop(self, samples: Sequence[int]) -> None:
        """Forgets what these samples keep; pages that no other sample has are free again."""
        self._check_steps()
        for b in self._check_samples(samples):
            for page in reversed(self._pages[b]):
                self._users[page] -= 1
                if not self._users[page]:
                    self._free.append(page)
            self._pages[b], self._kept[b] = [], 0
        self._publish(True, True)

    def _tables(self) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """The table as far as it is used, and the pages that all samples begin
        with; a captured step takes the whole table, which later steps fill."""
        if self._capturing():
            return self.table, None
        table = self.table[:, :self._used]
        return table, self.table[self._first, :self._common] if self._common else None

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               positions: torch.Tensor, offsets: torch.Tensor,
               q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-6, base: float = 10000.0, interleaved: bool = False) -> torch.Tensor:
        """``norm_rotate_append`` to a layer's pages: the rows that the last ``extend`` made
        room for, sample after sample."""
        return norm_rotate_append(q, k, v, positions, self.k[layer], self.v[layer],
                                  self._tables()[0], offsets, self.lengths, q_weight, k_weight,
                                  eps, base, interleaved)

    def attend(self, layer: int, q: torch.Tensor, offsets: torch.Tensor,
               window: Tuple[Optional[int], Optional[int]] = (None, None), sinks: int = 0,
               scale: Optional[float] = None) -> torch.Tensor:
        """``cache_attention`` over a layer's pages."""
        table, prefix = self._tables()
        return cache_attention(q, self.k[layer], self.v[layer], table, offsets, self.lengths,
                               prefix, window, sinks, scale)
