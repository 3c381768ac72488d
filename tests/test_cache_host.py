"""Pages of a stream: what needs no GPU.  Refusals of the C entries (nothing is
launched), the host's bookkeeping of VoxelCache."""
import pytest
import torch

import trispconv.pytorch as spconv
from trispconv_amd import _lib as L


def _refused(rc, words):
    assert rc == 1 and words in L.lib().tsc_last_error(), L.lib().tsc_last_error()


def test_append_entry_refuses():
    f = L.lib().tsc_norm_rotate_append

    def call(dtype=1, n=4, hq=2, hk=2, dim=16, axes=3, base=100.0, eps=1e-6, pos=16, out=16, pages=4,
             rows=8, table=16, entries=2, off=16, lengths=16, samples=1, v=16, k_pages=16):
        return f(16, 32, 16, 16, 32, 16, v, 32, 16, pos, 3, 0, axes, None, None, 0, 0, 0, eps, base, 0,
                 dtype, n, hq, hk, dim, k_pages, 256, 32, 16, 16, 256, 32, 16, pages, rows, table, 2,
                 entries, off, lengths, samples, out, None)

    _refused(call(dtype=3), b"dtype")
    _refused(call(n=-1), b"sizes")
    _refused(call(dim=15), b"even number")
    _refused(call(axes=5), b"axes")
    _refused(call(base=1.0), b"base")
    _refused(call(eps=-1.0), b"eps")
    _refused(call(pos=None), b"null")
    _refused(call(out=None), b"null")
    _refused(call(off=None), b"null")
    _refused(call(v=None), b"null")
    _refused(call(k_pages=None), b"null")
    _refused(call(table=None), b"null")
    _refused(call(lengths=None), b"null")
    _refused(call(samples=-1), b"samples")
    _refused(call(pages=-1), b"pages")
    _refused(call(pages=1 << 31), b"pages")
    _refused(call(rows=0), b"rows")
    _refused(call(rows=(1 << 20) + 1), b"rows")
    _refused(call(rows=64, entries=1 << 25), b"positions")
    assert call(n=0, pos=None, out=None) == 0


def test_attention_entry_refuses():
    lib = L.lib()

    def call(dtype=1, n_q=8, hq=4, hk=2, dim=16, sinks=0, scale=1.0, q=16, off=16, pages=4, rows=8,
             table=16, entries=2, lengths=16, samples=1, prefix=None, p_pages=0, k_pages=16, ws=None,
             ws_bytes=0):
        return lib.tsc_cache_attention(q, 64, 16, k_pages, 256, 32, 16, 16, 256, 32, 16, pages, rows,
                                       table, 2, entries, off, lengths, samples, prefix, p_pages, n_q,
                                       hq, hk, dim, -1, -1, sinks, scale, dtype, ws, ws_bytes, 16, None)

    _refused(call(dtype=5), b"dtype")
    _refused(call(n_q=-1), b"sizes")
    _refused(call(hq=3), b"evenly")
    _refused(call(hk=0), b"evenly")
    _refused(call(dim=0), b"head size")
    _refused(call(dim=257), b"head size")
    _refused(call(sinks=-1), b"sinks")
    _refused(call(scale=float("inf")), b"finite")
    _refused(call(q=None), b"null")
    _refused(call(off=None), b"null")
    _refused(call(table=None), b"null")
    _refused(call(lengths=None), b"null")
    _refused(call(k_pages=None), b"null")
    _refused(call(p_pages=1), b"null")
    _refused(call(p_pages=3, prefix=16), b"prefix")
    _refused(call(p_pages=-1, prefix=16), b"prefix")
    _refused(call(rows=0), b"rows")
    _refused(call(entries=1 << 28), b"positions")
    _refused(call(n_q=(1 << 31) - 1, hq=8, hk=2), b"rows of queries")
    assert call(n_q=0, q=None) == 0 and call(samples=0, off=None, table=None, lengths=None) == 0


def test_workspace_query():
    f = L.lib().tsc_cache_attention_workspace_bytes
    assert f(1, 1, 1, 0, 4, 4, 500, -1, -1, 0, 1) == -1
    assert f(1, 1, 1, 0, 4, 4, 64, -1, -1, 0, 7) == -1
    assert f(0, 0, 0, 0, 4, 4, 64, -1, -1, 0, 1) == 0
    assert f(4, 0, 1 << 20, 0, 4, 4, 64, -1, -1, 0, 1) == 0


def test_cpu_tensors_are_refused():
    q, pages = torch.zeros(4, 2, 16), torch.zeros(1, 8, 2, 16)
    table, off, n = (torch.zeros(s, dtype=torch.int32) for s in ((1, 1), (2,), (1,)))
    with pytest.raises(RuntimeError, match="GPU"):
        spconv.norm_rotate_append(q, q, q, torch.zeros(4, 3), pages, pages, table, off, n)
    with pytest.raises(RuntimeError, match="GPU"):
        spconv.cache_attention(q, pages, pages, table, off, n)


def _cache(**more):
    return spconv.VoxelCache(**{**dict(samples=3, positions=40, kv_heads=2, dim=8, layers=2, pages=8,
                                       page_rows=8, device="cpu"), **more})


def _entries(c, b):
    return c.table[b, :-(-int(c.lengths[b]) // c.page_rows)].tolist()


def test_cache_shapes():
    c = _cache(dtype=torch.float16)
    assert len(c.k) == len(c.v) == 2 and c.k[1].shape == (8, 8, 2, 8) and c.v[0].dtype == torch.float16
    assert c.k[0].stride()[3] == 1 and c.k[0].stride(1) == 8  # a head's rows lie together
    assert c.table.shape == (3, 5) and c.lengths.tolist() == [0, 0, 0]
    assert _cache(pages=None).k[0].shape[0] == 15
    for bad in (dict(samples=0), dict(dim=0), dict(page_rows=0), dict(positions=-1), dict(pages=-1)):
        with pytest.raises(ValueError):
            _cache(**bad)
    with pytest.raises(TypeError):
        _cache(dtype=torch.float64)


def test_cache_extend():
    c = _cache()
    memory = c.table.data_ptr(), c.lengths.data_ptr()
    c.extend([8, 0, 9])
    assert c.rows() == [8, 0, 9] == c.lengths.tolist() and c.free_pages() == 5
    c.extend(torch.tensor([1, 1, 0]))
    assert c.rows() == [9, 1, 9] and c.free_pages() == 3
    used = sum((_entries(c, b) for b in range(3)), [])
    assert len(set(used)) == len(used) == 5 and all(0 <= p < 8 for p in used)
    before = c.table.clone(), c.lengths.clone()
    for bad in ([0, 0, 32], [32, 0, 0], [8, 8, 16], [1, 2], [-1, 0, 0]):
        with pytest.raises(ValueError):
            c.extend(bad)
        assert torch.equal(c.table, before[0]) and torch.equal(c.lengths, before[1])
        assert c.free_pages() == 3 and c.rows() == [9, 1, 9]
    assert (c.table.data_ptr(), c.lengths.data_ptr()) == memory


def test_cache_share_and_drop():
    c = _cache()
    c.extend([20, 0, 0])
    for bad in ((0, [1], 20), (0, [1], 24), (0, [1, 1], 16), (0, [0], 8), (1, [2], 8), (0, [1], -8),
                (0, [2, -1], 8), (0, [3], 8), (-3, [1], 8)):
        with pytest.raises(ValueError):
            c.share(*bad)
    with pytest.raises(ValueError):
        c.drop([0, 3])
    c.share(0, [1, 2], 16)
    assert c.rows() == [20, 16, 16] and c.free_pages() == 5
    assert _entries(c, 1) == _entries(c, 2) == _entries(c, 0)[:2]
    table, prefix = c._tables()
    assert table.shape == (3, 3) and prefix.tolist() == _entries(c, 0)[:2]
    c.extend([0, 1, 1])
    assert c._tables()[1].tolist() == _entries(c, 0)[:2] and c.free_pages() == 3
    assert len({_entries(c, b)[2] for b in range(3)}) == 3
    c.drop([0])
    assert c.rows() == [0, 17, 17] and c.free_pages() == 4  # its shared pages are still used
    assert c._tables()[1].tolist() == _entries(c, 1)[:2]
    c.drop([1])
    assert c._tables()[1] is None and c.free_pages() == 5
    c.drop([2])
    assert c.free_pages() == 8 and c._tables()[0].shape == (3, 0)
    c.extend([40, 24, 0])
    assert c.free_pages() == 0 and c._tables()[1] is None


def test_block_refuses_another_number_of_samples():
    x = spconv.SparseConvTensor(torch.zeros(3, 16), torch.zeros(3, 4, dtype=torch.int32), [4, 4, 4], 1)
    x = spconv.SerialOrder("o")(x)
    with pytest.raises(ValueError, match="samples"):
        spconv.VoxelBlock(16, 2, "o")(x, _cache())
