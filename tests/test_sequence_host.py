"""The voxel-block operators' checks that need no GPU: argument errors of the
C entries (nothing is launched), CPU tensors, module parameters."""
import io

import pytest
import torch

import trispconv.pytorch as spconv
from trispconv_amd import _lib as L


def _refused(rc, words):
    assert rc == 1 and words in L.lib().tsc_last_error(), L.lib().tsc_last_error()


def test_linear_entry_refuses():
    f = L.lib().tsc_linear_act
    _refused(f(16, 8, 16, 8, None, 0, None, 0, 7, 1, 8, 8, 0, 16, None), b"dtype")
    _refused(f(16, 8, 16, 8, None, 9, None, 0, 1, 1, 8, 8, 0, 16, None), b"dtype")
    _refused(f(16, 8, 16, 8, None, 0, None, 0, 1, -1, 8, 8, 0, 16, None), b"sizes")
    _refused(f(16, 8, 16, 8, None, 0, None, 0, 1, 1, 8, 1 << 24, 0, 16, None), b"sizes")
    _refused(f(16, 8, 16, 8, None, 0, None, 0, 1, 1, 8, 8, 5, 16, None), b"activation")
    _refused(f(None, 8, 16, 8, None, 0, None, 0, 1, 1, 8, 8, 0, 16, None), b"null")
    _refused(f(16, 8, 16, 8, None, 0, None, 0, 1, 1, 8, 8, 0, None, None), b"null")
    _refused(f(16, -8, 16, 8, None, 0, None, 0, 1, 1, 8, 8, 0, 16, None), b"stride")
    _refused(f(16, 1 << 21, 16, 8, None, 0, None, 0, 1, 9, 8, 8, 0, 16, None), b"strides over")
    assert f(None, 0, None, 0, None, 0, None, 0, 1, 0, 8, 8, 0, None, None) == 0  # no rows


def test_rotate_entry_refuses():
    f = L.lib().tsc_norm_rotate_heads

    def call(dtype=1, n=4, hq=2, hk=2, dim=16, axes=3, base=100.0, eps=1e-6, pos=16, out=16):
        return f(16, 32, 16, 16, 32, 16, pos, 3, 0, axes, None, None, 0, 0, 0, eps, base, 0, dtype,
                 n, hq, hk, dim, out, out, None)

    _refused(call(dtype=3), b"dtype")
    _refused(call(n=-1), b"sizes")
    _refused(call(dim=15), b"even number")
    _refused(call(dim=258), b"even number")
    _refused(call(axes=0), b"axes")
    _refused(call(axes=5), b"axes")
    _refused(call(base=1.0), b"base")
    _refused(call(base=float("nan")), b"base")
    _refused(call(eps=-1.0), b"eps")
    _refused(call(pos=None), b"null")
    _refused(call(out=None), b"null")
    assert call(n=0, pos=None, out=None) == 0


def test_attention_entry_refuses():
    lib = L.lib()

    def call(dtype=1, samples=1, n_q=8, n_k=8, hq=4, hk=2, dim=16, sinks=0, scale=1.0, q=16,
             off=16, ws=None, ws_bytes=0):
        return lib.tsc_window_attention(q, 64, 16, 16, 32, 16, 16, 32, 16, off, off, samples, n_q,
                                        n_k, hq, hk, dim, -1, -1, sinks, scale, dtype, ws,
                                        ws_bytes, 16, None)

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
    # few rows over many keys: split, with scratch
    need = lib.tsc_window_attention_workspace_bytes(1, 1, 50_000, 4, 2, 64, -1, -1, 0, 1)
    assert need >= 2 * 4 * 66 * 4
    _refused(call(n_q=1, n_k=50_000, dim=64), b"workspace")
    _refused(call(n_q=1, n_k=50_000, dim=64, ws=16, ws_bytes=need - 1), b"workspace")
    # enough rows for every CU: not split
    assert lib.tsc_window_attention_workspace_bytes(4, 200_000, 200_000, 4, 4, 64, 512, 512, 0,
                                                    1) == 0
    assert lib.tsc_window_attention_workspace_bytes(1, 1, 1, 4, 4, 500, -1, -1, 0, 1) == -1
    assert call(n_q=0, q=None) == 0 and call(samples=0, off=None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 16)
    off = torch.tensor([0, 4], dtype=torch.int32)
    for go in (lambda: spconv.linear_act(x[:, 0], x[:, 1]),
               lambda: spconv.norm_rotate_heads(x, x, torch.zeros(4, 3)),
               lambda: spconv.window_attention(x, x, x, off)):
        with pytest.raises(RuntimeError, match="GPU"):
            go()


def test_block_parameters_and_state():
    m = spconv.VoxelBlock(48, 6, "o", kv_heads=2, window=(7, None), hidden=100)
    assert m.qkv.weight.shape == ((6 + 4) * 8, 48) and m.dim == 8
    assert m.up.weight.shape == (100, 48) and m.down.weight.shape == (48, 100)
    assert m.q_gain.shape == (8,) and spconv.VoxelBlock(48, 6, "o").up.out_features == 192
    buf = io.BytesIO()
    torch.save(m.state_dict(), buf)
    buf.seek(0)
    n = spconv.VoxelBlock(48, 6, "o", kv_heads=2, hidden=100)
    n.load_state_dict(torch.load(buf, weights_only=True))
    assert torch.equal(n.proj.weight, m.proj.weight)
    with pytest.raises(ValueError, match="divide"):
        spconv.VoxelBlock(48, 5, "o")
    x = spconv.SparseConvTensor(torch.zeros(3, 48), torch.zeros(3, 4, dtype=torch.int32), [4, 4, 4], 1)
    with pytest.raises(KeyError, match="SerialOrder"):
        m(x)


def test_serial_order_sorts_by_sample_and_interleaved_bits():
    """Runs on any device: torch's own sort."""
    idx = torch.tensor([[1, 0, 0, 0], [0, 1, 0, 0], [0, 0, 1, 0], [0, 0, 0, 1], [0, 2, 0, 0],
                        [0, 1, 1, 1]], dtype=torch.int32)
    x = spconv.SparseConvTensor(torch.arange(6.0)[:, None], idx, [4, 4, 4], 3)
    y = spconv.SerialOrder("o")(x)
    assert y.features.flatten().tolist() == [3.0, 2.0, 1.0, 5.0, 4.0, 0.0]
    assert y.indice_dict["o"].offsets.tolist() == [0, 5, 6, 6]


@pytest.mark.parametrize("samples,n_q,n_k", [(1, 0, 0), (3, 0, 10), (0, 0, 0), (0, 5, 5), (1, 5, 0)])
def test_attention_of_nothing_needs_no_scratch(samples, n_q, n_k):
    assert L.lib().tsc_window_attention_workspace_bytes(samples, n_q, n_k, 4, 2, 16, -1, -1, 0, 1) == 0
