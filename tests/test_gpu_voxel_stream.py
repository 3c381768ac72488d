"""VoxelBlocks over a stream: steps with a VoxelCache against the same rows at once."""
import copy

import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu
from sequence_oracle import act64, attend64, rotate64
from test_gpu_voxel_block import _input

pytestmark = [pytest.mark.gpu, needs_gpu]


def _blocks(n=2, **more):
    torch.manual_seed(4)
    blocks = [spconv.VoxelBlock(32, 4, "o", kv_heads=2, **{**dict(window=(200, 0), sinks=3), **more})
              for _ in range(n)]
    with torch.no_grad():
        for m in blocks:
            m.k_gain.add_(0.1 * torch.randn(m.dim))
    return blocks


def _cache(**more):
    return spconv.VoxelCache(**{**dict(samples=3, positions=700, kv_heads=2, dim=8, layers=2,
                                       page_rows=16, device=DEV), **more})


def _step(blocks, x, cache):
    x = spconv.SerialOrder("o")(x)
    cache.extend(x.indice_dict["o"].offsets.diff())
    for i, m in enumerate(blocks):
        x = m(x, cache, i)
    return x


def _stream64(blocks, parts):
    """Every part's rows, sample by sample, through the blocks in 64 bits: per
    block all rows of a sample at once, which a causal window allows."""
    out = []
    for b in range(3):
        f = torch.cat([x.features[x.indices[:, 0] == b] for x in parts]).cpu().double()
        idx = torch.cat([x.indices[x.indices[:, 0] == b] for x in parts]).cpu()
        for m in blocks:
            hq, hk, n = m.heads, m.kv_heads, len(f)
            qkv = m.qkv(m.norm1(f)).view(n, hq + 2 * hk, m.dim)
            q, _ = rotate64(qkv[:, :hq], idx[:, 1:], m.q_gain, m.eps, m.base)
            k, _ = rotate64(qkv[:, hq:hq + hk], idx[:, 1:], m.k_gain, m.eps, m.base)
            a, _ = attend64(q.float(), k.float(), qkv[:, hq + hk:].float(), [n], [n], m.window, m.sinks)
            f = f + m.proj(a.reshape(f.shape))
            f = f + m.down(act64(m.up(m.norm2(f)), m.activation))
        out.append(f)
    return out


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.float16, 1e-2),
                                       (torch.bfloat16, 6e-2)])
def test_steps_give_what_all_rows_at_once_give(dtype, tol):
    """Tolerances as for a block by itself: each of about twenty roundings to the
    features' type (2^-11, 2^-8 of activations of order one) may add its own."""
    blocks = _blocks()
    parts = [_input(rows, dtype=dtype, seed=7 + i)
             for i, rows in enumerate([(100, 0, 31), (1, 1, 1), (40, 7, 300), (1, 0, 2)])]
    ordered = [spconv.SerialOrder("o")(x) for x in parts]
    with torch.no_grad():
        want = _stream64([copy.deepcopy(m).to(dtype).double() for m in blocks], ordered)
    blocks = [m.to(DEV).to(dtype) for m in blocks]
    cache = _cache(dtype=dtype)
    outs = [_step(blocks, x, cache) for x in parts]
    assert cache.rows() == [142, 8, 334] == cache.lengths.tolist()
    for b in range(3):
        got = torch.cat([y.features[y.indices[:, 0] == b] for y in outs]).cpu().double()
        err = float((got - want[b]).abs().max() / want[b].abs().max())
        assert err <= tol, (b, err)


def test_continuations_of_one_scene():
    """Samples that share their first rows' pages give what each would with a copy."""
    blocks = [m.to(DEV) for m in _blocks(window=(None, 0))]
    scene = _input((160, 0, 0), seed=1)
    shared, copies = _cache(), _cache()
    _step(blocks, scene, shared)
    shared.share(0, [1, 2], 160)
    idx = scene.indices.repeat(3, 1)
    idx[:, 0] = torch.arange(3, device=DEV).repeat_interleave(160)
    _step(blocks, spconv.SparseConvTensor(scene.features.repeat(3, 1), idx, scene.spatial_shape, 3), copies)
    assert shared.free_pages() == copies.free_pages() + 20
    for i in range(3):
        x = _input((1, 2, 30), seed=20 + i)
        a, b = _step(blocks, x, shared), _step(blocks, x, copies)
        assert shared._tables()[1].shape == (10,) and copies._tables()[1] is None
        assert torch.allclose(a.features, b.features, rtol=1e-4, atol=1e-5)


def test_features_of_another_type_run_on_f32_copies():
    blocks = [m.to(DEV) for m in _blocks(1)]
    x = _input((20, 3, 5), dtype=torch.float16)
    y = _step(blocks, x, _cache(layers=1))
    assert y.features.dtype == torch.float16 and torch.isfinite(y.features).all()
    with pytest.raises(ValueError, match="k_pages"):
        _step(blocks, x, _cache(layers=1, dtype=torch.float16))


def test_captured_step():
    """A step captured once and replayed as the stream goes on."""
    block = _blocks(1)[0].to(DEV).half()
    parts = [spconv.SerialOrder("o")(_input((1, 1, 1), dtype=torch.float16, seed=30 + i)) for i in range(6)]
    first = spconv.SerialOrder("o")(_input((90, 40, 16), dtype=torch.float16, seed=2))
    eager, captured = (_cache(layers=1, dtype=torch.float16) for _ in range(2))
    for c in (eager, captured):
        c.extend([90, 40, 16])
        block(first, c, 0)
    x = parts[0]
    inputs = spconv.SparseConvTensor(x.features.clone(), x.indices.clone(), x.spatial_shape, 3)
    inputs.indice_dict["o"] = spconv.VoxelOrder(x.indice_dict["o"].offsets, x.indice_dict["o"].rows,
                                                inputs.indices)
    captured.extend([1, 1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(inputs, captured, 0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for refused in (lambda: captured.extend([1, 1, 1]), lambda: captured.drop([0]),
                        lambda: captured.share(0, [], 16)):
            with pytest.raises(RuntimeError, match="captured"):
                refused()
        out = block(inputs, captured, 0).features
    for i, x in enumerate(parts):
        if i:
            captured.extend([1, 1, 1])
        eager.extend([1, 1, 1])
        inputs.features.copy_(x.features), inputs.indices.copy_(x.indices)
        graph.replay()
        torch.cuda.synchronize()
        want = block(x, eager, 0).features
        assert torch.allclose(out, want, rtol=2 ** -8, atol=2 ** -8), i
    assert captured.rows() == eager.rows() == [96, 46, 22]


def test_a_step_without_voxels():
    block = _blocks(1)[0].to(DEV)
    cache = _cache(layers=1)
    assert _step([block], _input((0, 0, 0)), cache).features.shape == (0, 32)
    assert cache.rows() == [0, 0, 0]


def test_document_example():
    """The stream shown in the boundary document, as written there."""
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
    block = re.findall(r"```python\n(.*?)```", text.split("## Streams of voxels", 1)[1], flags=re.S)[0]
    names: dict = {}
    exec(compile(block, "INTEGRATION.md", "exec"), names)
    for i, rows in enumerate([(300, 0, 171), (5, 1, 1)]):
        y = names["step"](_input(rows, channels=16, dtype=torch.float16, seed=i))
        assert y.features.shape == (sum(rows), 128) and torch.isfinite(y.features).all()
    assert names["cache"].rows() == [305, 1, 172]
