"""SerialOrder and VoxelBlock between convolutions, and under graph capture."""
import copy

import numpy as np
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu
from sequence_oracle import act64, attend64, rotate64

pytestmark = [pytest.mark.gpu, needs_gpu]


def _cloud(seed, shape, per_sample):
    rng = np.random.default_rng(seed)
    parts = []
    for b, n in enumerate(per_sample):
        cells = rng.choice(shape[0] * shape[1] * shape[2], size=n, replace=False)
        z, r = np.divmod(cells, shape[1] * shape[2])
        y, x = np.divmod(r, shape[2])
        parts.append(np.stack([np.full(n, b), z, y, x], 1))
    idx = np.concatenate(parts).astype(np.int32)
    return torch.from_numpy(idx[rng.permutation(len(idx))])


def _input(per_sample=(300, 0, 171), channels=32, dtype=torch.float32, seed=0):
    shape = (20, 24, 22)
    idx = _cloud(seed, shape, per_sample)
    f = torch.randn(len(idx), channels, generator=torch.Generator().manual_seed(seed)).to(dtype)
    return spconv.SparseConvTensor(f.to(DEV), idx.to(DEV), list(shape), len(per_sample))


def test_serial_order():
    x = _input()
    y = spconv.SerialOrder("o")(x)
    order = y.indice_dict["o"]
    assert order.offsets.tolist() == [0, 300, 300, 471] and order.indices is y.indices
    assert torch.equal(y.indices, x.indices[order.rows])
    assert torch.equal(y.features, x.features[order.rows])

    def code(row):
        b, z, y_, x_ = (int(c) for c in row)
        return (b, sum(((z >> i & 1) << 2 | (y_ >> i & 1) << 1 | x_ >> i & 1) << 3 * i
                       for i in range(16)))

    codes = [code(r) for r in y.indices.cpu()]
    assert codes == sorted(codes)
    with pytest.raises(ValueError, match="65536"):
        spconv.SerialOrder("o")(spconv.SparseConvTensor(x.features, x.indices, [1, 1, 1 << 17], 3))


def _block64(m, f, idx, lens):
    """VoxelBlock in 64 bits on the CPU."""
    f = f.double()
    hq, hk = m.heads, m.kv_heads
    qkv = m.qkv(m.norm1(f)).view(len(f), hq + 2 * hk, m.dim)
    q, _ = rotate64(qkv[:, :hq], idx[:, 1:], m.q_gain, m.eps, m.base)
    k, _ = rotate64(qkv[:, hq:hq + hk], idx[:, 1:], m.k_gain, m.eps, m.base)
    # attend64 names a rounding by its inputs' type
    a, _ = attend64(q.float(), k.float(), qkv[:, hq + hk:].float(), lens, lens, m.window, m.sinks)
    f = f + m.proj(a.reshape(f.shape))
    return f + m.down(act64(m.up(m.norm2(f)), m.activation))


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.float16, 1e-2),
                                       (torch.bfloat16, 6e-2)])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1)])
def test_block(heads, kv, dtype, tol):
    """About ten layers of roundings deep: each rounding to the features' type
    (2^-11, 2^-8 of an activation of order one) may add to the output's."""
    torch.manual_seed(1)
    m = spconv.VoxelBlock(32, heads, "o", kv_heads=kv, window=(40, 24), sinks=3)
    with torch.no_grad():
        m.q_gain.add_(0.1 * torch.randn(m.dim))
    x = spconv.SerialOrder("o")(_input(dtype=dtype))
    ref_m = copy.deepcopy(m).to(dtype).double()
    with torch.no_grad():
        ref = _block64(ref_m, x.features.cpu(), x.indices.cpu(), [300, 0, 171])
    y = m.to(DEV).to(dtype)(x)
    assert y.indices is x.indices and y.features.dtype == dtype
    err = float((y.features.cpu().double() - ref).abs().max() / ref.abs().max())
    assert err <= tol, err


def test_between_convolutions():
    """A convolution, the order, two blocks, a convolution on the ordered rows:
    the same features, row by row, whatever order the voxels came in."""
    torch.manual_seed(2)
    net = spconv.SparseSequential(
        spconv.SubMConv3d(8, 32, 3, indice_key="in"), spconv.SerialOrder("o"),
        spconv.VoxelBlock(32, 2, "o", window=(30, 30)), spconv.VoxelBlock(32, 2, "o"),
        spconv.SubMConv3d(32, 16, 3, indice_key="out"), torch.nn.ReLU()).to(DEV)
    x = _input(channels=8)
    perm = torch.randperm(len(x.features), generator=torch.Generator().manual_seed(5)).to(DEV)
    z = spconv.SparseConvTensor(x.features[perm], x.indices[perm], x.spatial_shape, x.batch_size)
    a, b = net(x), net(z)
    assert torch.equal(a.indices, b.indices)
    assert torch.allclose(a.features, b.features, rtol=1e-4, atol=1e-5)
    assert a.features.abs().max() > 0


def test_refusals():
    x = _input()
    block = spconv.VoxelBlock(32, 2, "o").to(DEV)
    with pytest.raises(KeyError, match="SerialOrder"):
        block(x)
    y = spconv.SerialOrder("o")(x)
    down = spconv.SparseConv3d(32, 32, 3, stride=2, padding=1).to(DEV)
    with pytest.raises(ValueError, match="coordinates"):
        block(down(y))
    with pytest.raises(ValueError, match="divide"):
        spconv.VoxelBlock(32, 3, "o")
    with pytest.raises(ValueError, match="divide"):
        spconv.VoxelBlock(32, 4, "o", kv_heads=3)


@pytest.mark.parametrize("rows", [(300, 0, 171), (1, 1, 1)])
def test_graph_replays(rows):
    """The block captured once and replayed between eager work: every replay
    equals the eager result on what its input holds then."""
    torch.manual_seed(3)
    block = spconv.VoxelBlock(32, 2, "o", window=(40, 0), sinks=2).to(DEV).half()
    x = spconv.SerialOrder("o")(_input(rows, dtype=torch.float16))
    inputs = x.replace_feature(x.features.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            block(inputs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(inputs).features
    for i in range(4):
        inputs.features.copy_(torch.randn_like(inputs.features) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, block(inputs).features), i


def test_document_example():
    """The network shown in the boundary document, as written there."""
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
    block = re.findall(r"```python\n(.*?)```", text.split("## Voxel blocks", 1)[1], flags=re.S)[0]
    names: dict = {}
    exec(compile(block, "INTEGRATION.md", "exec"), names)
    y = names["net"](_input(channels=16, dtype=torch.float16))
    assert y.features.shape == (471, 64) and torch.isfinite(y.features).all()


def test_block_of_no_voxels():
    net = spconv.SparseSequential(spconv.SerialOrder("o"), spconv.VoxelBlock(32, 2, "o")).to(DEV)
    assert net(_input(per_sample=(0, 0))).features.shape == (0, 32)
