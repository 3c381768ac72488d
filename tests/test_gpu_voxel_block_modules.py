"""VoxelBlock with hooked and replaced projections, and features of another type
than its parameters."""
import copy

import pytest
import torch
import torch.nn as nn

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

NAMES = ["qkv", "proj", "up", "down"]


def _input(dtype=torch.float32, channels=32, n=300):
    g = torch.Generator().manual_seed(3)
    cells = torch.randperm(20 * 24 * 22, generator=g)[:n]
    idx = torch.stack([torch.arange(n) % 2, cells // (24 * 22), cells // 22 % 24, cells % 22], 1)
    f = torch.randn(n, channels, generator=g).to(dtype)
    x = spconv.SparseConvTensor(f.to(DEV), idx.int().to(DEV), [20, 24, 22], 2)
    return spconv.SerialOrder("o")(x)


def _block(**kw):
    torch.manual_seed(4)
    return spconv.VoxelBlock(32, 2, "o", window=(40, 24), sinks=3, **kw).to(DEV)


class Halved(nn.Module):
    """Half of a product, in another module than nn.Linear."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x) * 0.5


@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("name", NAMES)
def test_replaced_projection(name, activation):
    """A module in a projection's place is what runs; its sums may come from
    another kernel, so the results agree to f32's accuracy over the block."""
    x, block = _input(), _block(activation=activation)
    merged = copy.deepcopy(block)
    with torch.no_grad():
        getattr(merged, name).weight.mul_(0.5)
        getattr(merged, name).bias.mul_(0.5)
    plain = block(x).features
    setattr(block, name, Halved(getattr(block, name)))
    got, want = block(x).features, merged(x).features
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-5)
    assert not torch.allclose(got, plain, rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("name", NAMES)
def test_hooks_run(name):
    x, block = _input(), _block()
    plain, calls = block(x).features, []
    inner = getattr(block, name)
    pre = inner.register_forward_pre_hook(lambda m, args: calls.append("pre"))
    post = inner.register_forward_hook(lambda m, args, out: out * 0.5)
    halved = block(x).features
    assert calls == ["pre"] and not torch.allclose(halved, plain, rtol=1e-3, atol=1e-3)
    post.remove()
    assert torch.allclose(block(x).features, plain, rtol=1e-4, atol=1e-5) and calls == ["pre"] * 2
    pre.remove()
    assert torch.equal(block(x).features, plain)


def test_subclass_runs_its_own_forward():
    class Twice(nn.Linear):
        def forward(self, x):
            return super().forward(x) * 2

    x, block = _input(), _block()
    plain = block(x).features
    block.up.__class__ = Twice
    assert not torch.allclose(block(x).features, plain, rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("features,parameters", [
    (torch.float16, torch.float32), (torch.bfloat16, torch.float32), (torch.float64, torch.float32),
    (torch.float32, torch.float16), (torch.float16, torch.bfloat16), (torch.float64, torch.float64)])
def test_features_of_another_type(features, parameters):
    """As in the convolutions: f32 copies compute it, and the result has the
    features' type."""
    block = _block(kv_heads=1).to(parameters)
    x = _input(features)
    got = block(x)
    assert got.features.dtype is features and got.indices is x.indices
    want = copy.deepcopy(block).float()(x.replace_feature(x.features.float()))
    assert torch.equal(got.features, want.features.to(features))
    assert all(p.dtype is parameters for p in block.parameters())


def test_one_parameter_of_another_type():
    """A block in f16 whose norms are kept in f32, as mixed precision leaves it."""
    block = _block().half()
    block.norm1.float(), block.norm2.float()
    x = _input(torch.float16)
    want = copy.deepcopy(block).float()(x.replace_feature(x.features.float()))
    assert torch.equal(block(x).features, want.features.half())


def test_hooks_run_on_features_of_another_type():
    block, calls = _block(), []
    block.up.register_forward_hook(lambda m, args, out: calls.append(out.dtype))
    block(_input(torch.bfloat16))
    assert calls == [torch.float32]
