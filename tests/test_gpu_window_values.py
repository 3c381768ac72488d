"""window_attention on values near the ends of their type's range."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import attend64, check

pytestmark = [pytest.mark.gpu, needs_gpu]

WIDE = [torch.float32, torch.bfloat16]


def _run(q, k, v, window=(None, None), sinks=0):
    off = [torch.tensor([0, len(t)], dtype=torch.int32, device=DEV) for t in (q, k)]
    got = spconv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), *off, window=window, sinks=sinks)
    check(got, *attend64(q, k, v, [len(q)], [len(k)], window, sinks))


def _qkv(queries, keys, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + queries + keys + dim)
    q = torch.randn(queries, 2, dim, generator=g)
    k, v = (torch.randn(keys, 2, dim, generator=g) for _ in range(2))
    return q.to(dtype), k.to(dtype), v


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("queries,keys", [(1, 1), (40, 40), (1, 8000), (700, 700), (300, 8000)])
@pytest.mark.parametrize("size", [1e34, 1e-37])
def test_values_of_one_size(size, queries, keys, dtype):
    """Averages of values as large, or as small, as they are: no sum along the
    way leaves the range that weights of at most one would keep it in.  Few
    queries split the keys."""
    say("window_attention values:", size, queries, keys, dtype)
    for dim in (32, 64):
        q, k, v = _qkv(queries, keys, dim, dtype)
        _run(q, k, (v.abs().clamp(0.5, 2.0) * size).to(dtype))
        _run(q, k, (v.clamp(-2.0, 2.0) * size).to(dtype))   # both signs


@pytest.mark.parametrize("dtype", WIDE)
def test_one_key_of_the_largest_values(dtype):
    q, k, v = _qkv(1, 1, 64, dtype)
    _run(q, k, torch.full_like(v, 3e38).to(dtype))
    _run(q, k, torch.full_like(v, -2e36).to(dtype))


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("queries", [2, 560])
def test_large_values_at_scores_that_rise(queries, dtype):
    """Scores that rise by up to six between blocks of keys: weights grow beside
    their reference before it moves, and their values are large."""
    steps = torch.tensor([0.0, 3.0, 5.0, 4.0, 8.0, 8.5, 13.0, 0.0]).repeat_interleave(70)
    q, k, v = _qkv(queries, 560, 64, dtype)
    q = torch.full_like(q, 0.5)
    k = (0.1 * k.float() + steps[:, None, None] / 4).to(dtype)
    _run(q, k, (v.clamp(-2.0, 2.0) * 4e35).to(dtype))
