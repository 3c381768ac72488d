"""window_attention on scores so large that their steps in f32 exceed one."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu, say

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _offsets(n):
    return torch.tensor([0, n], dtype=torch.int32, device=DEV)


def _run(q, k, v, **kw):
    return spconv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), _offsets(len(q)), _offsets(len(k)),
                                   **kw).cpu()


def _expect(got, v, of, dtype):
    """The mean of the values at keys ``of`` (all of one score, the others further
    below than any weight reaches), to the sums' and one rounding."""
    want = v[of].double().mean(0, keepdim=True)
    step = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    bound = (2 * step + 2.0 ** -19) * v[of].double().abs().mean(0, keepdim=True) + 2.0 ** -24
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() / bound).max())


def _tensors(queries, keys, size, levels, dtype):
    """Every score is size^2 * 8 * (the key's level), a power of two, exactly."""
    g = torch.Generator().manual_seed(queries + keys)
    level = torch.tensor(levels)[torch.arange(keys) % len(levels)]
    q = torch.full((queries, 2, 64), size).to(dtype)
    k = (size * level)[:, None, None].expand(keys, 2, 64).to(dtype).clone()
    return q, k, torch.randn(keys, 2, 64, generator=g).to(dtype), level


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,keys", [(1, 3), (40, 100), (2, 5000), (300, 300)])
@pytest.mark.parametrize("levels", [[1.0, 0.5, 0.25], [-1.0, -0.5, -0.75], [0.75, 0.0, -0.5]])
def test_the_largest_score_takes_all(levels, queries, keys, dtype):
    """Scores from 2^20 to 2^33 (f16) or 2^50."""
    for exponent in (9, 11, 12, 13, 15) + (() if dtype is torch.float16 else (23,)):
        say("window_attention scores:", levels, queries, keys, exponent, dtype)
        q, k, v, level = _tensors(queries, keys, 2.0 ** exponent, levels, dtype)
        _expect(_run(q, k, v), v, level == level.max(), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,keys", [(3, 200), (2, 5000), (300, 400)])
def test_small_scores_after_far_ones(queries, keys, dtype):
    """The first keys' scores lie 2^33 below the others', which are all zero: what
    was summed at the first reference is worth nothing at the next."""
    q, k, v, _ = _tensors(queries, keys, 2.0 ** 15, [-1.0], dtype)
    k[70:] = 0
    _expect(_run(q, k, v), v, torch.arange(keys) >= 70, dtype)


@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_some_rows_of_a_long_walk(dtype):
    """64 rows a wave: rows with such scores beside rows whose scores are zero."""
    n = 8200
    g = torch.Generator().manual_seed(7)
    level = torch.tensor([0.5, 1.0, -1.0, 0.25])[torch.arange(n) % 4]
    q = torch.zeros(n, 16, 64)
    rows = torch.arange(5, n, 410)
    q[rows] = 2.0 ** 15
    k = (2.0 ** 15 * level)[:, None, None].expand(n, 16, 64)
    v = torch.randn(n, 16, 64, generator=g).to(dtype)
    got = _run(q.to(dtype), k.to(dtype), v)
    _expect(got[rows], v, level == 1.0, dtype)
    others = torch.ones(n, dtype=torch.bool)
    others[rows] = False
    _expect(got[others], v, torch.ones(n, dtype=torch.bool), dtype)
