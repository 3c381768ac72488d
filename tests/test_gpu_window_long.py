"""window_attention on long 16-bit walks: 64 rows a wave, tiles of 256 rows."""
import math

import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import F32, ROUNDING, check

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float16, torch.bfloat16]


def _offsets(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)


def _inputs(lq, lk, hq, hk, dim, dtype):
    """At least 4096 keys in reach and 512 tiles of 256 rows over the key heads:
    the calls that take 64 rows a wave."""
    assert dim <= 64 and (sum(lq) * (hq // hk) // 256 + len(lq)) * hk >= 512
    g = torch.Generator().manual_seed(sum(lq) + 3 * sum(lk) + dim + hk)
    q = torch.randn(sum(lq), hq, dim, generator=g).to(dtype)
    k, v = (torch.randn(sum(lk), hk, dim, generator=g).to(dtype) for _ in range(2))
    return q, k, v


def _seen(i, nq, nk, window, sinks):
    p, j = i + nk - nq, torch.arange(nk)
    ok = torch.ones(nk, dtype=torch.bool)
    if window[1] is not None:
        ok &= j <= p + window[1]
    if window[0] is not None:
        ok &= (j >= p - window[0]) | (j < sinks)
    return ok


def _rows(lq):
    """Rows around the tiles' edges, the samples' ends, and some between."""
    rows, q0 = set(), 0
    for n in lq:
        near = {0, 1, 31, 32, 63, 64, 255, 256, n // 2, n - 257, n - 65, n - 64, n - 2, n - 1}
        rows |= {q0 + i for i in near | set(range(17, n, 611)) if 0 <= i < n}
        q0 += n
    return sorted(rows)


def _check(got, q, k, v, lq, lk, window, sinks):
    """Single rows in 64 bits, with the bounds that the whole form has."""
    group, scale, dim = q.shape[1] // k.shape[1], q.shape[2] ** -0.5, q.shape[2]
    rows = _rows(lq)
    ref = torch.zeros(len(rows), *q.shape[1:], dtype=torch.float64)
    tol = torch.zeros_like(ref)
    for n, r in enumerate(rows):
        q0 = k0 = 0
        for nq, nk in zip(lq, lk):
            if r < q0 + nq:
                break
            q0, k0 = q0 + nq, k0 + nk
        ok = _seen(r - q0, nq, nk, window, sinks)
        if not ok.any():
            continue
        kk, vv = (t[k0:k0 + nk][ok].double().transpose(0, 1) for t in (k, v))  # (hk, keys, dim)
        x = q[r].double().view(-1, group, dim)
        s = torch.matmul(x, kk.transpose(1, 2).contiguous()) * scale
        p = torch.softmax(s, -1)
        mag = torch.matmul(x.abs(), kk.abs().transpose(1, 2).contiguous()) * scale
        rel = ((dim + 8) * F32 * mag).amax(-1, keepdim=True)
        ref[n] = torch.matmul(p, vv).view(-1, dim)
        tol[n] = (torch.matmul(p, vv.abs()) *
                  (2 * rel + 2.0 ** -21 + ROUNDING[q.dtype] + 2 * nk * F32)).view(-1, dim)
    assert math.isfinite(float(ref.abs().max()))
    check(got[rows], ref, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,lk,hq,hk,dim,window,sinks", [
    ([8200], [8200], 16, 16, 64, (None, None), 0),
    ([8200], [8200], 16, 16, 64, (None, 0), 0),
    ([8200], [8200], 16, 4, 64, (4300, None), 5),
    ([8200], [8200], 16, 16, 40, (4100, 0), 130),
    ([5003, 3300], [5003, 3300], 16, 8, 32, (None, 7), 0),
    ([5003, 3300], [6100, 3000], 16, 2, 64, (5000, 33), 40),
    ([4097, 1, 0, 4300], [4097, 77, 50, 4300], 16, 16, 24, (None, None), 0),
    ([8193], [8400], 16, 1, 63, (None, 0), 0),           # rows aligned to their elements only
])
def test_against_single_rows(lq, lk, hq, hk, dim, window, sinks, dtype):
    say("window_attention long:", lq, lk, hq, hk, dim, window, sinks, dtype)
    q, k, v = _inputs(lq, lk, hq, hk, dim, dtype)
    got = spconv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), _offsets(lq), _offsets(lk),
                                  window=window, sinks=sinks).cpu()
    assert torch.isfinite(got).all()
    _check(got, q, k, v, lq, lk, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_outgrow_their_reference(dtype):
    """One vote moves the references of both row blocks: rows whose scores rise
    beside rows whose scores do not."""
    lq = lk = [8200]
    q, k, v = _inputs(lq, lk, 16, 16, 64, dtype)
    steps = torch.linspace(0, 60, 41).repeat_interleave(200)[:, None, None]
    k = (0.1 * k.float() + steps / 8).to(dtype)
    q[::3] = 0.125
    q[1::3] *= 0.01
    got = spconv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), _offsets(lq), window=(None, 0)).cpu()
    _check(got, q, k, v, lq, lk, (None, 0), 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [((4200, 0), 3), ((None, 0), 0)])
def test_unseen_keys_may_hold_anything(window, sinks, dtype):
    lq = lk = [5100, 3300]
    q, k, v = _inputs(lq, lk, 16, 8, 64, dtype)

    def run():
        return spconv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), _offsets(lq), window=window,
                                       sinks=sinks).cpu()

    clean = run()
    bad = [4700, 5099, 5100 + 3000]
    for j, x in zip(bad, (float("nan"), float("inf"), float("-inf"))):
        v[j] = x
        k[j] = float("nan")
    got = run()
    hit = torch.zeros(sum(lq), dtype=torch.bool)
    q0 = 0
    for nq in lq:
        for i in range(nq):
            ok = _seen(i, nq, nq, window, sinks)
            hit[q0 + i] = any(ok[j - q0] for j in bad if q0 <= j < q0 + nq)
        q0 += nq
    assert 100 < int(hit.sum()) < sum(lq) - 100
    assert torch.equal(got[~hit], clean[~hit])
    assert torch.isnan(got[hit]).all()


def test_values_only_non_finite():
    """An infinite value reaches the rows that see it, as an infinity, in its own
    column."""
    lq = lk = [8200]
    q, k, v = _inputs(lq, lk, 16, 16, 64, torch.bfloat16)
    clean = spconv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), _offsets(lq), window=(None, 0)).cpu()
    v[8000, 2, 3] = float("inf")
    got = spconv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), _offsets(lq), window=(None, 0)).cpu()
    assert torch.equal(got[:8000], clean[:8000])
    assert (got[8000:, 2, 3] == float("inf")).all()
    got[8000:, 2, 3] = 0
    assert torch.isfinite(got).all()
