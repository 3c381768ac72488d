"""64-bit forms of the voxel-block operators, with bounds on what f32 sums and
one rounding to the output's type may add.  CPU only."""
from __future__ import annotations

import math

import torch

# half a unit in the last place, relative
ROUNDING = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# below these, a type's steps no longer shrink with the value
SMALLEST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
F32 = 2.0 ** -24


def act64(v, act):
    if act in (None, "none"):
        return v
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return v * torch.sigmoid(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))
    return v * torch.sigmoid(v)


def linear64(x, w, bias=None, act=None, residual=None):
    """The result and the bound on an output's error, elementwise.

    An f32 sum of K products is off by at most (K + 1) 2^-24 of the sum of
    their magnitudes (S); no activation's slope is over 1.13, and theirs are
    computed to 4e-7 of |v| (the polynomial's 1.5e-7, the exponential's
    argument and a few roundings)."""
    x, w = x.double(), w.double()
    v = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if bias is not None:
        v, mag = v + bias.double(), mag + bias.double().abs()
    out = act64(v, act)
    tol = 1.13 * (x.shape[1] + 4) * F32 * mag + (4e-7 * v.abs() if act not in (None, "relu") else 0)
    if residual is not None:
        out = out + residual.double()
        tol = tol + 2 * F32 * (v.abs() + residual.double().abs())
    return out, tol


def rotate64(x, positions, weight=None, eps=1e-6, base=10000.0, interleaved=False):
    """One tensor of heads.  The mean of D squares is off by at most (D + 2)
    2^-24 of itself, its root by half that, and about 12 roundings follow for
    each of the pair's two values."""
    x = x.double()
    half, axes = x.shape[-1] // 2, positions.shape[1]
    f = half // axes
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    angle = torch.zeros(x.shape[0], half, dtype=torch.float64)
    for a in range(axes):
        for i in range(f):
            angle[:, a * f + i] = positions[:, a].double() * base ** (-i / f)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    u, w = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :half], y[..., half:])
    both = [u * cos - w * sin, u * sin + w * cos]
    size = (u.abs() + w.abs()) * (x.shape[-1] / 2 + 13) * F32
    if interleaved:
        return torch.stack(both, -1).flatten(-2), torch.stack([size, size], -1).flatten(-2)
    return torch.cat(both, -1), torch.cat([size, size], -1)


def seen(lq, lk, left, right, sinks):
    """(lq, lk): which key a query sees."""
    p = torch.arange(lq)[:, None] + (lk - lq)
    j = torch.arange(lk)[None]
    ok = torch.ones(lq, lk, dtype=torch.bool)
    if right is not None:
        ok &= j <= p + right
    if left is not None:
        ok &= (j >= p - left) | (j < sinks)
    return ok


def attend64(q, k, v, lq, lk, window, sinks, scale=None):
    """A score's f32 error is at most (D + 4) 2^-24 sum |q||k| scale plus two
    roundings of the score (in units of log 2), which moves its exponential
    by as much, relatively; the exponential itself and its rounding to the
    type that multiplies v add 2^-22 and one rounding; the sums over n keys add
    n 2^-24.  All of it multiplies sum p|v|; twice, for the numerator and the
    denominator."""
    rounding = ROUNDING[q.dtype]
    q, k, v = q.double(), k.double(), v.double()
    scale = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    q0 = k0 = 0
    for nq, nk in zip(lq, lk):
        ok = seen(nq, nk, *window, sinks)
        for h in range(q.shape[1]):
            a, b = q[q0:q0 + nq, h], k[k0:k0 + nk, h // group]
            c = v[k0:k0 + nk, h // group]
            if nq == 0 or nk == 0:
                continue
            # a key that no query sees may hold anything
            used = ok.any(0)
            b, c = b.clone(), c.clone()
            b[~used], c[~used] = 0, 0
            s = (a @ b.t() * scale).masked_fill(~ok, -math.inf)
            some = ok.any(1)
            p = torch.zeros_like(s)
            p[some] = torch.softmax(s[some], -1)
            out[q0:q0 + nq, h] = p @ c
            mag = (a.abs() @ b.abs().t() * abs(scale)).masked_fill(~ok, 0)
            rel = ((a.shape[1] + 4) * F32 * mag + 4 * F32 * mag).amax(1, keepdim=True)
            tol[q0:q0 + nq, h] = (p @ c.abs()) * (2 * rel + 2.0 ** -21 + rounding + 2 * nk * F32)
        q0, k0 = q0 + nq, k0 + nk
    return out, tol


def check(got, ref, tol, what=""):
    """got within tol and one rounding of ref, everywhere; NaN only where ref has it."""
    got64, dt = got.detach().cpu().double(), got.dtype
    assert got64.shape == ref.shape, (what, got64.shape, ref.shape)
    if not ref.numel():
        return
    assert torch.equal(torch.isnan(got64), torch.isnan(ref)), f"{what}: NaN in other places"
    bound = ROUNDING[dt] * (ref.abs() + tol) + tol + SMALLEST[dt]
    over = ((got64 - ref).abs() / bound).nan_to_num(0.0)
    assert float(over.max()) <= 1.0, f"{what}: {float(over.max()):.2f} times the bound at " \
        f"{[int(i) for i in torch.unravel_index(over.argmax(), over.shape)]}"
