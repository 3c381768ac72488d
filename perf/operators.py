"""The calls of a voxel transformer block: what is timed, over which sizes.

A case is a dict of plain values.  ``op`` names the operator:

    linear  y = act(x W^T + bias) + residual            spconv.linear_act
    rotate  RMS norm of every query and key head and     spconv.norm_rotate_heads
            rotation by the voxel's coordinates
    attend  attention of packed sequences in a window,   spconv.window_attention
            the first ``sinks`` keys always visible

Every operator has a plain form here, in elementary torch operations in 32
bits with one rounding at the end, and a definition in 64 bits (``exact``).
"""
from __future__ import annotations

import itertools
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
EPS = 1e-6
# extents (z, y, x) of the grids that the coordinates come from
LIDAR, OBJECT, SCENE = "41x1600x1408", "64x64x64", "256x256x256"
GRIDS = (OBJECT, "160x160x160", SCENE, LIDAR)


def _linear(rows, c_in, c_out, dtype, act="none", bias=True, residual=False):
    return {"op": "linear", "rows": rows, "c_in": c_in, "c_out": c_out, "dtype": dtype,
            "act": act, "bias": bias, "residual": residual}


def _rotate(rows, q_heads, k_heads, dim, dtype, grid, gain="dim", interleaved=False,
            base=10000.0):
    return {"op": "rotate", "rows": rows, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "dtype": dtype, "grid": grid, "gain": gain, "interleaved": interleaved, "base": base}


def _attend(samples, keys, fewer, queries, q_heads, k_heads, dim, dtype, left, right, sinks):
    """Sample b has keys - b*fewer keys; queries 0: as many queries as keys,
    else that many, the last of the sample.  left or right -1: no limit."""
    return {"op": "attend", "samples": samples, "keys": keys, "fewer": fewer, "queries": queries,
            "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "dtype": dtype, "left": left,
            "right": right, "sinks": sinks}


def listed():
    cases = [
        # one new token: the projection of a streaming step, all latency
        ("linear_token", _linear(1, 512, 2048, "bf16", "gelu")),
        # the widening product of a block over one LiDAR scan: mostly its output's bytes
        ("linear_up_60k", _linear(60_013, 192, 768, "f16", "gelu")),
        # the narrowing product of that block, added to the block's input
        ("linear_down_60k", _linear(60_013, 768, 192, "bf16", residual=True)),
        # the same in the default precision, on a small scene
        ("linear_f32_20k", _linear(20_011, 96, 384, "f32", "gelu")),
        # the widest product: a large decoder over a whole scene
        ("linear_wide_64k", _linear(65_536, 1024, 4096, "bf16", "silu")),
        # one new token for each of four streams
        ("rotate_token", _rotate(4, 16, 4, 64, "bf16", SCENE)),
        # a small scene in the default precision
        ("rotate_f32_20k", _rotate(20_011, 6, 6, 32, "f32", LIDAR, gain="head")),
        # a whole scene, wide heads of a decoder
        ("rotate_500k", _rotate(500_000, 12, 12, 64, "bf16", SCENE)),
        # one new token for each of four streams over what they keep: causal, with sinks
        ("attend_token", _attend(4, 20_000, 1777, 1, 16, 4, 64, "bf16", 4095, 0, 16)),
        # two small scenes in the default precision, narrow heads, a short window
        ("attend_f32_2x10k", _attend(2, 10_007, 1003, 0, 6, 6, 32, "f32", 128, 128, 0)),
        # a batch of LiDAR scans, the ordinary window, a few register tokens in front
        ("attend_lidar_4x60k", _attend(4, 60_000, 1013, 0, 4, 4, 64, "f16", 512, 512, 8)),
        # an object whose voxels all see one another, step after step of a sampler
        ("attend_full_8k", _attend(1, 8192, 0, 0, 16, 16, 64, "bf16", -1, -1, 0)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A channel count: half of them multiples of 16, the others any number."""
    w = _log(rng, lo, hi)
    return max(16, w // 16 * 16) if rng.random() < 0.5 else w


def _scores(c):
    """Values in the plain form's matrix of scores."""
    qb, kb, blocks = _bands(c)
    return c["samples"] * c["q_heads"] * blocks * qb * (kb + c["sinks"])


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["op"], {"bytes": 0, "flops": 0})
        for k in m:
            m[k] = max(m[k], w[k])
    op = rng.choice(("linear", "rotate", "attend"))
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    while True:
        if op == "linear":
            c = _linear(_log(rng, 1, 200_000), _width(rng, 16, 2048), _width(rng, 16, 4096), dtype,
                        rng.choice(ACTS), rng.random() < 0.8, rng.random() < 0.4)
        elif op == "rotate":
            k = rng.choice((1, 2, 3, 4, 6, 8, 12))
            c = _rotate(_log(rng, 1, 500_000), k * rng.choice((1, 1, 2, 4)), k,
                        rng.choice((16, 32, 40, 48, 64, 64, 72, 96, 128)), dtype, rng.choice(GRIDS),
                        rng.choice(("none", "dim", "head")), rng.random() < 0.3,
                        rng.choice((100.0, 10000.0)))
        else:
            k = rng.choice((1, 2, 3, 4, 6, 8))
            samples = rng.randint(1, 6)
            keys = _log(rng, 1, 60_000)
            left, right = (_log(rng, 16, 4096) if rng.random() < 0.9 else -1 for _ in range(2))
            right = 0 if rng.random() < 0.3 else right
            c = _attend(samples, keys, rng.randint(0, keys // samples),
                        rng.choice((0, 0, 0, 1, 1, rng.randint(1, 64))), k * rng.choice((1, 1, 2, 4)),
                        k, rng.choice((16, 32, 40, 64, 64, 80, 128)), dtype, left, right,
                        rng.choice((0, 0, 1, 4, 16)))
            if _scores(c) > 2_000_000_000:
                continue
        w = work(c)
        # products in the default precision run on a slower unit
        if all(w[k] <= most[op][k] / (8 if k == "flops" and dtype == "f32" else 1) for k in w):
            return c


# ----------------------------------------------------------------- inputs
def _lengths(c):
    """(queries, keys) of each sample."""
    lk = [max(0, c["keys"] - b * c["fewer"]) for b in range(c["samples"])]
    return [n if c["queries"] == 0 else c["queries"] for n in lk], lk


def _offsets(lengths):
    return torch.tensor([0, *itertools.accumulate(lengths)], dtype=torch.int32, device=DEV)


def prepare(case, seed):
    """The tensors a network has in hand at the call; nothing is laid out or
    planned ahead, these operators read them as they are."""
    g = torch.Generator(DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dt)

    s = {"case": case}
    if case["op"] == "linear":
        n, ci, co = case["rows"], case["c_in"], case["c_out"]
        s["x"] = randn(n, ci)
        s["weight"] = randn(co, ci, scale=ci ** -0.5)
        s["bias"] = randn(co, scale=0.1) if case["bias"] else None
        s["residual"] = randn(n, co) if case["residual"] else None
    elif case["op"] == "rotate":
        n, hq, hk, d = case["rows"], case["q_heads"], case["k_heads"], case["dim"]
        # queries, keys and values lie side by side, as one projection leaves them
        qkv = randn(n, hq + 2 * hk, d, scale=2.0)
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        z, y, x = (int(v) for v in case["grid"].split("x"))
        cell = torch.randint(0, z * y * x, (n,), generator=g, device=DEV)
        coords = torch.stack([torch.zeros_like(cell), cell // (y * x), cell // x % y, cell % x], 1)
        s["positions"] = coords.to(torch.int32)[:, 1:]  # (z, y, x) of (b, z, y, x) rows
        gain = {"none": None, "dim": (d,), "head": (None, d)}[case["gain"]]
        for name, h in (("q_weight", hq), ("k_weight", hk)):
            s[name] = None if gain is None else \
                randn(*[h if v is None else v for v in gain], scale=0.1, shift=1.0)
    else:
        lq, lk = _lengths(case)
        s["q"] = randn(sum(lq), case["q_heads"], case["dim"])
        s["k"] = randn(sum(lk), case["k_heads"], case["dim"])
        s["v"] = randn(sum(lk), case["k_heads"], case["dim"])
        s["offsets_q"] = _offsets(lq)
        s["offsets_k"] = _offsets(lk)
    return s


# ------------------------------------------------------------ plain forms
def _act(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _plain_linear(s):
    v = s["x"].float() @ s["weight"].float().t()
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _act(v, s["case"]["act"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(s["x"].dtype)


def _plain_rotate(s):
    case = s["case"]
    d = case["dim"]
    f = d // 2 // 3  # pairs per axis
    i = torch.arange(f, device=DEV, dtype=torch.float32)
    turn = s["positions"].float()[:, :, None] * case["base"] ** (-i / f)  # (rows, axes, f)
    turn = torch.nn.functional.pad(turn.flatten(1), (0, d // 2 - 3 * f))[:, None]
    cos, sin = torch.cos(turn), torch.sin(turn)

    def one(x, weight):
        v = x.float()
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
        if weight is not None:
            v = v * weight.float()
        if case["interleaved"]:
            a, b = v[..., 0::2], v[..., 1::2]
            return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2).to(x.dtype)
        a, b = v[..., :d // 2], v[..., d // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def _bands(c):
    """The plain form's blocks: (queries of a block, keys beside each block,
    blocks).  Keys 0: each block sees every key."""
    lq, lk = _lengths(c)
    mq, mk = max(max(lq), 1), max(max(lk), 1)
    if c["left"] >= 0 and c["right"] >= 0:
        span = c["left"] + c["right"]
        qb = min(mq, max(64, span // 2))
        if qb + span < mk:
            return qb, qb + span, -(-mq // qb)
    return mq, mk, 1


def _plain_attend(s):
    """Every sample padded to the longest; blocks of queries against the band
    of keys that their windows cover, and the sinks beside them."""
    c = s["case"]
    lq, lk = _lengths(c)
    B, hq, hk, d = c["samples"], c["q_heads"], c["k_heads"], c["dim"]
    if not sum(lq):
        return torch.zeros_like(s["q"])
    if not sum(lk):
        return torch.zeros_like(s["q"])
    qb, kb, blocks = _bands(c)
    banded = blocks > 1 or kb < max(lk)
    left = c["left"] if c["left"] >= 0 else 1 << 30
    right = c["right"] if c["right"] >= 0 else 1 << 30
    off_q, off_k = s["offsets_q"].long(), s["offsets_k"].long()
    n_q, n_k = off_q.diff(), off_k.diff()
    i = torch.arange(blocks * qb, device=DEV).view(1, blocks, qb)
    pos = i + (n_k - n_q).view(B, 1, 1)                                     # (B, blocks, qb)
    there = i < n_q.view(B, 1, 1)
    rows = (i + off_q[:-1].view(B, 1, 1)).clamp_max(s["q"].shape[0] - 1)
    j = torch.arange(kb, device=DEV).view(1, 1, kb)
    if banded:
        j = pos[:, :, :1] - left + j                                       # (B, blocks, kb)
    sink = torch.arange(c["sinks"] if banded else 0, device=DEV).view(1, 1, -1)
    key = torch.cat([j.expand(B, blocks, kb), sink.expand(B, blocks, -1)], 2)
    p, at = pos[..., None], key[:, :, None]
    seen = (at >= 0) & (at < n_k.view(B, 1, 1, 1)) & (at <= p + right)
    first = torch.arange(key.shape[2], device=DEV) < kb
    # a sink inside the window is counted there, and not again in its own column
    near, sinks = at >= p - left, at < c["sinks"]
    seen = seen & (torch.where(first, near, sinks & ~near) if banded else near | sinks)
    seen = seen[:, :, None, None]                                          # over the heads
    cols = (key + off_k[:-1].view(B, 1, 1)).clamp(0, s["k"].shape[0] - 1)
    q = s["q"].float()[rows].view(B, blocks, qb, hk, hq // hk, d).permute(0, 1, 3, 4, 2, 5)
    k = s["k"].float()[cols].permute(0, 1, 3, 4, 2)[:, :, :, None]          # (B, blocks, hk, 1, d, keys)
    v = s["v"].float()[cols].permute(0, 1, 3, 2, 4)[:, :, :, None]
    w = torch.matmul(q, k) * d ** -0.5
    w = w.masked_fill(~seen, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - top.masked_fill(top == -math.inf, 0.0))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w, v) / total.masked_fill(total == 0, 1.0)
    o = o.permute(0, 1, 4, 2, 3, 5).reshape(B, blocks * qb, hq, d)
    out = torch.empty_like(s["q"])
    there = there.reshape(B, -1)
    out[rows.reshape(B, -1)[there]] = o[there].to(out.dtype)
    return out


def run(state):
    c = state["case"]
    if not own:
        return {"linear": _plain_linear, "rotate": _plain_rotate,
                "attend": _plain_attend}[c["op"]](state)
    import trispconv.pytorch as spconv
    if c["op"] == "linear":
        return spconv.linear_act(state["x"], state["weight"], state["bias"], activation=c["act"],
                                 residual=state["residual"])
    if c["op"] == "rotate":
        return spconv.norm_rotate_heads(state["q"], state["k"], state["positions"],
                                        q_weight=state["q_weight"], k_weight=state["k_weight"],
                                        eps=EPS, base=c["base"], interleaved=c["interleaved"])
    window = tuple(None if v < 0 else v for v in (c["left"], c["right"]))
    return spconv.window_attention(state["q"], state["k"], state["v"], state["offsets_q"],
                                   state["offsets_k"], window=window, sinks=c["sinks"])


# ------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "linear":
        n, ci, co = case["rows"], case["c_in"], case["c_out"]
        out = n * co * (2 if case["residual"] else 1)
        return {"bytes": e * (n * ci + ci * co + out + (co if case["bias"] else 0)),
                "flops": 2 * n * ci * co}
    if case["op"] == "rotate":
        values = case["rows"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        # squares and their sum, the norm's two products, four products and two sums for a pair
        return {"bytes": 2 * e * values + 12 * case["rows"], "flops": 7 * values}
    # pairs of a query and a key it sees, and keys that some query sees, for one head
    pairs = keys = 0
    lq, lk = _lengths(case)
    s = case["sinks"]
    for nq, nk in zip(lq, lk):
        p = torch.arange(nk - nq, nk, dtype=torch.int64)
        hi = (p + case["right"] + 1).clamp(0, nk) if case["right"] >= 0 else torch.full_like(p, nk)
        lo = (p - case["left"]).clamp(0, nk) if case["left"] >= 0 else torch.zeros_like(p)
        pairs += int(((hi - lo).clamp_min(0) + torch.minimum(hi, lo).clamp_max(s)).sum())
        if nq and nk:
            first, last = int(lo[0]), int(hi[-1])
            keys += max(0, last - first) + min(s, first, last)
    return {"bytes": e * case["dim"] * (2 * sum(lq) * case["q_heads"] + 2 * keys * case["k_heads"]),
            "flops": 4 * case["dim"] * case["q_heads"] * pairs}


# ------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    def of_act(v, act):
        if act == "relu":
            return torch.where(v > 0, v, torch.zeros_like(v))
        if act == "gelu":
            return v * torch.special.ndtr(v)
        if act == "gelu_tanh":
            return v * torch.sigmoid(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))
        if act == "silu":
            return v * torch.sigmoid(v)
        return v

    def of_linear(s):
        out = torch.empty(s["x"].shape[0], s["weight"].shape[0], dtype=torch.float64, device=DEV)
        wt = s["weight"].double().t()
        for at in range(0, out.shape[0], 8192):
            v = s["x"][at:at + 8192].double() @ wt
            if s["bias"] is not None:
                v = v + s["bias"].double()
            v = of_act(v, s["case"]["act"])
            out[at:at + 8192] = v if s["residual"] is None else v + s["residual"][at:at + 8192].double()
        return out

    def of_rotate(s):
        c = s["case"]
        half, f = c["dim"] // 2, c["dim"] // 2 // 3
        speed = [c["base"] ** (-(j % f) / f) if j < 3 * f else 0.0 for j in range(half)]
        axis = torch.tensor([min(j // f, 2) for j in range(half)], device=DEV)
        angle = s["positions"].double()[:, axis] * torch.tensor(speed, dtype=torch.float64, device=DEV)
        spin = torch.polar(torch.ones_like(angle), angle)[:, None]
        outs = []
        for x, weight in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
            for at in range(0, x.shape[0], 65536):
                v = x[at:at + 65536].double()
                v = v * torch.rsqrt(v.square().sum(-1, keepdim=True) / c["dim"] + EPS)
                if weight is not None:
                    v = v * weight.double()
                first, second = (slice(0, None, 2), slice(1, None, 2)) if c["interleaved"] else \
                    (slice(0, half), slice(half, None))
                z = torch.complex(v[..., first].contiguous(), v[..., second].contiguous())
                z = z * spin[at:at + 65536]
                out[at:at + 65536][..., first] = z.real
                out[at:at + 65536][..., second] = z.imag
            outs.append(out)
        return tuple(outs)

    def of_attend(s):
        """Sample by sample, head by head, a few hundred queries at a time against
        the keys between the first and the last that any of them sees."""
        c = s["case"]
        group, scale = c["q_heads"] // c["k_heads"], 1 / math.sqrt(c["dim"])
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        q0 = k0 = 0
        for nq, nk in zip(*_lengths(c)):
            for a in range(0, nq if nk else 0, 512):
                b = min(nq, a + 512)
                p = torch.arange(a, b, device=DEV)[:, None] + (nk - nq)
                lo = max(0, a + nk - nq - c["left"]) if c["left"] >= 0 else 0
                hi = min(nk, b + nk - nq + c["right"]) if c["right"] >= 0 else nk
                j = torch.tensor(sorted(set(range(min(c["sinks"], nk))) | set(range(lo, hi))),
                                 dtype=torch.long, device=DEV)
                if not len(j):
                    continue
                hidden = torch.zeros(b - a, len(j), dtype=torch.bool, device=DEV)
                if c["left"] >= 0:
                    hidden |= (j < p - c["left"]) & (j >= c["sinks"])
                if c["right"] >= 0:
                    hidden |= j > p + c["right"]
                q = s["q"][q0 + a:q0 + b].double().view(b - a, c["k_heads"], group, -1)
                q = q.permute(1, 2, 0, 3).reshape(c["k_heads"], group * (b - a), -1)
                k, v = (s[t][k0 + j].double().permute(1, 0, 2) for t in "kv")
                w = (torch.bmm(q, k.transpose(1, 2).contiguous()) * scale).view(
                    c["k_heads"], group, b - a, len(j))
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                w = w.masked_fill(hidden.all(1)[:, None], 0.0).view(c["k_heads"], -1, len(j))
                o = torch.bmm(w, v.contiguous()).view(c["k_heads"], group, b - a, -1)
                out[q0 + a:q0 + b] = o.permute(2, 0, 1, 3).reshape(b - a, c["q_heads"], -1)
            q0, k0 = q0 + nq, k0 + nk
        return out

    s = prepare(case, seed)
    return {"linear": of_linear, "rotate": of_rotate, "attend": of_attend}[case["op"]](s)
