"""The calls of a stream of voxels that keeps its keys and values in pages: what
is timed, over which sizes.

A case is a dict of plain values.  ``op`` names the operator:

    append  RMS norm of every query and key head, rotation by the      spconv.norm_rotate_append
            voxel's coordinates, keys and values into their pages
    attend  attention of the new rows over each sample's pages, in a   spconv.cache_attention
            window, the first ``sinks`` keys always visible
    shared  the same where all samples begin with the same pages,      spconv.cache_attention
            which are read once for all                                (prefix=)

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
EPS = 1e-6
# extents (z, y, x) of the grids that the coordinates come from
LIDAR, OBJECT, SCENE = "41x1600x1408", "64x64x64", "256x256x256"
GRIDS = (OBJECT, "160x160x160", SCENE, LIDAR)


def _append(samples, rows, fewer, kept, q_heads, k_heads, dim, dtype, page, grid, gain="dim",
            interleaved=False, base=10000.0):
    """Sample b brings rows - b*fewer new rows behind kept + 7 b that it holds."""
    return {"op": "append", "samples": samples, "rows": rows, "fewer": fewer, "kept": kept,
            "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "dtype": dtype, "page": page,
            "grid": grid, "gain": gain, "interleaved": interleaved, "base": base}


def _attend(samples, keys, fewer, rows, fewer_rows, q_heads, k_heads, dim, dtype, page, left=-1,
            right=0, sinks=0):
    """Sample b's last rows - b*fewer_rows (one at least) of keys - b*fewer
    positions are new; left or right -1: no limit."""
    return {"op": "attend", "samples": samples, "keys": keys, "fewer": fewer, "rows": rows,
            "fewer_rows": fewer_rows, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "dtype": dtype, "page": page, "left": left, "right": right, "sinks": sinks, "prefix": 0}


def _shared(samples, prefix, keys, fewer, rows, q_heads, k_heads, dim, dtype, page, left=-1,
            sinks=0):
    """prefix pages for all, then keys - b*fewer positions of sample b's own."""
    return {"op": "shared", "samples": samples, "keys": keys, "fewer": fewer, "rows": rows,
            "fewer_rows": 0, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "dtype": dtype,
            "page": page, "left": left, "right": 0, "sinks": sinks, "prefix": prefix}


def listed():
    cases = [
        # one new token for each of four streams: all latency
        ("append_token", _append(4, 1, 0, 2000, 16, 4, 64, "bf16", 64, SCENE)),
        # two small scenes in the default precision, nothing kept yet
        ("append_f32_2x10k", _append(2, 10_007, 1003, 0, 6, 6, 32, "f32", 64, LIDAR, gain="head")),
        # the next sweep of four LiDAR streams
        ("append_4x60k", _append(4, 60_000, 1013, 15_000, 12, 12, 64, "f16", 64, LIDAR)),
        # one new token for each of four young streams
        ("attend_token_4x900", _attend(4, 900, 113, 1, 0, 16, 4, 64, "bf16", 64)),
        # streams that keep a scan and look at its last rows and the register tokens in front
        ("attend_token_window", _attend(24, 60_000, 1013, 1, 0, 16, 4, 64, "f16", 64, 4095, 0, 16)),
        # a decoder at work on many scenes of different lengths
        ("attend_token_64x32k", _attend(64, 32_768, 301, 1, 0, 16, 4, 64, "bf16", 64)),
        # the default precision, narrow heads without sharing
        ("attend_token_f32", _attend(16, 10_007, 401, 1, 0, 6, 6, 32, "f32", 64)),
        # streams that bring different numbers of voxels at once, one of them next to none
        ("attend_chunks_20k", _attend(4, 20_000, 1777, 512, 170, 16, 4, 64, "bf16", 64)),
        # the largest steps over two whole scenes, wide heads
        ("attend_chunks_32k", _attend(2, 32_000, 1003, 2048, 40, 16, 4, 128, "bf16", 64)),
        # eight objects drawn from one condition, voxel by voxel
        ("shared_token_8x2k", _shared(8, 32, 150, 13, 1, 16, 4, 64, "bf16", 64)),
        # many continuations of one scene
        ("shared_token_64x32k", _shared(64, 512, 1000, 13, 1, 16, 4, 64, "bf16", 64)),
        # the same with a block of voxels a step
        ("shared_rows_16x8k", _shared(16, 128, 600, 31, 24, 8, 8, 64, "f16", 64)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["op"], {"bytes": 0, "flops": 0})
        for k in m:
            m[k] = max(m[k], w[k])
    op = rng.choice(("append", "attend", "attend", "shared"))
    while True:
        dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
        k = rng.choice((1, 2, 3, 4, 6, 8))
        q = k * rng.choice((1, 1, 2, 4, 8))
        dim = rng.choice((16, 32, 40, 64, 64, 80, 96, 128))
        page = rng.choice((16, 32, 64, 64, 64, 128, 20, 48))
        if op == "append":
            rows = _log(rng, 1, 60_000)
            samples = _log(rng, 1, 64)
            c = _append(samples, rows, rng.randint(0, rows // samples), _log(rng, 1, 8000), q, k,
                        dim, dtype, page, rng.choice(GRIDS), rng.choice(("none", "dim", "head")),
                        rng.random() < 0.3, rng.choice((100.0, 10000.0)))
            fits = sum(_lengths(c)[1]) * k * dim <= 240_000 * 12 * 64
        elif op == "attend":
            rows = rng.choice((1, 1, 1, rng.randint(2, 64), _log(rng, 64, 2048)))
            samples = _log(rng, 1, 64 if rows == 1 else 8)
            keys = rows + _log(rng, 1, 32_000)
            left = _log(rng, 16, 4096) if rng.random() < 0.4 else -1
            c = _attend(samples, keys, rng.randint(0, (keys - rows) // samples), rows,
                        rng.randint(0, rows // samples), q, k, dim, dtype, page, left,
                        rng.choice((0, 0, -1)), rng.choice((0, 0, 4, 16)))
            fits = samples * q * rows * _span(c) <= 2_100_000_000
        else:
            rows = rng.choice((1, 1, 1, rng.randint(2, 32)))
            keys = rows + _log(rng, 1, 2000)
            samples = _log(rng, 2, 64)
            c = _shared(samples, max(1, _log(rng, 64, 32_768) // page), keys,
                        rng.randint(0, (keys - rows) // samples), rows, q, k, dim, dtype, page,
                        _log(rng, 256, 8192) if rng.random() < 0.2 else -1,
                        rng.choice((0, 0, 16)))
            fits = True
        w = work(c)
        # products in the default precision run on a slower unit
        slow = {"bytes": 1, "flops": 8 if dtype == "f32" else 1}
        if fits and all(w[k] <= most[op][k] / slow[k] for k in w):
            return c


# ----------------------------------------------------------------- inputs
def _lengths(c):
    """(new rows, positions with them) of each sample."""
    if c["op"] == "append":
        lq = [max(0, c["rows"] - b * c["fewer"]) for b in range(c["samples"])]
        return lq, [c["kept"] + 7 * b + n for b, n in enumerate(lq)]
    lq = [max(1, c["rows"] - b * c["fewer_rows"]) for b in range(c["samples"])]
    first = c["prefix"] * c["page"]
    return lq, [first + max(n, c["keys"] - b * c["fewer"]) for b, n in enumerate(lq)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(c, g):
    """Page numbers (samples, most pages of a sample) and the pages there are:
    in no order, as samples come and go, and some of them free."""
    _, lk = _lengths(c)
    P, R = c.get("prefix", 0), c["page"]
    counts = [max(0, -(-n // R) - P) for n in lk]
    total = P + sum(counts)
    total += total // 16 + 1
    ids = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    at = _ints([P, *(P + n for n in itertools.accumulate(counts))])[:-1, None]
    j = torch.arange(max(max(counts), 1), device=DEV)
    table = ids[(at + torch.minimum(j, _ints(counts)[:, None] - 1).clamp_min(0)).clamp_max(total - 1).long()]
    return torch.cat([ids[:P].expand(c["samples"], P), table], 1).contiguous(), total


def prepare(case, seed):
    """What a stream has in hand at the call: its pages, where each sample's are,
    and the new rows."""
    g = torch.Generator(DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hk, d, R = case["q_heads"], case["k_heads"], case["dim"], case["page"]

    def randn(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dt)

    lq, lk = _lengths(case)
    s = {"case": case}
    s["table"], pages = _pages(case, g)
    # the rows of a head lie together in a page
    s["k_pages"], s["v_pages"] = (randn(pages, hk, R, d).transpose(1, 2) for _ in range(2))
    s["offsets"] = _ints([0, *itertools.accumulate(lq)])
    s["lengths"] = _ints(lk)
    if case["op"] != "append":
        s["q"] = randn(sum(lq), hq, d)
        s["prefix"] = s["table"][0, :case["prefix"]].clone() if case["op"] == "shared" else None
        return s
    # queries, keys and values lie side by side, as one projection leaves them
    n = sum(lq)
    qkv = randn(n, hq + 2 * hk, d, scale=2.0)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    z, y, x = (int(v) for v in case["grid"].split("x"))
    cell = torch.randint(0, z * y * x, (n,), generator=g, device=DEV)
    coords = torch.stack([torch.zeros_like(cell), cell // (y * x), cell // x % y, cell % x], 1)
    s["positions"] = coords.to(torch.int32)[:, 1:]  # (z, y, x) of (b, z, y, x) rows
    gain = {"none": None, "dim": (d,), "head": (None, d)}[case["gain"]]
    for name, h in (("q_weight", hq), ("k_weight", hk)):
        s[name] = None if gain is None else \
            randn(*[h if v is None else v for v in gain], scale=0.1, shift=1.0)
    return s


# ------------------------------------------------------------ plain forms
def _plain_append(s):
    c = s["case"]
    d, R = c["dim"], c["page"]
    f = d // 2 // 3  # pairs per axis
    i = torch.arange(f, device=DEV, dtype=torch.float64)
    turn = s["positions"].double()[:, :, None] * c["base"] ** (-i / f)  # (rows, axes, f)
    turn = torch.nn.functional.pad(turn.flatten(1), (0, d // 2 - 3 * f))[:, None]
    cos, sin = torch.cos(turn).float(), torch.sin(turn).float()

    def one(x, weight):
        v = x.float()
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
        if weight is not None:
            v = v * weight.float()
        if c["interleaved"]:
            a, b = v[..., 0::2], v[..., 1::2]
            return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2).to(x.dtype)
        a, b = v[..., :d // 2], v[..., d // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)

    row = torch.arange(s["q"].shape[0], device=DEV)
    off = s["offsets"].long()
    b = torch.searchsorted(off, row, right=True) - 1
    at = row - off[b + 1] + s["lengths"].long()[b]
    page = s["table"].long()[b, at // R]
    s["k_pages"][page, at % R] = one(s["k"], s["k_weight"])
    s["v_pages"][page, at % R] = s["v"]
    return one(s["q"], s["q_weight"]), s["k_pages"], s["v_pages"]


def _span(c):
    """Positions that the plain form takes of a sample behind the prefix and the
    sinks: the longest sample's, or what a window and its rows can reach."""
    lq, lk = _lengths(c)
    most = max(lk) - c["prefix"] * c["page"]
    return most if c["left"] < 0 or c["prefix"] else min(most, max(lq) + c["left"])


def _plain_attend(s):
    """Every sample padded to the most rows and keys; the prefix once."""
    c = s["case"]
    lq, _ = _lengths(c)
    B, hq, hk, d, R = c["samples"], c["q_heads"], c["k_heads"], c["dim"], c["page"]
    G, rows, span, P = hq // hk, max(lq), _span(c), c["prefix"]
    off, n_k = s["offsets"].long(), s["lengths"].long()
    n_q, table = off.diff(), s["table"].long()
    i = torch.arange(rows, device=DEV)
    pos = i + (n_k - n_q)[:, None]                                          # (B, rows)
    there = i < n_q[:, None]
    q = s["q"].float()[(i + off[:-1, None]).clamp_max(s["q"].shape[0] - 1)]
    q = q.view(B, rows, hk, G, d).permute(0, 2, 3, 1, 4)                    # (B, hk, G, rows, d)
    j = torch.arange(span, device=DEV).expand(B, span)
    banded = P == 0 and c["left"] >= 0 and span < max(_lengths(c)[1])
    if banded:
        j = j + (pos[:, :1] - c["left"]).clamp_min(0)
    j = j + P * R
    sinks = torch.arange(c["sinks"] if banded else 0, device=DEV).expand(B, -1)

    def seen(j, near, far=None):
        at, p = j[:, None, :], pos[:, :, None]
        ok = at < n_k[:, None, None]
        if c["right"] >= 0:
            ok = ok & (at <= p + c["right"])
        if c["left"] >= 0:
            inside = at >= p - c["left"]
            # a sink inside the window is counted there, and not again in its own column
            ok = ok & (inside if near else ~inside if far else inside | (at < c["sinks"]))
        return ok[:, None, None]

    if banded:
        sees = torch.cat([seen(j, True), seen(sinks, False, True)], -1)
        j = torch.cat([j, sinks], 1)
    else:
        sees = seen(j, False)
    page = torch.gather(table, 1, (j // R).clamp_max(table.shape[1] - 1))
    k = s["k_pages"][page, j % R].float().permute(0, 2, 3, 1)               # (B, hk, d, keys)
    v = s["v_pages"][page, j % R].float().permute(0, 2, 1, 3)               # (B, hk, keys, d)
    w = torch.matmul(q.reshape(B, hk, G * rows, d), k).view(B, hk, G, rows, -1) * d ** -0.5
    w = w.masked_fill(~sees, -math.inf)
    top = w.amax(-1, keepdim=True)
    if P:
        jp = torch.arange(P * R, device=DEV)
        at = s["prefix"].long()[jp // R]
        kp = s["k_pages"][at, jp % R].float().permute(1, 2, 0)              # (hk, d, prefix)
        vp = s["v_pages"][at, jp % R].float().permute(1, 0, 2)              # (hk, prefix, d)
        qp = q.permute(1, 0, 2, 3, 4).reshape(hk, B * G * rows, d)
        wp = torch.matmul(qp, kp).view(hk, B, G, rows, P * R).transpose(0, 1) * d ** -0.5
        wp = wp.masked_fill(~seen(jp.expand(B, -1), False), -math.inf)
        top = torch.maximum(top, wp.amax(-1, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0.0)
    w = torch.exp(w - top)
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, hk, G * rows, -1), v).view(B, hk, G, rows, d)
    if P:
        wp = torch.exp(wp - top)
        total = total + wp.sum(-1, keepdim=True)
        op = torch.matmul(wp.transpose(0, 1).reshape(hk, B * G * rows, P * R), vp)
        o = o + op.view(hk, B, G, rows, d).transpose(0, 1)
    o = o / total.masked_fill(total == 0, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, rows, hq, d)[there].to(s["q"].dtype)


def run(state):
    c = state["case"]
    if not own:
        return _plain_append(state) if c["op"] == "append" else _plain_attend(state)
    import trispconv.pytorch as spconv
    cache = [state[n] for n in ("k_pages", "v_pages", "table", "offsets", "lengths")]
    if c["op"] == "append":
        q = spconv.norm_rotate_append(state["q"], state["k"], state["v"], state["positions"],
                                      *cache, q_weight=state["q_weight"],
                                      k_weight=state["k_weight"], eps=EPS, base=c["base"],
                                      interleaved=c["interleaved"])
        return q, state["k_pages"], state["v_pages"]
    window = tuple(None if v < 0 else v for v in (c["left"], c["right"]))
    return spconv.cache_attention(state["q"], *cache, prefix=state["prefix"], window=window,
                                  sinks=c["sinks"])


# ------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    lq, lk = _lengths(case)
    hq, hk, d, R = case["q_heads"], case["k_heads"], case["dim"], case["page"]
    if case["op"] == "append":
        n = sum(lq)
        # squares and their sum, the norm's two products, four products and two sums for a pair
        return {"bytes": 2 * e * n * (hq + 2 * hk) * d + 12 * n, "flops": 7 * n * (hq + hk) * d}
    # pairs of a query and a key it sees, and keys that some query sees, for one head
    pairs = keys = 0
    s, first, prefix = case["sinks"], case["prefix"] * R, None
    for nq, nk in zip(lq, lk):
        p = torch.arange(nk - nq, nk, dtype=torch.int64)
        hi = (p + case["right"] + 1).clamp(0, nk) if case["right"] >= 0 else torch.full_like(p, nk)
        lo = (p - case["left"]).clamp(0, nk) if case["left"] >= 0 else torch.zeros_like(p)
        pairs += int(((hi - lo).clamp_min(0) + torch.minimum(hi, lo).clamp_max(s)).sum())
        a, b = int(lo[0]), int(hi[-1])
        keys += max(0, b - max(a, first)) + max(0, min(s, a, b) - first)
        prefix = a if prefix is None else min(prefix, a)
    keys += max(0, first - prefix) + min(s, prefix, first)
    return {"bytes": e * d * (2 * sum(lq) * hq + 2 * keys * hk), "flops": 4 * d * hq * pairs}


# ------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    R, d, hk = case["page"], case["dim"], case["k_heads"]
    lq, lk = _lengths(case)
    table = s["table"].tolist()

    def places(b, lo, hi):
        """(pages, rows of them) of sample b's positions lo to hi."""
        j = torch.arange(lo, hi, device=DEV)
        return torch.tensor(table[b], device=DEV)[j // R], j % R

    if case["op"] == "append":
        half, f = d // 2, d // 2 // 3
        speed = [case["base"] ** (-(j % f) / f) if j < 3 * f else 0.0 for j in range(half)]
        axis = torch.tensor([min(j // f, 2) for j in range(half)], device=DEV)
        angle = s["positions"].double()[:, axis] * torch.tensor(speed, dtype=torch.float64, device=DEV)
        spin = torch.polar(torch.ones_like(angle), angle)[:, None]
        first, second = (slice(0, None, 2), slice(1, None, 2)) if case["interleaved"] else \
            (slice(0, half), slice(half, None))

        def turned(x, weight):
            v = x.double()
            v = v * torch.rsqrt(v.square().sum(-1, keepdim=True) / d + EPS)
            if weight is not None:
                v = v * weight.double()
            z = torch.complex(v[..., first].contiguous(), v[..., second].contiguous()) * spin
            out = torch.empty_like(v)
            out[..., first], out[..., second] = z.real, z.imag
            return out

        k, v = turned(s["k"], s["k_weight"]), s["v"].double()
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        at = 0
        for b, (n, end) in enumerate(zip(lq, lk)):
            where = places(b, end - n, end)
            k_pages[where], v_pages[where] = k[at:at + n], v[at:at + n]
            at += n
        return turned(s["q"], s["q_weight"]), k_pages, v_pages

    # sample by sample, head by head, some rows at a time against every key of theirs
    group, scale = case["q_heads"] // hk, 1 / math.sqrt(d)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, end) in enumerate(zip(lq, lk)):
        where = places(b, 0, end)
        k, v = (s[t][where].double().permute(1, 0, 2).contiguous() for t in ("k_pages", "v_pages"))
        kt, j = k.transpose(1, 2).contiguous(), torch.arange(end, device=DEV)
        for a in range(0, n, 256):
            m = min(n, a + 256) - a
            p = torch.arange(a, a + m, device=DEV)[:, None] + (end - n)
            hidden = torch.zeros(m, end, dtype=torch.bool, device=DEV)
            if case["left"] >= 0:
                hidden |= (j < p - case["left"]) & (j >= case["sinks"])
            if case["right"] >= 0:
                hidden |= j > p + case["right"]
            q = s["q"][at + a:at + a + m].double().view(m, hk, group, d)
            q = q.permute(1, 2, 0, 3).reshape(hk, group * m, d)
            w = (torch.bmm(q, kt) * scale).view(hk, group, m, end).masked_fill(hidden, -math.inf)
            o = torch.bmm(torch.softmax(w, -1).view(hk, group * m, end), v)
            out[at + a:at + a + m] = o.view(hk, group, m, d).permute(2, 0, 1, 3).reshape(m, -1, d)
        at += n
    return out
