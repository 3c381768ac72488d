"""window_attention against its 64-bit form."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import attend64, check, seen

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _qkv(lq, lk, hq, hk, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + sum(lq) + 3 * sum(lk) + dim)
    q = torch.randn(sum(lq), hq, dim, generator=g).to(dtype)
    k, v = (torch.randn(sum(lk), hk, dim, generator=g).to(dtype) for _ in range(2))
    return q, k, v


def _offsets(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)


def _run(q, k, v, lq, lk, window, sinks, **kw):
    return spconv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), _offsets(lq), _offsets(lk),
                                   window=window, sinks=sinks, **kw)


# (queries, keys) of each sample, window, sinks
LENGTHS = [
    ([1], [1], (None, None), 0),
    ([3, 0, 5], [3, 0, 5], (1, 1), 0),
    ([2, 4], [0, 4], (None, None), 2),                  # a sample without keys
    ([9, 3], [2, 3], (1, 0), 1),                        # queries before every key: empty rows
    ([1, 1, 1, 1], [700, 1, 64, 129], (100, 0), 4),     # one new token each
    ([1], [3000], (None, 0), 0),
    ([2, 1], [1500, 4000], (None, None), 0),
    ([5, 33], [200, 300], (40, 0), 3),
    ([63, 64, 65], [63, 64, 65], (None, 0), 0),
    ([127, 130, 1], [127, 130, 1], (16, 16), 0),
    ([300], [300], (0, 0), 0),                          # each its own key only
    ([257, 190], [257, 190], (31, 64), 5),
    ([400, 100], [500, 350], (128, 0), 16),
    ([520], [520], (64, None), 2),
    ([350], [350], (5, 3), 200),                        # sinks wider than a tile
    ([1000], [1000], (100, 100), 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,lk,window,sinks", LENGTHS)
def test_lengths_and_windows(lq, lk, window, sinks, dtype):
    for hq, hk, dim in ((2, 2, 64), (4, 1, 32)):
        say("window_attention:", lq, lk, window, sinks, hq, hk, dim, dtype)
        q, k, v = _qkv(lq, lk, hq, hk, dim, dtype)
        got = _run(q, k, v, lq, lk, window, sinks)
        assert got.dtype == dtype and got.is_contiguous()
        check(got, *attend64(q, k, v, lq, lk, window, sinks), what=f"{hq} {hk} {dim}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,dim", [(1, 1, 1), (2, 1, 7), (3, 3, 16), (6, 2, 24), (5, 1, 40),
                                       (2, 2, 48), (4, 4, 72), (2, 1, 80), (3, 1, 96), (2, 2, 100),
                                       (8, 2, 128), (2, 1, 136), (1, 1, 200), (2, 1, 256)])
def test_heads(hq, hk, dim, dtype):
    say("window_attention heads:", hq, hk, dim, dtype)
    for lq, lk, window, sinks in (([150, 77], [150, 77], (50, 20), 3), ([1, 2], [333, 90], (None, 0), 0)):
        q, k, v = _qkv(lq, lk, hq, hk, dim, dtype)
        check(_run(q, k, v, lq, lk, window, sinks), *attend64(q, k, v, lq, lk, window, sinks),
              what=f"{lq}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_and_scale(dtype):
    """Scores of some hundreds, rising and falling along the keys, so that the
    running maximum moves often; and a scale of the caller's, negative too."""
    lq = lk = [300]
    q, k, v = _qkv(lq, lk, 2, 2, 64, dtype)
    ramp = torch.linspace(-1, 1, 300)[:, None, None]
    for factor in (ramp * 20, -ramp * 20, 20 * torch.sin(20 * ramp)):
        kk = (k.float() * factor).to(dtype)
        check(_run(q, kk, v, lq, lk, (None, None), 0), *attend64(q, kk, v, lq, lk, (None, None), 0))
    for scale in (0.0, 0.5, -0.3):
        check(_run(q, k, v, lq, lk, (50, 50), 0, scale=scale),
              *attend64(q, k, v, lq, lk, (50, 50), 0, scale=scale), what=f"scale {scale}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """Views of a packed projection, head-major tensors and tensors aligned to
    their elements only give the bits of contiguous ones."""
    lq = lk = [130, 61]
    q, k, v = _qkv(lq, lk, 4, 2, 64, dtype)
    want = _run(q, k, v, lq, lk, (40, 30), 2)
    packed = torch.cat([q, k, v], 1).to(DEV)
    off = _offsets(lq)
    got = spconv.window_attention(packed[:, :4], packed[:, 4:6], packed[:, 6:], off,
                                  window=(40, 30), sinks=2)
    assert torch.equal(got, want)
    for pad in (1, 2, 8):
        room = [torch.full((*t.shape[:2], t.shape[2] + pad), float("nan"), dtype=dtype, device=DEV)
                for t in (q, k, v)]
        for r, t in zip(room, (q, k, v)):
            r[..., pad:] = t.to(DEV)
        got = spconv.window_attention(*(r[..., pad:] for r in room), off, window=(40, 30), sinks=2)
        assert torch.equal(got, want), pad
    major = [t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(spconv.window_attention(*major, off, window=(40, 30), sinks=2), want)
    spread = torch.zeros(2 * len(off), dtype=torch.int32, device=DEV)
    spread[::2] = off
    assert torch.equal(spconv.window_attention(*major, spread[::2], window=(40, 30), sinks=2), want)
    # a key and value for all heads and rows, by a stride of zero
    one = k[:1, :1].to(DEV)
    got = spconv.window_attention(q.to(DEV), one.expand(191, 2, 64), v.to(DEV), off, window=(40, 30))
    check(got, *attend64(q, k[:1, :1].expand(191, 2, 64), v, lq, lk, (40, 30), 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,lk", [([200, 90], [200, 90]), ([1, 1], [500, 300]), ([3], [4000])])
def test_unseen_keys_may_hold_anything(lq, lk, dtype):
    """NaN and infinities at keys: the queries that do not see them keep their
    bits, those that do are not finite."""
    window, sinks = (20, 10), 2
    q, k, v = _qkv(lq, lk, 4, 2, 64, dtype)
    clean = _run(q, k, v, lq, lk, window, sinks).cpu()
    bad = [5, sum(lk) - 60, 70, lk[0] - 1]
    for j, x in zip(bad, (float("nan"), float("inf"), float("-inf"), float("nan"))):
        k[j], v[j] = x, x
    got = _run(q, k, v, lq, lk, window, sinks).cpu()
    hit = torch.zeros(sum(lq), dtype=torch.bool)
    q0 = k0 = 0
    for nq, nk in zip(lq, lk):
        ok = seen(nq, nk, *window, sinks)
        for j in bad:
            if k0 <= j < k0 + nk:
                hit[q0:q0 + nq] |= ok[:, j - k0]
        q0, k0 = q0 + nq, k0 + nk
    check(got[~hit], clean[~hit].double(), torch.zeros_like(clean[~hit], dtype=torch.float64))
    assert not torch.isfinite(got[hit]).all(-1).any()


def test_values_only_non_finite():
    """An infinite value reaches the queries that see it, as an infinity."""
    lq = lk = [100]
    q, k, v = _qkv(lq, lk, 1, 1, 32, torch.float16)
    v[50, 0, 3] = float("inf")
    got = _run(q, k, v, lq, lk, (5, 5), 0).cpu()[:, 0]
    near = torch.zeros(100, dtype=torch.bool)
    near[45:56] = True
    assert (got[near, 3] == float("inf")).all() and torch.isfinite(got[~near]).all()
    others = [d for d in range(32) if d != 3]
    assert torch.isfinite(got[:, others]).all()


def test_scores_of_minus_infinity():
    """A seen key whose score is -inf has no weight; a query with no other
    seen key gives zeros."""
    q = torch.ones(2, 1, 32, dtype=torch.float16)
    k = torch.ones(2, 1, 32, dtype=torch.float16)
    k[0] = float("-inf")
    v = torch.full((2, 1, 32), 3.0, dtype=torch.float16)
    got = _run(q, k, v, [2], [2], (None, 0), 0).cpu()
    assert (got[0] == 0).all() and (got[1] == 3).all()


def test_offsets_out_of_range_touch_nothing_outside():
    """Offsets that lie are cut to the tensors."""
    q, k, v = (t.to(DEV) for t in _qkv([64], [64], 1, 1, 32, torch.float16))
    for bad in ([0, 1 << 30], [-(1 << 30), 64], [64, 0], [1 << 30, -5]):
        off = torch.tensor(bad, dtype=torch.int32, device=DEV)
        assert spconv.window_attention(q, k, v, off, window=(8, 8)).shape == q.shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("lq,lk", [([3000, 2100], [3000, 2100]), ([1, 1], [9000, 5000])])
def test_same_bits_every_time_on_any_stream(lq, lk):
    q, k, v = (t.to(DEV) for t in _qkv(lq, lk, 4, 2, 64, torch.bfloat16))
    oq, ok = _offsets(lq), _offsets(lk)

    def go():
        return spconv.window_attention(q, k, v, oq, ok, window=(300, 200), sinks=4)

    want = go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = go()
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(go(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_samples(dtype):
    """More samples than lanes of a wave, most of them tiny, some empty."""
    lk = [(7 * i) % 23 for i in range(300)]
    q, k, v = _qkv(lk, lk, 2, 2, 32, dtype)
    check(_run(q, k, v, lk, lk, (4, 4), 1), *attend64(q, k, v, lk, lk, (4, 4), 1))


def test_long_sample_far_rows():
    """Rows past 2^31 bytes of the key tensor, reached through its strides:
    one key every 600 kB."""
    n, stride = 4000, 300_000
    q, k, v = _qkv([1], [n], 1, 1, 64, torch.float16)
    room = torch.zeros(n * stride, dtype=torch.float16, device=DEV)
    wide = room.view(n, 1, stride)
    wide[..., :64], wide[..., 64:128] = k.to(DEV), v.to(DEV)
    got = spconv.window_attention(q.to(DEV), wide[..., :64], wide[..., 64:128], _offsets([1]),
                                  _offsets([n]), window=(None, None))
    check(got, *attend64(q, k, v, [1], [n], (None, None), 0))


def test_refusals():
    q, k, v = (t.to(DEV) for t in _qkv([8], [8], 4, 2, 16, torch.float16))
    off = _offsets([8])
    f = spconv.window_attention
    with pytest.raises(RuntimeError, match="GPU"):
        f(q.cpu(), k, v, off)
    with pytest.raises(TypeError, match="unsupported dtype"):
        f(q.double(), k.double(), v.double(), off)
    with pytest.raises(ValueError, match="are not"):
        f(q, k, v[:7], off)
    with pytest.raises(ValueError, match="v is"):
        f(q, k, v.float(), off)
    with pytest.raises(ValueError, match="evenly"):
        f(q[:, :3], k, v, off)
    with pytest.raises(ValueError, match="need offsets_k"):
        f(q[:5], k, v, off)
    with pytest.raises(ValueError, match="int32"):
        f(q, k, v, off.long())
    with pytest.raises(ValueError, match="int32"):
        f(q, k, v, off, off.cpu())
    with pytest.raises(ValueError, match="offsets must be"):
        f(q, k, v, off, _offsets([4, 4]))
    with pytest.raises(ValueError, match="negative"):
        f(q, k, v, off, window=(-1, 0))
    with pytest.raises(ValueError, match="sinks"):
        f(q, k, v, off, sinks=-1)
    big = torch.zeros(8, 1, 257, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="head size"):
        f(big, big, big, off)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_outgrow_their_reference(dtype):
    """Keys in rising blocks: each block's scores exceed all before by more than
    the weights may grow, then fall back; split keys as well."""
    steps = torch.tensor([0.0, 3.0, 9.0, 4.0, 20.0, 19.0, 40.0, 0.0]).repeat_interleave(70)
    for lq, lk in (([560], [560]), ([2], [560])):
        q, k, v = _qkv(lq, lk, 2, 2, 64, dtype)
        q = torch.full_like(q, 0.5)
        k = (0.1 * k.float() + steps[:, None, None] / 4).to(dtype)
        check(_run(q, k, v, lq, lk, (None, None), 0), *attend64(q, k, v, lq, lk, (None, None), 0))


def test_many_streams_of_one_token():
    lq, lk = [1] * 300, [5 + (i * 37) % 200 for i in range(300)]
    q, k, v = _qkv(lq, lk, 8, 2, 64, torch.bfloat16)
    check(_run(q, k, v, lq, lk, (63, 0), 2), *attend64(q, k, v, lq, lk, (63, 0), 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 200])
def test_long_tail_of_small_weights(queries, dtype):
    """One key 12 above thousands of others, which together still make up a
    thirtieth of the sum: their weights keep their accuracy in 16 bits."""
    n = 6000
    q, k, v = _qkv([queries], [n], 1, 1, 32, dtype)
    q, k, v = torch.zeros_like(q), torch.zeros_like(k), torch.ones_like(v)
    q[..., 0], k[3, 0, 0], v[3] = 1.0, 12.0, 0.0
    check(_run(q, k, v, [queries], [n], (None, None), 0, scale=1.0),
          *attend64(q, k, v, [queries], [n], (None, None), 0, scale=1.0))


@pytest.mark.parametrize("lq,lk", [([0], [0]), ([0, 0], [5, 3]), ([], [])])
def test_no_queries(lq, lk):
    q, k, v = _qkv(lq, lk, 4, 2, 16, torch.float16)
    assert _run(q, k, v, lq, lk, (None, None), 0).shape == (0, 4, 16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,lk", [([300, 70], [300, 70]), ([2, 1], [900, 4000])])
def test_rows_of_no_sample(lq, lk, dtype):
    """Rows before the first sample and behind the last give zeros, with the
    keys split and without; the samples' rows are as they would be alone."""
    q, k, v = _qkv(lq, lk, 4, 2, 64, dtype)
    want = _run(q, k, v, lq, lk, (900, 30), 2)
    pad = torch.full((5, 4, 64), float("nan"), dtype=dtype)
    wide = torch.cat([pad, q, pad, pad]).to(DEV)
    torch.full_like(wide, float("nan"))  # what the outputs' memory may hold
    got = spconv.window_attention(wide, k.to(DEV), v.to(DEV), _offsets(lq) + 5, _offsets(lk),
                                  window=(900, 30), sinks=2)
    assert (got[:5] == 0).all() and (got[-10:] == 0).all()
    check(got[5:-10], *attend64(q, k, v, lq, lk, (900, 30), 2))
    check(want, *attend64(q, k, v, lq, lk, (900, 30), 2))


def test_no_samples():
    q, k, v = (t.to(DEV) for t in _qkv([40], [40], 4, 2, 64, torch.float16))
    torch.full_like(q, float("nan"))
    off = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert (spconv.window_attention(q, k, v, off) == 0).all()
