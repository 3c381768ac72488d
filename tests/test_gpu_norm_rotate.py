"""norm_rotate_heads against its 64-bit form."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import check, rotate64

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _heads(n, hq, hk, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + n + dim)
    packed = (torch.randn(n, hq + 2 * hk, dim, generator=g) * 2).to(dtype)
    return packed, g


def _positions(n, axes, g, extent=1600, dtype=torch.int32):
    return torch.randint(0, extent, (n, axes), generator=g).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,hq,hk,dim,axes", [
    (0, 2, 2, 16, 3), (1, 1, 1, 2, 1), (1, 16, 4, 64, 3), (3, 2, 1, 6, 4), (5, 3, 3, 16, 3),
    (63, 6, 6, 32, 3), (64, 4, 4, 64, 1), (65, 5, 5, 40, 2), (130, 2, 2, 96, 3), (77, 8, 2, 128, 3),
    (33, 3, 1, 250, 4), (40, 1, 1, 256, 3), (1000, 4, 4, 48, 3), (21, 7, 7, 72, 3), (9, 3, 0, 64, 3),
    (300, 12, 12, 64, 3)])
def test_sizes(n, hq, hk, dim, axes, dtype):
    say("norm_rotate_heads:", n, hq, hk, dim, axes, dtype)
    packed, g = _heads(n, hq, hk, dim, dtype)
    pos = _positions(n, axes, g)
    dev = packed.to(DEV)
    for interleaved in (False, True):
        for gain in (None, "dim", "head"):
            wq, wk = (None if gain is None else
                      (1 + 0.1 * torch.randn(*((dim,) if gain == "dim" else (h, dim)), generator=g))
                      .to(dtype) for h in (hq, hk))
            q, k = spconv.norm_rotate_heads(dev[:, :hq], dev[:, hq:hq + hk], pos.to(DEV),
                                            None if wq is None else wq.to(DEV),
                                            None if wk is None else wk.to(DEV),
                                            interleaved=interleaved)
            assert q.is_contiguous() and q.dtype == dtype
            check(q, *rotate64(packed[:, :hq], pos, wq, interleaved=interleaved), what="q")
            check(k, *rotate64(packed[:, hq:hq + hk], pos, wk, interleaved=interleaved), what="k")


@pytest.mark.parametrize("dtype", DTYPES)
def test_coordinates_far_from_the_origin(dtype):
    """Columns 1..3 of (b, z, y, x) rows, negative and large positions, f32
    ones with fractions, a base near one: the angle is reduced before it is
    rounded to f32."""
    packed, g = _heads(50, 2, 2, 64, dtype)
    rows = torch.randint(-2 ** 24, 2 ** 24, (50, 4), generator=g).to(torch.int32)
    q, _ = spconv.norm_rotate_heads(packed[:, :2].to(DEV), packed[:, 2:4].to(DEV),
                                    rows.to(DEV)[:, 1:], base=100.0)
    check(q, *rotate64(packed[:, :2], rows[:, 1:], base=100.0))
    pos = torch.rand(50, 2, generator=g) * 4000 - 2000
    q, _ = spconv.norm_rotate_heads(packed[:, :2].to(DEV), packed[:, 2:4].to(DEV), pos.to(DEV),
                                    base=1.5)
    check(q, *rotate64(packed[:, :2], pos, base=1.5))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """Heads and rows of odd strides, tensors aligned to their elements only:
    the same bits; NaN between the rows is not read."""
    n, h, dim = 70, 3, 64
    packed, g = _heads(n, h, h, dim, dtype)
    pos = _positions(n, 3, g).to(DEV)
    want = spconv.norm_rotate_heads(packed[:, :h].to(DEV).contiguous(),
                                    packed[:, h:2 * h].to(DEV).contiguous(), pos)
    for pad in (1, 4, 8):
        room = torch.full((n, 2 * h, dim + pad), float("nan"), dtype=dtype, device=DEV)
        room[..., pad:] = packed[:, :2 * h].to(DEV)
        got = spconv.norm_rotate_heads(room[:, :h, pad:], room[:, h:, pad:], pos)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), pad
    # heads outermost, and positions of a wider row
    heads = packed[:, :2 * h].to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(n, 7, dtype=torch.int32, device=DEV)
    wide[:, 2:5] = pos
    got = spconv.norm_rotate_heads(heads[:, :h], heads[:, h:], wide[:, 2:5])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_zero_and_non_finite_heads():
    """A head of zeros stays zero; NaN and infinities stay in their head."""
    packed, g = _heads(8, 2, 2, 32, torch.float16)
    packed[3, 0] = 0
    clean = packed.clone()
    packed[5, 1, 7], packed[6, 2, 0] = float("nan"), float("inf")
    pos = _positions(8, 3, g).to(DEV)
    a = spconv.norm_rotate_heads(clean[:, :2].to(DEV), clean[:, 2:4].to(DEV), pos)
    b = spconv.norm_rotate_heads(packed[:, :2].to(DEV), packed[:, 2:4].to(DEV), pos)
    a, b = torch.cat(a, 1).cpu(), torch.cat(b, 1).cpu()
    assert torch.equal(a[3, 0], torch.zeros(32, dtype=torch.float16))
    keep = torch.ones(8, 4, dtype=torch.bool)
    keep[5, 1] = keep[6, 2] = False
    assert torch.equal(a[keep], b[keep])
    assert torch.isnan(b[5, 1]).all() and torch.isnan(b[6, 2]).any()


def test_gain_of_another_type_and_a_side_stream():
    packed, g = _heads(500, 4, 2, 64, torch.bfloat16)
    pos = _positions(500, 3, g)
    w = 1 + 0.1 * torch.randn(4, 64, generator=g)
    args = (packed[:, :4].to(DEV), packed[:, 4:6].to(DEV), pos.to(DEV), w.to(DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q, k = spconv.norm_rotate_heads(*args)
    side.synchronize()
    check(q, *rotate64(packed[:, :4], pos, w))
    check(k, *rotate64(packed[:, 4:6], pos))


def test_refusals():
    packed, g = _heads(6, 2, 2, 16, torch.float16)
    q, k = packed[:, :2].to(DEV), packed[:, 2:4].to(DEV)
    pos = _positions(6, 3, g).to(DEV)
    f = spconv.norm_rotate_heads
    with pytest.raises(RuntimeError, match="GPU"):
        f(q.cpu(), k, pos)
    with pytest.raises(TypeError, match="unsupported dtype"):
        f(q.double(), k.double(), pos)
    with pytest.raises(ValueError, match="not \\(N, Hq, D\\)"):
        f(q, k[:5], pos)
    with pytest.raises(ValueError, match="k is"):
        f(q, k.float(), pos)
    with pytest.raises(ValueError, match="even number"):
        f(q[..., :15], k[..., :15], pos)
    with pytest.raises(ValueError, match="positions must be"):
        f(q, k, pos.long())
    with pytest.raises(ValueError, match="positions must be"):
        f(q, k, pos[:5])
    with pytest.raises(ValueError, match="axes"):
        f(q, k, torch.zeros(6, 5, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="q_weight must be"):
        f(q, k, pos, torch.ones(3, 16, device=DEV))
    with pytest.raises(ValueError, match="k_weight must be"):
        f(q, k, pos, torch.ones(16, device=DEV), torch.ones(16, device=DEV).half())
    with pytest.raises(ValueError, match="base"):
        f(q, k, pos, base=1.0)
    with pytest.raises(ValueError, match="eps"):
        f(q, k, pos, eps=-1.0)
