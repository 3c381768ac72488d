"""linear_act against its 64-bit form."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import check, linear64

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def _tensors(n, c_in, c_out, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + n + 7 * c_in + 31 * c_out)
    x = torch.randn(n, c_in, generator=g).to(dtype)
    w = (torch.randn(c_out, c_in, generator=g) * max(c_in, 1) ** -0.5).to(dtype)
    b = (torch.randn(c_out, generator=g) * 0.1).to(dtype)
    r = torch.randn(n, c_out, generator=g).to(dtype)
    return x, w, b, r


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c_in,c_out", [
    (0, 8, 8), (1, 1, 1), (1, 512, 2048), (2, 17, 3), (3, 75, 50), (15, 0, 5), (16, 64, 64),
    (17, 2048, 96), (31, 40, 130), (64, 96, 384), (65, 130, 257), (127, 192, 768), (128, 768, 192),
    (129, 72, 136), (300, 33, 17), (257, 1024, 20), (1000, 64, 1000), (2500, 100, 100),
    (4099, 128, 256)])
def test_sizes(n, c_in, c_out, dtype):
    say("linear_act:", n, c_in, c_out, dtype)
    x, w, b, r = _tensors(n, c_in, c_out, dtype)
    xd, wd, bd, rd = (t.to(DEV) for t in (x, w, b, r))
    for bias, act, res in ((None, None, None), (b, "gelu", None), (b, None, r), (None, "silu", r)):
        got = spconv.linear_act(xd, wd, None if bias is None else bd, act,
                                None if res is None else rd)
        assert got.dtype == dtype and got.is_contiguous()
        check(got, *linear64(x, w, bias, act, res), what=f"{n} {c_in} {c_out} {act}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(act, dtype):
    """Arguments from -40 to 40, zero and both infinities, through a 1x1 weight
    of one, so that nothing but the activation is computed."""
    x = torch.cat([torch.linspace(-40, 40, 4001), torch.linspace(-6, 6, 1001),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 300.0, -300.0])]).to(dtype)[:, None]
    w = torch.ones(1, 1, dtype=dtype)
    check(spconv.linear_act(x.to(DEV), w.to(DEV), activation=act), *linear64(x, w, act=act),
          what=str(act))
    inf = float("inf")
    x = torch.tensor([[inf], [-inf], [float("nan")]], dtype=dtype)
    got = spconv.linear_act(x.to(DEV), w.to(DEV), activation=act).cpu().flatten().tolist()
    assert got[0] == inf and got[2] != got[2]
    assert got[1] == (-inf if act is None else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c_in,c_out", [(64, 128), (75, 33), (192, 200)])
def test_strides_and_alignment(c_in, c_out, dtype):
    """Rows inside wider ones, and tensors aligned to their elements only,
    give the bits of contiguous ones; what lies between the rows is NaN."""
    n = 333
    x, w, b, r = _tensors(n, c_in, c_out, dtype)
    want = spconv.linear_act(x.to(DEV), w.to(DEV), b.to(DEV), "silu", r.to(DEV))

    def inside(t, before, after):
        room = torch.full((t.shape[0], t.shape[1] + before + after), float("nan"), dtype=dtype,
                          device=DEV)
        room[:, before:before + t.shape[1]] = t.to(DEV)
        return room[:, before:before + t.shape[1]]

    for before, after in ((1, 0), (8, 8), (3, 5)):
        got = spconv.linear_act(inside(x, before, after), inside(w, before, after), b.to(DEV),
                                "silu", inside(r, before, after))
        assert torch.equal(got, want), (before, after)
    shared = torch.empty(1 + n * c_in, dtype=dtype, device=DEV)[1:].view(n, c_in)
    shared.copy_(x)
    assert torch.equal(spconv.linear_act(shared, w.to(DEV), b.to(DEV), "silu", r.to(DEV)), want)
    # a transposed view and a broadcast residual
    got = spconv.linear_act(x.to(DEV).t().contiguous().t(), w.to(DEV), b.to(DEV), "silu",
                            r[:1].to(DEV).expand(n, c_out))
    check(got, *linear64(x, w, b, "silu", r[:1].expand(n, c_out)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_rows_stay_apart(dtype):
    """An infinite or NaN row of x, or of w, reaches its own row or column only."""
    n, c_in, c_out = 200, 72, 140
    x, w, b, _ = _tensors(n, c_in, c_out, dtype)
    clean = spconv.linear_act(x.to(DEV), w.to(DEV), b.to(DEV)).cpu()
    x[7, 3], x[130, 71], w[139, 0] = float("nan"), float("inf"), float("nan")
    got = spconv.linear_act(x.to(DEV), w.to(DEV), b.to(DEV)).cpu()
    keep = torch.ones(n, c_out, dtype=torch.bool)
    keep[7], keep[130], keep[:, 139] = False, False, False
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(got[7]).all() and torch.isnan(got[:, 139]).all()
    assert not torch.isfinite(got[130]).any()


@pytest.mark.parametrize("bias_dtype", DTYPES)
def test_bias_of_another_type(bias_dtype):
    x, w, b, _ = _tensors(70, 48, 90, torch.float16)
    b = b.to(bias_dtype)
    check(spconv.linear_act(x.to(DEV), w.to(DEV), b.to(DEV)), *linear64(x, w, b))


def test_rows_do_not_depend_on_the_others():
    """Any number of rows: the same bits for a row whose kernel is the same,
    and every call the same bits."""
    x, w, b, _ = (t.to(DEV) for t in _tensors(5000, 96, 160, torch.bfloat16))
    a = spconv.linear_act(x, w, b, "gelu")
    assert torch.equal(a, spconv.linear_act(x, w, b, "gelu"))
    assert torch.equal(a[:4500], spconv.linear_act(x[:4500], w, b, "gelu"))


def test_on_another_stream():
    x, w, b, r = (t.to(DEV) for t in _tensors(3000, 128, 256, torch.float16))
    want = spconv.linear_act(x, w, b, "gelu", r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = spconv.linear_act(x, w, b, "gelu", r)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    x, w, b, r = (t.to(DEV) for t in _tensors(10, 8, 6, torch.float16))
    with pytest.raises(RuntimeError, match="GPU"):
        spconv.linear_act(x.cpu(), w, b)
    with pytest.raises(TypeError, match="unsupported dtype"):
        spconv.linear_act(x.double(), w.double())
    with pytest.raises(ValueError, match="weight is"):
        spconv.linear_act(x, w.float())
    with pytest.raises(ValueError, match="weight is"):
        spconv.linear_act(x, w.cpu())
    with pytest.raises(ValueError, match="not \\(N, C_in\\)"):
        spconv.linear_act(x, w[:, :7])
    with pytest.raises(ValueError, match="not \\(N, C_in\\)"):
        spconv.linear_act(x[None], w)
    with pytest.raises(ValueError, match="bias must have"):
        spconv.linear_act(x, w, b[:5])
    with pytest.raises(TypeError, match="unsupported dtype"):
        spconv.linear_act(x, w, b.double())
    with pytest.raises(ValueError, match="activation"):
        spconv.linear_act(x, w, b, "swish")
    with pytest.raises(ValueError, match="residual"):
        spconv.linear_act(x, w, b, None, r[:9])
    with pytest.raises(ValueError, match="residual is"):
        spconv.linear_act(x, w, b, None, r.float())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c_in,c_out", [(16_400, 40, 256), (33_000, 33, 64), (16_500, 72, 190),
                                          (1000, 100, 900), (12_900, 520, 1100),
                                          (12_850, 513, 1031)])
def test_every_tile_size(n, c_in, c_out, dtype):
    """Calls large enough for the larger tiles, whole and ragged, aligned and not."""
    say("linear_act tiles:", n, c_in, c_out, dtype)
    x, w, b, r = _tensors(n, c_in, c_out, dtype)
    got = spconv.linear_act(x.to(DEV), w.to(DEV), b.to(DEV), "gelu", r.to(DEV))
    check(got, *linear64(x, w, b, "gelu", r), what=f"{n} {c_in} {c_out}")


@pytest.mark.parametrize("n,c_out", [(140, 130), (1000, 900)])
def test_f32_values_that_three_parts_do_not_carry(n, c_out):
    """f32 products run as three bf16 parts of each value: rows of the smallest
    and the largest values, zeros, and infinities against weights whose lower
    parts are zero must come out as from f32 sums."""
    c_in = 96
    x, w, b, _ = _tensors(n, c_in, c_out, torch.float32)
    w = w.bfloat16().float()
    x[3] *= 1e-33
    x[40] *= 2.0 ** -100
    x[70] = 0
    x[100] *= 1e35
    w[5] *= 1e-30
    check(spconv.linear_act(x.to(DEV), w.to(DEV)), *linear64(x, w))
    x[9], x[130, 7] = float("inf"), float("inf")
    got = spconv.linear_act(x.to(DEV), w.to(DEV)).cpu()
    want, _ = linear64(x, w)
    rows = [9, 130]
    assert torch.equal(torch.isnan(got[rows]), torch.isnan(want[rows]))
    fine = ~torch.isnan(want[rows])
    assert torch.equal(got[rows][fine], want[rows][fine].float())


def test_one_wide_row_stride():
    """Rows further apart than a tile's 32-bit offsets reach are copied first."""
    x, w, b, _ = _tensors(20, 64, 96, torch.float16)
    room = torch.zeros(20, 1 << 21, dtype=torch.float16, device=DEV)
    room[:, :64] = x.to(DEV)
    check(spconv.linear_act(room[:, :64], w.to(DEV), b.to(DEV)), *linear64(x, w, b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,c_in,c_out", [(10_700, 520, 1100), (10_500, 513, 1031), (10_497, 576, 1152)])
def test_tiles_of_192_columns(n, c_in, c_out, dtype):
    """Calls that 192 columns a tile cut with less left empty than 256."""
    say("linear_act tiles of 192:", n, c_in, c_out, dtype)
    x, w, b, r = _tensors(n, c_in, c_out, dtype)
    for bias, act, res in ((None, None, r), (b, "gelu", None)):
        got = spconv.linear_act(x.to(DEV), w.to(DEV), None if bias is None else bias.to(DEV), act,
                                None if res is None else res.to(DEV))
        check(got, *linear64(x, w, bias, act, res), what=f"{n} {c_in} {c_out} {act}")
