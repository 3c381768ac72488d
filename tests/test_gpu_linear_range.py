"""linear_act on f32 operands that three bf16 values do not hold."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import check, linear64

pytestmark = [pytest.mark.gpu, needs_gpu]

# one call for each f32 kernel and tile: few rows, 32 x 32, 64 x 64, 128 x 64, 128 x 128
CALLS = [(5, 96, 40), (40, 96, 130), (1000, 96, 900), (33_000, 40, 64), (16_500, 72, 250),
         (1000, 75, 901)]


def _operands(n, c_in, c_out, seed=0):
    g = torch.Generator().manual_seed(seed + n + c_out)
    return torch.randn(n, c_in, generator=g), torch.randn(c_out, c_in, generator=g)


@pytest.mark.parametrize("n,c_in,c_out", CALLS)
@pytest.mark.parametrize("small,large", [(1e-36, 1e17), (1e-37, 1e19), (3e-38, 1e24),
                                         (1e-40, 1e29), (1e-42, 1e30)])
def test_small_against_large(n, c_in, c_out, small, large):
    """Every value of one operand below 2^-110, on either side: products are
    ordinary numbers and their sums as accurate as f32 sums."""
    say("linear_act range:", n, c_in, c_out, small, large)
    x, w = _operands(n, c_in, c_out)
    for a, b in ((x * small, w * large), (x * large, w * small)):
        check(spconv.linear_act(a.to(DEV), b.to(DEV)), *linear64(a, b), what=f"{small} {large}")


@pytest.mark.parametrize("n,c_in,c_out", CALLS)
def test_small_rows_among_others(n, c_in, c_out):
    """Some rows and columns with small values, alone or among larger ones in
    the row; the others keep the bits that they have without them."""
    x, w = _operands(n, c_in, c_out, 1)
    w[1::2] *= 2.0 ** 90
    clean = spconv.linear_act(x.to(DEV), w.to(DEV)).cpu()
    rows = torch.arange(0, n, 7)
    x[rows] *= 2.0 ** -125
    x[3, :5] = torch.tensor([2.0 ** -149, -2.0 ** -130, 2.0 ** -126, 0.0, 2.0 ** -111])
    cols = torch.arange(0, c_out, 11)
    w[cols] *= 2.0 ** -133
    got = spconv.linear_act(x.to(DEV), w.to(DEV)).cpu()
    check(got, *linear64(x, w))
    keep = torch.ones(n, c_out, dtype=torch.bool)
    keep[rows], keep[3], keep[:, cols] = False, False, False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("n,c_in,c_out", CALLS)
def test_one_product_that_vanishes_in_parts(n, c_in, c_out):
    """1e-41 against 1e38, all else zero: 1e-3, not 0."""
    x, w = torch.zeros(n, c_in), torch.zeros(c_out, c_in)
    x[n - 1, c_in - 1], w[c_out - 2, c_in - 1] = 1e-41, 1e38
    x[0, 3], w[2, 3] = -1e38, 1e-41
    check(spconv.linear_act(x.to(DEV), w.to(DEV)), *linear64(x, w))
