"""GELU of linear_act where x Phi(x) is far smaller than x."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu
from sequence_oracle import ROUNDING, SMALLEST

pytestmark = [pytest.mark.gpu, needs_gpu]

# relative: f32, a fit of 2.3e-8 and about a dozen roundings of 2^-24; 16-bit
# types, a fit of 1e-4 beside one rounding of 2^-11 or 2^-8
RELATIVE = {torch.float32: 8e-7, torch.float16: 1e-4, torch.bfloat16: 1e-4}


@pytest.mark.parametrize("dtype", list(RELATIVE))
@pytest.mark.parametrize("rows,columns", [(7, 2000), (40, 500), (30_000, 2), (300, 1024), (33_000, 64)])
def test_relative_error(rows, columns, dtype):
    """Values from -13 (where the result is -8e-38) to 13, on every kernel that ends
    in an activation: weights of one entry that are powers of two, so that the
    activation's argument is exact."""
    g = torch.Generator().manual_seed(rows)
    w = torch.tensor([2.0 ** -(j % 4) for j in range(columns)]).to(dtype)[:, None]
    x = ((torch.rand(rows, 1, generator=g) - 0.5) * 26).to(dtype)
    x[:4, 0] = torch.tensor([-4.0, -8.0, -12.9, -1.0])
    got = spconv.linear_act(x.to(DEV), w.to(DEV), activation="gelu").cpu().double()
    v = x.double() * w.double().t()
    ref = v * 0.5 * torch.erfc(v * -(0.5 ** 0.5))  # (torch's ndtr cancels below -8)
    tol = RELATIVE[dtype] + ROUNDING[dtype] * 1.001
    over = (got - ref).abs() / (tol * ref.abs() + SMALLEST[dtype])
    assert float(over.max()) <= 1.0, (float(over.max()), float(v.flatten()[over.argmax()]))


@pytest.mark.parametrize("dtype", list(RELATIVE))
@pytest.mark.parametrize("rows", [4, 30, 33_000])
def test_ends(rows, dtype):
    w = torch.ones(64, 1, dtype=dtype)
    inf = float("inf")
    x = torch.tensor([inf, -inf, float("nan"), -40.0] + [0.0] * (rows - 4)).to(dtype)[:, None]
    got = spconv.linear_act(x.to(DEV), w.to(DEV), activation="gelu").cpu()
    assert (got[0] == inf).all() and (got[1] == 0).all() and torch.isnan(got[2]).all()
    assert (got[3] == 0).all() and (got[4:] == 0).all()
