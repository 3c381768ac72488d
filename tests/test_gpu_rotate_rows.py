"""norm_rotate_heads on more rows than one grid of waves has."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import check, rotate64

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("dim", [2, 8])
def test_more_than_2_to_26_rows(dim):
    """A wave a row is 64 threads a row, and a launch holds fewer than 2^32."""
    n = 2 ** 26 + 7
    say("norm_rotate_heads rows:", n, dim)
    g = torch.Generator(DEV).manual_seed(1)
    q = torch.randn(n, 1, dim, generator=g, device=DEV, dtype=torch.float16)
    pos = torch.randint(0, 1000, (n, 1), generator=g, device=DEV, dtype=torch.int32)
    got, none = spconv.norm_rotate_heads(q, q[:, :0], pos)
    assert none.shape == (n, 0, dim)
    for part in (slice(0, 50), slice(n // 2, n // 2 + 50), slice(n - 50, n)):
        check(got[part], *rotate64(q[part].cpu(), pos[part].cpu()))
