"""window_attention's refusal of heads without values."""
import pytest
import torch

import trispconv.pytorch as spconv
from gpu_util import DEV, needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]


def test_heads_of_no_values_are_refused():
    off = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    for heads, dim, words in ((2, 0, "head size"), (0, 16, "evenly"), (0, 0, "evenly")):
        x = torch.zeros(4, heads, dim, device=DEV, dtype=torch.float16)
        with pytest.raises(ValueError, match=words):
            spconv.window_attention(x, x, x, off)
