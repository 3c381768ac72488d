"""The workspace of cache_attention: asked for where a call is split, refused where
it is too small.  Nothing is launched."""
import pytest

from trispconv_amd import _lib as L

# (samples, rows, positions, prefix rows, query heads, key heads, head size, left, right, sinks)
SPLIT = [(1, 1, 30_000, 0, 4, 2, 64, -1, 0, 0), (4, 4, 2_000, 0, 4, 2, 64, -1, 0, 0),
         (2, 600, 30_000, 0, 4, 2, 128, -1, 0, 0), (8, 8, 2_100, 2_048, 4, 2, 64, -1, 0, 0),
         (64, 64, 9_000, 8_192, 4, 2, 64, 4_095, 0, 8), (2, 300, 9_000, 8_192, 4, 2, 64, -1, 0, 0)]
WHOLE = [(1, 1, 900, 0, 4, 2, 64, -1, 0, 0), (64, 64, 30_000, 0, 4, 2, 64, 500, 0, 0)]


def _bytes(case, dtype):
    return L.lib().tsc_cache_attention_workspace_bytes(*case, dtype)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("case", SPLIT)
def test_split_calls(case, dtype):
    """At least two parts of a sum, a reference and the values of every row and head."""
    samples, rows, positions, prefix, hq, hk, dim, left, right, sinks = case
    need = _bytes(case, dtype)
    assert need >= 2 * rows * hq * (dim + 2) * 4 and need % 4 == 0
    for ws, there in ((None, 0), (None, need), (16, 0), (16, need - 1)):
        rc = L.lib().tsc_cache_attention(16, hq * dim, dim, 16, 16 * hk * dim, hk * dim, dim, 16, 16 * hk * dim,
                                         hk * dim, dim, 8, 1, 16, positions, positions, 16, 16, samples,
                                         16 if prefix else None, prefix, rows, hq, hk, dim, left, right, sinks,
                                         1.0, dtype, ws, there, 16, None)
        assert rc == 1 and b"workspace of %d bytes" % need in L.lib().tsc_last_error()


@pytest.mark.parametrize("case", WHOLE)
def test_calls_that_are_not_split(case):
    assert _bytes(case, 1) == 0
