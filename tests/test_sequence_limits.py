"""Sizes at which the voxel-block operators' C entries refuse (nothing is launched)."""
from trispconv_amd import _lib as L


def test_attention_refuses_key_counts_that_its_tiles_would_pass():
    """Key numbers are 32-bit, and a walk looks up to a tile past the last key:
    the last of 2^31 - 1 keys would send it to negative ones."""
    lib = L.lib()

    def call(n_k, n_q=8):
        return lib.tsc_window_attention(16, 64, 16, 16, 0, 16, 16, 0, 16, 16, 16, 1, n_q, n_k, 4, 2,
                                        16, 100, 0, 0, 1.0, 1, None, 0, 16, None)

    for n_k in (2 ** 31 - 1, 2 ** 31 - 1024):
        assert call(n_k) == 1 and b"keys" in lib.tsc_last_error(), lib.tsc_last_error()
    assert call(2 ** 31 - 1025, n_q=0) == 0  # accepted (without queries nothing is launched)


def test_launches_of_too_many_threads_are_refused():
    """A launch of 2^32 threads wraps without an error and leaves rows unwritten."""
    lib = L.lib()
    # 2^25 samples of one token on four key heads: a wave each
    n = 2 ** 25
    rc = lib.tsc_window_attention(16, 64, 16, 16, 64, 16, 16, 64, 16, 16, 16, n, n, n, 4, 4, 16, -1, -1,
                                  0, 1.0, 1, None, 0, 16, None)
    assert rc == 1 and b"too many tiles" in lib.tsc_last_error(), (rc, lib.tsc_last_error())
    for dtype in (0, 1, 2):  # 2^24 tiles of 128 x 64
        rc = lib.tsc_linear_act(16, 8, 16, 8, None, 0, None, 0, dtype, 2 ** 31 - 1, 8, 64, 0, 16, None)
        assert rc == 1 and b"too many tiles" in lib.tsc_last_error(), (rc, lib.tsc_last_error())
