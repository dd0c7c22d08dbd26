"""CPU: the number of tiles that one attention call over the 8-bit cache takes.
No GPU work is issued: both calls are refused."""

import ctypes

import pytest

from metal_liger_b200 import _C

STRIDES = (ctypes.c_int64 * 3)(8, 8, 8)


@pytest.mark.parametrize("batch,heads", [(16385, 32766), (16384, 32768 - 1), (65535, 32767)])
def test_calls_whose_tile_numbers_would_pass_31_bits_are_refused(cuda_lib, batch, heads):
    """Four tiles (two of a cache of 64 positions, two that a segment counts more)
    for each sequence and head: 2^31 - 8, 2^31 - 2^16 and 2^33 of them.  A warp's
    last tile is its first plus its share, up to a few hundred past the total, so
    the total stays 2^17 below 2^31."""
    assert 4 * batch * heads >= 2 ** 31 - 2 ** 17
    c = _C.Kv8Cache(16, 16, 16, 16, 16, 16, 0, 1, batch, heads, 64, 64, 64)
    rc = cuda_lib.ml_kv8_attention(ctypes.byref(c), 16, STRIDES, heads, 1, 16, 0, None, 0, 1.0, 16,
                                   16, 1 << 40, None)
    assert rc == 1 and b"too many" in cuda_lib.ml_last_error()
