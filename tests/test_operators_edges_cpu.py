"""CPU: the ends of what the dense-layer operators accept - launch sizes, row counts, settings - and what they refuse there."""
import ctypes

import pytest
import torch

from point2cyl_amd import _lib, ops, optim

ONE = ctypes.c_void_p(16)              # a non-null, 16-byte aligned dummy: arguments are checked before anything is dereferenced


def test_quantize_launches_fit_a_grid():
    """A launch holds fewer than 2^32 threads; a workgroup of 256 takes four rows of up to 1024 elements or one longer row."""
    L = _lib.lib()
    assert L.p2c_quantize_rows_at_once(0) == 0
    for K in (1, 64, 1000, 1024, 1025, 2048, 5000, 131072):
        rows = L.p2c_quantize_rows_at_once(K)
        assert rows >= 1 << 20 and (rows + 3) // 4 * 256 < 1 << 32
        if K > 1024:
            assert rows * 256 < 1 << 32
    top = (1 << 30) - 64               # ... and a tile of 64 rows is a workgroup of 256 in the requantising product
    assert -(-top // 64) * 256 < 1 << 32
    for M in (top + 1, (1 << 31) - 1):
        assert L.p2c_quantize_rows(ONE, 0, 8, M, 8, 64, ONE, ONE, None) == -1
        assert L.p2c_int8_linear_requant(ONE, 64, ONE, ONE, ONE, None, None, 0, 0, 1.0, 20.0, ONE, 64, ONE, M, 8, 8, 64, None) == -1
