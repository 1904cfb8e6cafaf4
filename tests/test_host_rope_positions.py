"""Positions beyond 2^53, which 64-bit floats do not hold one by one, are refused where the host knows them.  No GPU."""
import ctypes

import numpy as np
import pytest

BUF = np.zeros(64, np.uint8).ctypes.data // 16 * 16 + 16          # never dereferenced
S = (ctypes.c_int64 * 3)(4096, 64, 64)


def rope(lib, start, seq=8, batch=1, positions=None):
    return lib.ua_rope(BUF, BUF, BUF, BUF, BUF, positions, 1, 0, 0, start, batch, seq, 1, 1, 64, 64, 0, 0, 0, 1.0, S, S, S, S, None)


@pytest.mark.parametrize("start", [2 ** 53, 2 ** 53 - 7, -(2 ** 53) - 1, 2 ** 62, -(2 ** 63)])
def test_refused(lib, start):
    assert rope(lib, start) == -2


def test_taken(lib):
    assert rope(lib, 2 ** 53 - 8, batch=0) == rope(lib, -(2 ** 53), batch=0) == rope(lib, 2 ** 62, batch=0, positions=BUF) == 0
