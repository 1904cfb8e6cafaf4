"""Softmax scales whose reciprocal, or whose scores, leave fp32's range: the backward would divide statistics by them.  No GPU."""
import math

import pytest

from tests.test_host_swa import BUF, S, fwd


@pytest.mark.parametrize("scale", [1e-45, 1e-39, 2.0 ** -65, 2.0 ** 65, 3e38, math.inf])
def test_refused(lib, scale):
    assert fwd(lib, scale=scale) == -3
    assert lib.ua_swa_bwd(*[BUF] * 9, 1, 4, 2, 16, 16, 64, 0, *[S] * 7, 0, 0, -1, 0, 0, scale, None, 0, None) == -3
    assert lib.ua_swa_bwd_delta(*[BUF] * 7, 1, 4, 2, 16, 16, 64, 0, *[S] * 5, 0, 0, -1, 0, 0, scale, None) == -3
    assert lib.ua_swa_decode(*[BUF] * 6, 2, 1, 4, 2, 64, 64, 0, *[S] * 4, -1, 0, scale, None, 0, None) == -3


@pytest.mark.parametrize("scale", [2.0 ** -64, 1.0, 2.0 ** 64])
def test_taken(lib, scale):
    assert fwd(lib, sq=0, scale=scale) == 0
