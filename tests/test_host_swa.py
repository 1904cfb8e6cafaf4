"""What the sliding-window operators refuse and need before any launch.  No GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

import ultraattn_amd as ua

BUF = np.zeros(64, np.uint8).ctypes.data // 16 * 16 + 16          # an aligned address that is never dereferenced
S = (ctypes.c_int64 * 3)(1 << 20, 1024, 64)
BAD = (ctypes.c_int64 * 3)(1 << 20, 1028, 64)
NONE = (ctypes.c_int64 * 3)(0, 0, 0)


def fwd(lib, q=BUF, k=BUF, lse=BUF, batch=1, heads=4, kv=2, sq=16, sk=16, dim=64, dtype=0, qs=S, ks=S, os=S, start=0, left=-1, right=0, sinks=0, scale=0.1):
    return lib.ua_swa_fwd(q, k, BUF, BUF, lse, batch, heads, kv, sq, sk, dim, dtype, qs, ks, S, os, start, 0, left, right, sinks, scale, None, 0, None)


def test_forward_refuses(lib):
    assert fwd(lib, q=None) == -1 and fwd(lib, k=None) == -1 and fwd(lib, lse=None) == -1 and fwd(lib, qs=None) == -1
    assert fwd(lib, heads=3) == -2 and fwd(lib, kv=0) == -2 and fwd(lib, batch=-1) == -2 and fwd(lib, sq=-1) == -2 and fwd(lib, sk=2 ** 29) == -2
    assert fwd(lib, left=-2) == -2 and fwd(lib, right=-2) == -2 and fwd(lib, sinks=-1) == -2 and fwd(lib, start=2 ** 61) == -2
    assert fwd(lib, batch=2 ** 20, heads=2 ** 11, sq=2 ** 20) == -2 and fwd(lib, batch=2 ** 20, heads=2 ** 12, kv=1, sq=0) == -2
    assert fwd(lib, dim=96) == -3 and fwd(lib, dtype=2) == -3 and fwd(lib, scale=0.0) == -3 and fwd(lib, scale=math.nan) == -3
    assert fwd(lib, q=BUF + 2) == -4 and fwd(lib, qs=BAD) == -4 and fwd(lib, os=NONE) == -4
    assert fwd(lib, batch=0, q=None) == 0 and fwd(lib, sq=0) == 0                    # nothing to do
    huge = (ctypes.c_int64 * 3)(0, 1 << 23, 64)
    assert fwd(lib, ks=huge) == -2


def test_backward_refuses(lib):
    ok = [BUF] * 9 + [1, 4, 2, 16, 16, 64, 0] + [S] * 7 + [0, 0, -1, 0, 0, 0.1, None, 0, None]
    for i in list(range(9)) + list(range(16, 23)):
        assert lib.ua_swa_bwd(*ok[:i], None, *ok[i + 1:]) == -1
    for i, x, rc in ((14, 32, -3), (15, 2, -3), (28, -0.1, -3), (10, 5, -2), (12, -1, -2), (0, BUF + 4, -4), (16, BAD, -4), (20, NONE, -4)):
        assert lib.ua_swa_bwd(*ok[:i], x, *ok[i + 1:]) == rc, i
    assert lib.ua_swa_bwd(*ok[:9], 0, *ok[10:]) == 0
    delta = [BUF] * 7 + [1, 4, 2, 16, 16, 64, 0] + [S] * 5 + [0, 0, -1, 0, 0, 0.1, None]
    for i in list(range(7)) + list(range(14, 19)):
        assert lib.ua_swa_bwd_delta(*delta[:i], None, *delta[i + 1:]) == -1
    assert lib.ua_swa_bwd_delta(*delta[:12], 80, *delta[13:]) == -3 and lib.ua_swa_bwd_delta(*delta[:10], 0, *delta[11:]) == 0
    assert lib.ua_swa_bwd_delta(*delta[:2], BUF + 2, *delta[3:]) == -4


def test_decode_refuses(lib):
    ok = [BUF] * 6 + [2, 1, 4, 2, 64, 64, 0] + [S] * 4 + [-1, 0, 0.1, None, 0, None]
    for i in list(range(6)) + list(range(13, 17)):
        assert lib.ua_swa_decode(*ok[:i], None, *ok[i + 1:]) == -1
    for i, x, rc in ((6, -1, -2), (9, 3, -2), (10, -1, -2), (10, 2 ** 29, -2), (11, 96, -3), (12, 2, -3), (17, -2, -2), (18, -1, -2), (19, 0.0, -3), (5, BUF + 2, -4),
                     (13, BAD, -4), (16, NONE, -4)):
        assert lib.ua_swa_decode(*ok[:i], x, *ok[i + 1:]) == rc, i
    assert lib.ua_swa_decode(*ok[:6], 0, *ok[7:]) == 0 and lib.ua_swa_decode(*ok[:7], 0, *ok[8:]) == 0


def test_workspaces(lib):
    """Large launches need none; nothing overflows at the largest arguments; what is refused needs nothing."""
    assert lib.ua_swa_workspace_bytes(1, 64, 8, 8192, 8192, 128, 0, 0, -1, 0, 0) == 0
    few = lib.ua_swa_workspace_bytes(1, 2, 1, 100, 8192, 128, 8092, 0, -1, 0, 0)
    assert few > 2 * 100 * 129 * 4 and few % 256 == 0
    assert lib.ua_swa_workspace_bytes(1, 2, 1, 100, 8192, 96, 0, 0, -1, 0, 0) == 0
    for f in (lib.ua_swa_workspace_bytes, lib.ua_swa_bwd_workspace_bytes):
        assert 0 <= f(1, 1, 1, 2 ** 28, 2 ** 28, 128, 2 ** 60, -2 ** 60, 2 ** 60, 2 ** 60, 2 ** 60) < 2 ** 44
        assert f(0, 1, 1, 5, 5, 64, 0, 0, -1, 0, 0) == 0 and f(1, 1, 1, 0, 5, 64, 0, 0, -1, 0, 0) == 0
    assert 0 <= lib.ua_swa_decode_workspace_bytes(1, 1, 1, 1, 2 ** 28, 128, 2 ** 62, 2 ** 62) < 2 ** 30
    assert lib.ua_swa_decode_workspace_bytes(4096, 1, 8, 8, 4096, 128, -1, 0) == 0


def test_operators_refuse_host_tensors(lib):
    x = torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16)
    lse = torch.zeros(1, 2, 16)
    for call in (lambda: ua.swa_fwd(x, x, x), lambda: ua.swa_bwd(x, x, x, x, x, lse), lambda: ua.swa_decode(x, x, x, torch.ones(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ua.swa_fwd(x.float(), x.float(), x.float())
    with pytest.raises((TypeError, ValueError)):
        ua.swa_fwd(x, x, x, window=(1, 2, 3))
