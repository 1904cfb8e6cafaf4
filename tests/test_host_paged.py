"""What the paged cache's operators refuse and need before any launch.  No GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

import ultraattn_amd as ua

BUF = np.zeros(64, np.uint8).ctypes.data // 16 * 16 + 16          # an aligned address that is never dereferenced
S = (ctypes.c_int64 * 3)(1 << 20, 1024, 64)
L = (ctypes.c_int64 * 4)(1 << 24, 1 << 20, 1024, 64)
BAD = (ctypes.c_int64 * 3)(1 << 20, 1028, 64)
NONE = (ctypes.c_int64 * 3)(0, 0, 0)


def refused(f, ok, changes):
    for i, x, rc in changes:
        assert f(*ok[:i], x, *ok[i + 1:]) == rc, (i, x)


def test_decode_refuses(lib):
    # q k v o lse table lens n_new parents | batch tokens heads kv pages page most dim dtype | strides | 4 x strides | left sinks scale ws bytes stream
    ok = [BUF] * 9 + [2, 3, 4, 2, 9, 16, 5, 64, 0] + [5, 3] + [S] * 4 + [-1, 0, 0.1, None, 0, None]
    f = lib.ua_paged_decode
    refused(f, ok, [(i, None, -1) for i in (0, 1, 2, 3, 4, 5, 6, 20, 21, 22, 23)])
    refused(f, ok, [(9, -1, -2), (10, -1, -2), (10, 257, -2), (11, 3, -2), (11, 0, -2), (12, 0, -2), (13, -1, -2), (14, 0, -2), (14, 2 ** 30, -2), (15, -1, -2), (18, -1, -2),
                    (19, -1, -2), (24, -2, -2), (25, -1, -2), (9, 2 ** 28, -2)])
    refused(f, ok, [(16, 96, -3), (17, 2, -3), (26, 0.0, -3), (26, math.nan, -3), (26, 2.0 ** 70, -3)])
    refused(f, ok, [(i, BUF + 2, -4) for i in range(9) if i != 4] + [(20, BAD, -4), (21, BAD, -4), (22, BAD, -4), (23, NONE, -4)])
    assert f(*ok[:9], 0, *ok[10:]) == 0 and f(*ok[:10], 0, *ok[11:]) == 0                # nothing to do


def test_append_refuses(lib):
    # q k v q_out k_pages v_pages freqs table lens n_new parents | batch tokens heads kv pages page most dim rotary dtype interleaved scale | strides | 6 x strides
    ok = [BUF] * 11 + [2, 3, 4, 2, 9, 16, 5, 64, 32, 0, 0, 1.0] + [5, 3] + [S] * 6 + [None]
    f = lib.ua_paged_append
    refused(f, ok, [(i, None, -1) for i in (*range(9), *range(25, 31))])
    refused(f, ok, [(11, -1, -2), (12, -1, -2), (12, 257, -2), (13, -1, -2), (14, 0, -2), (15, -1, -2), (16, 0, -2), (17, -1, -2), (18, 0, -2), (19, 31, -2), (19, 66, -2), (23, -1, -2),
                    (24, -1, -2)])
    refused(f, ok, [(18, 1024, -3), (20, 3, -3), (22, 0.0, -3), (22, math.nan, -3)])
    refused(f, ok, [(i, BUF + 2, -4) for i in (7, 8, 9, 10)])
    assert f(*ok[:11], 0, *ok[12:]) == 0 and f(*ok[:12], 0, *ok[13:]) == 0


def test_keep_refuses(lib):
    # k v table lens n_new path n_kept | layers batch tokens n_path kv pages page most dim dtype | strides | 2 x strides
    ok = [BUF] * 7 + [3, 2, 9, 4, 2, 9, 16, 5, 64, 0] + [5, 4] + [L] * 2 + [None]
    f = lib.ua_paged_keep
    refused(f, ok, [(i, None, -1) for i in (0, 1, 2, 3, 5, 6, 19, 20)])
    refused(f, ok, [(7, -1, -2), (7, 65536, -2), (8, 65536, -2), (8, -1, -2), (9, -1, -2), (10, -1, -2), (11, 0, -2), (12, -1, -2), (13, 0, -2), (14, -1, -2), (15, 0, -2), (17, -1, -2),
                    (18, -1, -2), (15, 2 ** 30, -2)])
    refused(f, ok, [(16, 3, -3), (16, -1, -3)])
    refused(f, ok, [(i, BUF + 1, -4) for i in range(7)])
    for i in (7, 8, 9, 10, 12, 14):
        assert f(*ok[:i], 0, *ok[i + 1:]) == 0


def test_workspaces(lib):
    f = lib.ua_paged_decode_workspace_bytes
    few = f(1, 1, 32, 8, 16, 512, 128, -1, 0)
    assert few > 0 and few % 256 == 0 and few % (32 * 128 * 4 + 256) == 0
    assert f(4096, 1, 8, 8, 16, 256, 128, -1, 0) == 0 and f(1, 1, 32, 8, 16, 1, 128, -1, 0) == 0            # fills the device; one block
    assert f(1, 1, 32, 8, 16, 512, 96, -1, 0) == 0 and f(1, 1, 32, 5, 16, 512, 128, -1, 0) == 0 and f(0, 1, 1, 1, 1, 1, 64, -1, 0) == f(1, 0, 1, 1, 1, 1, 64, -1, 0) == 0
    assert f(1, 40, 32, 8, 16, 4096, 128, -1, 0) > 0
    assert 0 <= f(1, 1, 1, 1, 2 ** 29, 2 ** 31 - 1, 128, 2 ** 62, 2 ** 62) < 2 ** 30
    assert 0 <= f(2 ** 20, 16, 1, 1, 1, 2 ** 31 - 1, 128, 2 ** 62, 2 ** 62) < 2 ** 44


def test_operators_refuse_host_tensors(lib):
    x, pool = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    one, table, f = torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32), torch.ones(32, dtype=torch.float64)
    for call in (lambda: ua.paged_append(x, x, x, pool, pool, table, one, f), lambda: ua.paged_decode(x, pool, pool, table, one),
                 lambda: ua.paged_keep(pool, pool, table, one, 3, table, one)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ua.paged_decode(x.float(), pool.float(), pool.float(), table, one)
    with pytest.raises(TypeError):
        ua.paged_keep(pool.int(), pool.int(), table, one, 3, table, one)
