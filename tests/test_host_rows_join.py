"""What the C entries that join rows refuse before they touch the device."""
import ctypes

import numpy as np


def test_refusals(lib):
    s, ls = (ctypes.c_int64 * 3)(64 * 64, 64, 64), (ctypes.c_int64 * 3)(16, 1, 16)
    odd = (ctypes.c_int64 * 3)(64 * 64, 60, 64)
    buf = np.zeros(64, np.uint8).ctypes.data // 16 * 16 + 16          # never dereferenced
    arr, two = (ctypes.c_void_p * 2)(buf, buf), (ctypes.c_void_p * 2)(buf, None)
    merge = lambda o=arr, l=arr, n=2, out=buf, lse=buf, shape=(1, 16, 1, 64), dt=1: lib.ua_rows_merge(o, l, n, out, lse, *shape, dt, None)  # noqa: E731
    assert merge(n=0) == merge(n=17) == merge(shape=(1, 16, 1, 96)) == merge(dt=2) == merge(dt=-1) == -3
    assert merge(o=None) == merge(l=None) == merge(out=None) == merge(lse=None) == merge(o=two) == merge(l=two) == -1
    assert merge(shape=(-1, 16, 1, 64)) == merge(shape=(1, 16, 0, 64)) == merge(shape=(2 ** 15, 2 ** 15, 1, 64)) == merge(shape=(1, 2 ** 20, 2 ** 9, 64)) == -2
    assert merge(out=buf + 8) == -4
    assert merge(shape=(0, 16, 1, 64)) == merge(shape=(1, 0, 1, 64)) == 0
    ok = (buf, buf, buf + 64, buf, buf + 128, buf)
    update = lambda p=ok, shape=(1, 16, 1, 64), f=(0, 0, 0), st=(s, ls, s, ls, s, ls): lib.ua_rows_update(*p, *shape, 1, *f, *st, None)  # noqa: E731
    assert update(shape=(1, 16, 1, 32)) == -3 and update(p=(None, *ok[1:])) == update(st=(s, ls, s, ls, s, None)) == -1
    assert update(st=(odd, ls, s, ls, s, ls)) == update(st=(s, ls, odd, ls, s, ls)) == update(st=(s, ls, s, ls, odd, ls)) == -4
    assert update(p=(buf, buf, buf + 64, buf, buf, buf), f=(0, 0, 1)) == -2                                # in place of rows of another type
    assert update(p=(buf, buf, buf + 64, buf, buf, buf), st=(s, ls, s, ls, (ctypes.c_int64 * 3)(64 * 128, 128, 64), ls)) == -2
    assert update(st=(s, ls, s, ls, s, (ctypes.c_int64 * 3)(16, 16, 1))) == -2
    total = lambda parts=arr, n=2, out=buf, st=s, dim=64: lib.ua_rows_sum(parts, n, 0, out, 1, 16, 1, dim, 0, st, 1.0, None)  # noqa: E731
    assert total(n=17) == total(dim=80) == -3 and total(parts=None) == total(st=None) == total(parts=two) == -1 and total(st=odd) == total(out=buf + 2) == -4
    delta = lambda o=buf, d=buf, st=s, dim=64: lib.ua_rows_delta(o, d, buf, 1, 16, 1, dim, 0, st, s, None)  # noqa: E731
    assert delta(o=None) == -1 and delta(dim=256) == -3 and delta(st=odd) == delta(d=buf + 8) == -4
