"""Frequencies of rotary positions against their formulas, and what the rotary operators refuse.  No GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

import ultraattn_amd as ua


def test_frequencies():
    f, s = ua.rope_freqs(8, base=100.0)
    assert f.dtype == torch.float64 and s == 1.0
    np.testing.assert_allclose(f.numpy(), [1.0, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15)
    np.testing.assert_allclose(ua.rope_freqs(8, base=100.0, scaling="linear", factor=4.0)[0].numpy(), f.numpy() / 4, rtol=1e-15)
    n, s = ua.rope_freqs(64, scaling="ntk", factor=8.0)
    plain = ua.rope_freqs(64)[0]
    assert s == 1.0 and n[0] == 1.0
    np.testing.assert_allclose(n[-1].item(), plain[-1].item() / 8, rtol=1e-12)         # the last pair is interpolated


def test_yarn_keeps_fast_pairs_and_interpolates_slow_ones():
    plain = ua.rope_freqs(128)[0]
    f, s = ua.rope_freqs(128, scaling="yarn", factor=16.0, original_length=4096)
    turns = 4096 * plain / (2 * math.pi)
    assert s == pytest.approx(0.1 * math.log(16) + 1)
    assert torch.equal(f[turns > 32], plain[turns > 32])
    torch.testing.assert_close(f[turns < 1], plain[turns < 1] / 16, rtol=1e-15, atol=0)
    between = (turns >= 1) & (turns <= 32)
    assert between.sum() > 4
    g = (turns[between] - 1) / 31
    torch.testing.assert_close(f[between], plain[between] * (g + (1 - g) / 16), rtol=1e-14, atol=0)
    assert (f[1:] <= f[:-1]).all()


@pytest.mark.parametrize("args", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, base=-1.0), dict(rotary_dim=8, factor=2.0),
                                  dict(rotary_dim=8, scaling="cubic"), dict(rotary_dim=2, scaling="ntk", factor=2.0),
                                  dict(rotary_dim=8, scaling="yarn", factor=2.0), dict(rotary_dim=8, scaling="linear", factor=0.0),
                                  dict(rotary_dim=8, scaling="yarn", factor=2.0, original_length=64, slow=4.0, fast=4.0)])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        ua.rope_freqs(**args)


def test_operators_refuse_host_tensors(lib):
    x, f = torch.zeros(1, 2, 3, 8), torch.ones(4, dtype=torch.float64)
    with pytest.raises(ValueError):
        ua.rope_fwd(x, x, f)
    with pytest.raises(TypeError):
        ua.rope_bwd(x.int(), None, f)
    with pytest.raises(TypeError):
        ua.rope_fwd([1.0], None, f)
    with pytest.raises(ValueError):
        ua.rope_append(x, x, x, x, x, torch.zeros(1, dtype=torch.int32), f)


def test_c_entry_refuses_before_any_launch(lib):
    buf = np.zeros(64, np.uint8).ctypes.data // 16 * 16 + 16     # never dereferenced
    s = (ctypes.c_int64 * 3)(64, 64, 64)

    def rope(q=buf, f=buf, batch=1, seq=1, heads=1, kv=1, dim=64, rotary=64, dtype=0, scale=1.0, st=s):
        return lib.ua_rope(q, buf, buf, buf, f, None, 0, 0, 0, 0, batch, seq, heads, kv, dim, rotary, dtype, 0, 0, scale, st, s, s, s, None)

    assert rope(q=None) == -1 and rope(f=None) == -1 and rope(st=None) == -1
    assert rope(batch=-1) == -2 and rope(dim=0) == -2 and rope(rotary=3) == -2 and rope(rotary=66) == -2 and rope(rotary=0) == -2
    assert rope(dim=1024) == -3 and rope(dtype=3) == -3 and rope(scale=0.0) == -3 and rope(scale=math.nan) == -3
    assert rope(batch=0, q=None) == 0 and rope(seq=0) == 0                     # nothing to do
    assert rope(batch=1 << 16, seq=1 << 16) == -2
    append = [buf] * 8 + [1, 1, 1, 1, 4, 64, 64, 0, 0, 1.0] + [s] * 6 + [None]
    for i in range(8):
        assert lib.ua_rope_append(*append[:i], None, *append[i + 1:]) == -1
    assert lib.ua_rope_append(*append[:12], -1, *append[13:]) == -2
