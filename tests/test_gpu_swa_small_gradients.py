"""fp16 holds values below 6e-5 with fewer bits and none below 3e-8: dS of small gradients, or of long rows, lies there."""
import math

import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, Reference, inputs, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -8, 2.0 ** -12])
@pytest.mark.parametrize("seq_q,seq_k,window,sinks", [(700, 700, (-1, 0), 0), (200, 3500, (-1, -1), 0), (900, 900, (300, 0), 3)])
def test_small_gradients_keep_their_bits(dim, size, seq_q, seq_k, window, sinks):
    """dO of `size` gives dQ and dK of that size, as far as fp16 holds those: the error over all of dQ and dK, in the mean of squares, is at
    most that of three roundings.  (A rounding of half a step u at most is u / sqrt(3) in that mean at most.  Their own is one; dQ and dK are sums of
    dS K, which independent roundings of dS move by u / sqrt(3) of themselves, and those of O, in delta, by no more.  Below 2^-14 their own is 2^-25 / sqrt(3).)"""
    q, k, v, do = inputs(1, seq_q, seq_k, 2, 1, dim, torch.float16)
    do = do.clamp(-8, 8)
    small = (do * size).half()
    how = dict(window=window, sinks=sinks)
    out, lse = ua.swa_fwd(q, k, v, **how)
    got = ua.swa_bwd(small, q, k, v, out, lse, **how)
    ref = Reference(q, k, v, visible(seq_q, seq_k, window, sinks), dout=small)
    u = torch.finfo(torch.float16).eps / 2
    for name, x in zip(("dq", "dk", "dv"), got):
        want = getattr(ref, name)
        err, whole = (x.double() - want).square().mean().sqrt().item(), want.square().mean().sqrt().item()
        room = 3 * u / math.sqrt(3) * whole + 2.0 ** -25 / math.sqrt(3)
        assert err <= room, (name, err / whole, room / whole)


@pytest.mark.parametrize("dim", [64, 128])
def test_large_gradients_are_not_infinite(dim):
    """dS up to the type's largest value, beside rows whose dS is small; and rows of one size in the first blocks of a walk, of another later."""
    q, k, v, do = inputs(1, 600, 600, 2, 1, dim, torch.float16, std=0.5)
    for first in (True, False):
        grow = torch.logspace(-5, 3, 600, device=DEV)
        d = (do.float().clamp(-3, 3) * (grow if first else grow.flip(0))[None, :, None, None]).half()
        out, lse = ua.swa_fwd(q, k, v, (100, 0), 4)
        dq, dk, dv = ua.swa_bwd(d, q, k, v, out, lse, (100, 0), 4)
        Reference(q, k, v, visible(600, 600, (100, 0), 4), dout=d).check(dq=dq, dk=dk, dv=dv)
