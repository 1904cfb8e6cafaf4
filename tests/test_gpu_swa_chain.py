"""A training step's run: rope_fwd -> swa_fwd -> swa_bwd -> rope_bwd, against autograd of the definition in float64.

Stages are held to their own bounds at the inputs they were given (swa_util).  For the whole run, the turned rows are off by at most
r = u |x'| + 2^-21 (|x| + |its partner|), so that with d = the row's largest scale (|q'| r_k + r_q |k'| + r_q r_k) summed over the head

    P        off by at most g P, g = exp(2 d) - 1 (numerator exp(d), row sum exp(d))
    dS       off by at most g |dS| + (1 + g) P sum g P |dP|  =: w (delta is the sum of P dP; dP has exact operands)
    dQ', dK' off by at most scale (w |K'| + (|dS| + w) r_k), and alike with Q'; dV by sum g P |dO|

which is added to the backward's own bound, taken there; the turn back adds |a| + |b| of a pair, and its own rounding.
"""
import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, Reference, inputs, visible

pytestmark = pytest.mark.gpu


def pair(x, n):
    """The other half of a pair, halves of the first 2 n columns; what does not turn has none."""
    y = torch.zeros_like(x)
    y[..., :n], y[..., n:2 * n] = x[..., n:2 * n], x[..., :n]
    return y


def turn(x, angle):
    n = angle.shape[-1]
    c, s = angle.cos()[None, :, None], angle.sin()[None, :, None]
    one, two = x[..., :n], x[..., n:2 * n]
    return torch.cat([one * c - two * s, two * c + one * s, x[..., 2 * n:]], -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim,rotary,heads,kv_heads", [(128, 128, 4, 2), (64, 32, 3, 1)])
@pytest.mark.parametrize("seq,window,sinks", [(1, (-1, 0), 0), (65, (20, 0), 3), (300, (100, 0), 4)])
def test_training_step(dtype, dim, rotary, heads, kv_heads, seq, window, sinks):
    q, k, v, do = inputs(2, seq, seq, heads, kv_heads, dim, dtype, seed=7, std=0.5)
    freqs, _ = ua.rope_freqs(rotary, device=DEV)
    q1, k1 = ua.rope_fwd(q, k, freqs, start=11)
    out, lse = ua.swa_fwd(q1, k1, v, window=window, sinks=sinks)
    dq1, dk1, dv = ua.swa_bwd(do, q1, k1, v, out, lse, window=window, sinks=sinks)
    dq, dk = ua.rope_bwd(dq1, dk1, freqs, start=11)

    seen = visible(seq, seq, window, sinks)
    ref = Reference(q1, k1, v, seen, dout=do)
    ref.check(out=out, lse=lse, dq=dq1, dk=dk1, dv=dv)

    n, u, group, scale = rotary // 2, torch.finfo(dtype).eps / 2, heads // kv_heads, dim ** -0.5
    angle = (11 + torch.arange(seq, device=DEV)).double()[:, None] * freqs.double()
    leaves = [x.double().requires_grad_() for x in (q, k, v)]
    by_head = lambda x, m: x.permute(0, 2, 1, 3).repeat_interleave(m, dim=1)  # noqa: E731
    Q, K, V = by_head(turn(leaves[0], angle), 1), by_head(turn(leaves[1], angle), group), by_head(leaves[2], group)
    P = torch.softmax((torch.matmul(Q, K.transpose(-1, -2)) * scale).masked_fill(~seen, -torch.inf), -1)
    O, DO = torch.matmul(P, V), by_head(do.double(), 1)
    want = torch.autograd.grad(O, leaves, DO)

    with torch.no_grad():
        step = 2.0 ** -25 if dtype == torch.float16 else 0.0
        off = lambda x, y: u * y.abs() + step + 2.0 ** -21 * (x.abs() + pair(x.abs(), n))  # noqa: E731
        RQ = by_head(off(q.double(), turn(q.double(), angle)), 1)
        RK = by_head(off(k.double(), turn(k.double(), angle)), group)
        d = scale * (torch.matmul(Q.abs(), RK.transpose(-1, -2)) + torch.matmul(RQ, (K.abs() + RK).transpose(-1, -2)))
        g = torch.expm1(2 * d.masked_fill(~seen, 0).amax(-1, keepdim=True))
        dP = torch.matmul(DO, V.transpose(-1, -2))
        dS = P * (dP - (P * dP).sum(-1, keepdim=True))
        w = g * dS.abs() + (1 + g) * P * (g * P * dP.abs()).sum(-1, keepdim=True)
        back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
        share = lambda x: back(x.unflatten(1, (kv_heads, group)).sum(2))  # noqa: E731
        both = dS.abs() + w
        moved = {"dq": back(scale * (torch.matmul(w, K.abs()) + torch.matmul(both, RK))),
                 "dk": share(scale * (torch.matmul(w.transpose(-1, -2), Q.abs()) + torch.matmul(both.transpose(-1, -2), RQ))),
                 "dv": share(torch.matmul((g * P).transpose(-1, -2), DO.abs()))}
        for name, got, exact in (("dq", dq, want[0]), ("dk", dk, want[1]), ("dv", dv, want[2])):
            bound = getattr(ref, name + "_bound") + moved[name]
            if name != "dv":
                bound = torch.cat([(bound + pair(bound, n))[..., :2 * n], bound[..., 2 * n:]], -1)     # |cos|, |sin| <= 1
                size = exact.abs() + bound                                                              # the turn back's input and result
                bound = bound + u * size + step + 2.0 ** -20 * (size + pair(size, n))                  # (a turned pair is at most sqrt 2 of it)
            err = (got.double() - exact).abs()
            assert torch.isfinite(got).all() and (err <= bound).all(), (name, float((err - bound).max()), float(err.max()))
