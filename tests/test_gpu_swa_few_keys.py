"""Rows of 2 to 8 keys make their delta from their output as it was before it was rounded: dQ against the definition, under a bound without O's rounding.

Bound, in the terms of swa_util (u half a step of the type, e = 2^-24): delta is a sum of n products of P, off by ep, and dO V, a sum of D products off by
(D + 4) e, so |d delta| <= (ep + (n + D + 4) e) sum P |dO| |V|; dP likewise; dS is rounded once (fp16 holds it times 2^8 at least
while dP is below 128: 2^-33 where it is small), and dQ.
"""
import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, Reference, inputs, visible

pytestmark = pytest.mark.gpu


def dq_bound(q, k, v, do, seen):
    """(dQ, bound, number of keys) of one sequence, [H, Sq, D]."""
    u, e, dim = torch.finfo(q.dtype).eps / 2, 2.0 ** -24, q.shape[-1]
    scale, tiny = dim ** -0.5, 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    group = q.shape[2] // k.shape[2]
    heads = lambda x, n: x[0].double().transpose(0, 1).repeat_interleave(n, 0)  # noqa: E731
    Q, K, V, DO = heads(q, 1), heads(k, group), heads(v, group), heads(do, 1)
    t = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    S = (torch.matmul(Q, t(K)) * scale).masked_fill(~seen, -torch.inf)
    n = seen.sum(-1)[None, :, None].double()
    P = torch.softmax(S, -1).nan_to_num(0.0)
    size = ((dim + 4) * e * scale * torch.matmul(Q.abs(), t(K).abs())).masked_fill(~seen, 0).amax(-1, keepdim=True)
    ep = 2 * size + 8 * e * S.masked_fill(~seen, 0).abs().amax(-1, keepdim=True).clamp_min(1) + n * e
    dP, terms = torch.matmul(DO, t(V)), torch.matmul(DO.abs(), t(V).abs())
    delta = (P * dP).sum(-1, keepdim=True)
    # P's own error moves delta by its differences only, but ep of every term bounds that
    d_delta = (ep + (n + dim + 4) * e) * (P * terms).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    ds = (u + ep + 4 * e) * dS.abs() + (1 + u) * P * (d_delta + (dim + 4) * e * terms) + tiny * 2.0 ** -8 * seen
    dQ = torch.matmul(dS, K) * scale
    return dQ, (u * dQ.abs() + tiny + torch.matmul(ds + n * e * dS.abs(), K.abs()) * scale) * 1.01, n.flatten()


# windows and sinks that are full at 8 and at 9 keys, growing rows at the start, rows that run out of keys, sinks before the window
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks,start", [((7, 0), 0, None), ((4, 0), 3, 100), ((3, 0), 4, 100), ((3, 0), 5, 100), ((0, 0), 8, 150), ((2, 3), 2, 150), ((-1, 0), 0, 0),
                                                ((100, 0), 0, 200)])
def test_remade_deltas(dtype, dim, window, sinks, start):
    q, k, v, do = inputs(1, 200, 300, 6, 3, dim, dtype, 7)
    seen = visible(200, 300, window, sinks, start)
    out, lse = ua.swa_fwd(q, k, v, window, sinks, None, start)
    dq = ua.swa_bwd(do, q, k, v, out, lse, window, sinks, None, start)[0]
    want, bound, n = dq_bound(q, k, v, do, seen)
    few = (n >= 2) & (n <= 8)
    assert few.any() or sinks == 5
    got = dq[0].transpose(0, 1).double()
    over = ((got - want).abs() > bound)[:, few]
    assert not over.any(), (int(over.sum()), float(((got - want).abs() / bound)[:, few].max()))
    Reference(q, k, v, seen, dout=do).check(out=out, lse=lse, dq=dq)                    # and all rows, those of nine keys among them, under the whole bound


def test_both_sides_of_the_limit():
    """Eight keys are remade, nine are not: O's rounding in delta takes some of those rows over the bound without it, so the bound would notice."""
    count = {}
    for window, sinks in (((4, 0), 3), ((3, 0), 5)):
        q, k, v, do = inputs(1, 200, 300, 6, 3, 64, torch.bfloat16, 7)
        seen = visible(200, 300, window, sinks, 100)
        out, lse = ua.swa_fwd(q, k, v, window, sinks, None, 100)
        dq = ua.swa_bwd(do, q, k, v, out, lse, window, sinks, None, 100)[0]
        want, bound, n = dq_bound(q, k, v, do, seen)
        off = ((dq[0].transpose(0, 1).double() - want).abs() > bound).any(0).any(-1)
        for keys in (8, 9):
            if (n == keys).any():
                count[keys] = int(off[n == keys].sum())
    assert count[8] == 0 and count[9] > 0, count
