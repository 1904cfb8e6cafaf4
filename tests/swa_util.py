"""Sliding-window attention in 64 bits, and how far a result in 32 with operands of 16 may be off: what its roundings add up to at most.

u is half a step of the type (2^-8 for bf16's 8 bits, 2^-11 for fp16's 11: `eps / 2`), e = 2^-24 half a step of fp32.

    scores   S is a sum of D products: |dS| <= (D + 4) e scale sum |q| |k| =: es (its row's largest is used)
    P        relative: es twice (numerator and row sum), exponential and scaling 8 e max(1, |S|), sums of n terms n e =: ep
    O        u |O| + (u + ep + n e) sum P |V|; P in fp16 below its normal range is off by 2^-25 of the row's reference, which is at most the row sum
    LSE      es + n e + 8 e max(1, |LSE|)
    dV       u |dV| + (u + ep + e n) sum P |dO|
    dS       P (dP - delta) with |d dP| <= (D + 4) e sum |dO| |V| and |d delta| <= sum |dO| |dO_bound| of the forward's result, which the backward is given:
             (u + ep + 4 e) |dS| + P (...); fp16: 2^-25 beside that
    any      result in fp16 is rounded to a multiple of 2^-24 where it is below 2^-14: 2^-25 more (u |x| is less there)
    dQ, dK   u |dQ| + scale sum_j (dS's bound + n e |dS|) |K|, and alike
"""
import math

import torch

DEV = "cuda:0"


def inputs(batch, seq_q, seq_k, heads, kv_heads, dim, dtype, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = lambda s, h: (torch.randn(batch, s, h, dim, generator=g, device=DEV) * std).to(dtype)  # noqa: E731
    return make(seq_q, heads), make(seq_k, kv_heads), make(seq_k, kv_heads), make(seq_q, heads)


def visible(seq_q, seq_k, window, sinks=0, q_start=None, k_start=0):
    q_start = k_start + seq_k - seq_q if q_start is None else q_start
    p = [q_start + i for i in range(seq_q)]
    n = torch.arange(seq_k, device=DEV)[None]
    # the differences are made of Python numbers: positions may be anywhere
    d = torch.tensor([min(max(x - k_start, -2 ** 40), 2 ** 40) for x in p], device=DEV, dtype=torch.int64)[:, None]
    left, right = window
    seen = torch.ones(seq_q, seq_k, dtype=torch.bool, device=DEV)
    if right >= 0:
        seen &= n <= d + right
    if left >= 0:
        seen &= (n >= d - left) | (n < min(max(sinks - k_start, 0), 2 ** 40))
    return seen


class Reference:
    """Everything [B, H, Sq, Sk] in float64; `seen` [Sq, Sk] or [B, 1, Sq, Sk]."""

    def __init__(self, q, k, v, seen, scale=None, dout=None):
        u, e, dim = torch.finfo(q.dtype).eps / 2, 2.0 ** -24, q.shape[-1]
        tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
        scale = dim ** -0.5 if scale is None else scale
        group = q.shape[2] // k.shape[2]
        heads = lambda x, n: x.double().permute(0, 2, 1, 3).repeat_interleave(n, dim=1)  # noqa: E731
        Q, K, V = heads(q, 1), heads(k, group), heads(v, group)
        back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
        mm = lambda a, b: torch.matmul(a, b)  # noqa: E731
        S = mm(Q, K.transpose(-1, -2)) * scale
        hide = ~seen.expand_as(S)
        S.masked_fill_(hide, -math.inf)
        n = seen.sum(-1, keepdim=True).double()
        some = n > 0
        lse = torch.where(some.expand_as(S[..., :1]), torch.logsumexp(S, -1, keepdim=True), torch.full_like(S[..., :1], -math.inf))
        P = torch.exp(S - torch.where(some, lse, torch.zeros_like(lse)))
        es = (dim + 4) * e * scale * mm(Q.abs(), K.abs().transpose(-1, -2)).masked_fill(hide, 0)
        es = es.amax(-1, keepdim=True) if es.shape[-1] else torch.zeros_like(lse)
        big = S.masked_fill(hide, 0).abs().amax(-1, keepdim=True).clamp_min(1) if es.shape[-1] and S.shape[-1] else torch.ones_like(lse)
        ep = 2 * es + 8 * e * big + n * e
        O = mm(P, V)
        o_bound = u * O.abs() + tiny + (u + ep + n * e) * mm(P, V.abs()) + tiny * mm((~hide).double(), V.abs())
        self.out, self.out_bound = back(O), back(o_bound) * 1.01
        self.lse = lse.squeeze(-1)
        self.lse_bound = (es + n * e + 8 * e * lse.abs().clamp_min(1)).squeeze(-1)
        if dout is None:
            return
        DO = heads(dout, 1)
        rows = torch.full_like(n, float(seen.shape[-2] * group))
        share = lambda x: back(x.unflatten(1, (k.shape[2], group)).sum(2))  # noqa: E731
        Pt = P.transpose(-1, -2)
        dV = mm(Pt, DO)
        dv_bound = mm(((u + ep + rows * e) * P).transpose(-1, -2), DO.abs())
        dP, delta = mm(DO, V.transpose(-1, -2)), (DO * O).sum(-1, keepdim=True)
        dS = P * (dP - delta)
        d_err = (DO.abs() * (o_bound * 1.01 + dim * e * O.abs())).sum(-1, keepdim=True) + (dim + 4) * e * mm(DO.abs(), V.abs().transpose(-1, -2))
        ds_bound = (u + ep + 4 * e) * dS.abs() + (1 + u) * P * d_err + tiny * (~hide)
        self.dv, self.dk, self.dq = share(dV), share(mm(dS.transpose(-1, -2), Q) * scale), back(mm(dS, K) * scale)
        self.dv_bound = (u * self.dv.abs() + tiny + share(dv_bound)) * 1.01
        self.dq_bound = (u * self.dq.abs() + tiny + back(mm(ds_bound + n * e * dS.abs(), K.abs()) * scale)) * 1.01
        self.dk_bound = (u * self.dk.abs() + tiny + share(mm((ds_bound + rows * e * dS.abs()).transpose(-1, -2), Q.abs()) * scale)) * 1.01

    def check(self, **got):
        for name, x in got.items():
            want, bound = getattr(self, name), getattr(self, name + "_bound")
            assert x.shape == want.shape, (name, x.shape, want.shape)
            fin = torch.isfinite(want)
            assert torch.equal(torch.isfinite(x), fin), f"{name}: other entries are finite"
            assert torch.equal(x[~fin].double(), want[~fin]), name
            err = (x.double() - want)[fin].abs()
            over = err > bound[fin]
            assert not over.any(), (name, int(over.sum()), float((err / bound[fin].clamp_min(1e-300)).max()), float(err.max()))
