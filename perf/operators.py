"""Sliding-window attention and rotary positions as users call them, as cases for timing: what a program has in
hand before the call, the call, and what it cannot do without.  With ``own`` a pass calls this framework's operators, otherwise it
computes them in their plain form, elementary torch operations in 32 bits.

Families of cases (``kind``):

* ``swa``     attention in which a query sees the keys of a window around its position and the first ``sinks`` keys of the
              sequence: the forward alone (prompts, evaluation) or forward and backward (a training step).  Keys and values may have fewer
              heads than queries; ``q_start`` places the queries against the keys (a shard of a longer sequence).
* ``decode``  a few new tokens of every sequence against its cache, whose lengths are on the device.
* ``rope``    rotary positions of Q and K, forward, or of their gradients, backward.
* ``append``  the serving form: Q and K of the new tokens rotated, K and V written to their places in the cache.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PAIRS_MAX = 8 * 16384 * 16384       # query-key pairs, hidden ones too, of the largest case
CACHE_MAX = 64 * 16384 * 8 * 128    # elements of the largest key cache
ROPE_MAX = 2 * 8192 * 40 * 128      # elements of Q and K together of the largest rotation


def _swa(dtype, dim, batch, heads, kv_heads, seq_q, seq_k, left, right, sinks, backward, q_start=-1, packed_kv=False):
    return dict(kind="swa", dtype=dtype, dim=dim, batch=batch, heads=heads, kv_heads=kv_heads, seq_q=seq_q, seq_k=seq_k, left=left, right=right,
                sinks=sinks, backward=backward, q_start=q_start if q_start >= 0 else seq_k - seq_q, packed_kv=packed_kv)


def _decode(dtype, dim, batch, tokens, heads, kv_heads, room, shortest, longest, left, sinks):
    return dict(kind="decode", dtype=dtype, dim=dim, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, room=room, shortest=shortest,
                longest=longest, left=left, sinks=sinks)


def _rope(dtype, dim, rotary, batch, seq, heads, kv_heads, start, interleaved, backward, scattered=False):
    return dict(kind="rope", dtype=dtype, dim=dim, rotary=rotary, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, start=start,
                interleaved=interleaved, backward=backward, scattered=scattered)


def _append(dtype, dim, rotary, batch, tokens, heads, kv_heads, room, shortest, longest, interleaved):
    return dict(kind="append", dtype=dtype, dim=dim, rotary=rotary, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, room=room,
                shortest=shortest, longest=longest, interleaved=interleaved)


def listed():
    cases = [
        # a prompt of one short sentence: all latency
        ("fwd_one_tile", _swa("bf16", 128, 1, 4, 2, 100, 100, 31, 0, 2, False)),
        # prompts of an odd length, small heads, K and V as views of one projection's output
        ("fwd_ragged_fp16", _swa("fp16", 64, 2, 12, 4, 1777, 1777, 511, 0, 3, False, packed_kv=True)),
        # an ordinary training step's layer
        ("train_4k", _swa("bf16", 128, 1, 16, 16, 4096, 4096, 1023, 0, 4, True)),
        # the longest: a training step over a long sequence, four query heads on each key head
        ("train_gqa_16k", _swa("bf16", 128, 1, 8, 2, 16384, 16384, 4095, 0, 16, True)),
        # one rank's queries against the chunk of keys that another rank sent: the last rows see none of them
        ("train_shard_fp16", _swa("fp16", 64, 2, 10, 5, 1333, 2048, 700, 0, 0, True, q_start=1500)),
        # one sequence answers, a window over its cache
        ("decode_one", _decode("bf16", 128, 1, 1, 32, 8, 4096, 4000, 4000, 1023, 4)),
        # a serving batch whose layer has no window: the whole caches are read
        ("decode_batch_16k", _decode("bf16", 128, 64, 1, 32, 8, 16384, 8192, 16384, -1, 0)),
        # a few tokens proposed at once, seven query heads on a key head, young and empty sequences among the batch
        ("decode_ragged_fp16", _decode("fp16", 64, 9, 3, 14, 2, 1000, 0, 1000, 299, 5)),
        # Q and K of a training step
        ("rope_8k", _rope("bf16", 128, 128, 2, 8192, 32, 8, 0, False, False)),
        # gradients of packed sequences far out, in 32 bits, pairs side by side, a part of the head
        ("rope_far_bwd_fp32", _rope("fp32", 64, 48, 3, 1111, 6, 6, 900000, True, True, scattered=True)),
        # one sequence answers
        ("append_one", _append("bf16", 128, 128, 1, 1, 32, 8, 4096, 4000, 4000, False)),
        # a serving batch, a few tokens each, two of them still without room for all
        ("append_batch", _append("fp16", 64, 32, 48, 4, 14, 2, 1024, 2, 1024, True)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choices(("swa", "decode", "rope", "append"), (5, 4, 2, 1))[0]
    dtype, dim = rng.choice(("bf16", "bf16", "fp16")), rng.choice((64, 128, 128))
    kv_heads, group = rng.choice((1, 2, 3, 5, 8)), rng.choice((1, 1, 2, 4, 7))
    heads = kv_heads * group
    if kind == "swa":
        batch, backward = rng.choice((1, 1, 2, 3)), rng.random() < 0.6
        seq_k = _log_int(rng, 64, 16384)
        seq_q = seq_k if rng.random() < 0.6 else _log_int(rng, 1, seq_k)
        left = -1 if rng.random() < 0.15 else _log_int(rng, 64, 4096)
        right = rng.choice((0, 0, 0, 0, -1, 64, 130)) if left >= 0 else 0
        start = seq_k - seq_q if rng.random() < 0.7 else rng.randint(0, seq_k)
        return _swa(dtype, dim, batch, heads, kv_heads, seq_q, seq_k, left, right, rng.choice((0, 1, 4, 70)), backward, q_start=start,
                    packed_kv=rng.random() < 0.3)
    if kind == "decode":
        room = _log_int(rng, 64, 32768)
        longest = rng.randint(1, room)
        return _decode(dtype, dim, _log_int(rng, 1, 96), rng.choice((1, 1, 1, 2, 3, 5)), heads, kv_heads, room, rng.randint(0, longest), longest,
                       rng.choice((-1, _log_int(rng, 64, 4096))), rng.choice((0, 1, 4, 70)))
    rotary = rng.choice((dim, dim, dim // 2, dim - 16, 20))
    if kind == "rope":
        dtype = rng.choice((dtype, dtype, "fp32"))
        return _rope(dtype, dim, rotary, rng.choice((1, 2, 3)), _log_int(rng, 1, 16384), heads, kv_heads, rng.choice((0, _log_int(rng, 1, 2000000))),
                     rng.random() < 0.5, rng.random() < 0.5, scattered=rng.random() < 0.4)
    room = _log_int(rng, 16, 4096)
    longest = rng.randint(1, room)
    return _append(dtype, dim, rotary, _log_int(rng, 1, 64), rng.choice((1, 1, 2, 4)), heads, kv_heads, room, rng.randint(0, longest), longest,
                   rng.random() < 0.5)


def draw(rng):
    while True:
        c = _draw_once(rng)
        if c["kind"] == "swa":
            fits = c["batch"] * c["heads"] * c["seq_q"] * c["seq_k"] <= PAIRS_MAX
        elif c["kind"] == "rope":
            fits = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"]) * c["dim"] * (2 if c["dtype"] == "fp32" else 1) <= ROPE_MAX
        else:
            fits = c["batch"] * c["room"] * c["kv_heads"] * c["dim"] <= (CACHE_MAX if c["kind"] == "decode" else CACHE_MAX // 64)
        if fits:
            return c


def _lengths(case):
    """The cache lengths of a batch, spread over the case's range."""
    return np.linspace(case["shortest"], case["longest"], case["batch"]).astype(np.int64)


def _frequencies(rotary):
    return 10000.0 ** (-np.arange(0, rotary, 2, dtype=np.float64) / rotary)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt, dim, kind = TYPES[case["dtype"]], case["dim"], case["kind"]

    def normal(*shape):
        return torch.empty(*shape, dtype=dt, device=DEVICE).normal_(generator=g)

    s = dict(case=case)
    if kind == "swa":
        s["q"] = normal(case["batch"], case["seq_q"], case["heads"], dim)
        if case["packed_kv"]:
            kv = normal(case["batch"], case["seq_k"], 2, case["kv_heads"], dim)
            s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        else:
            s["k"], s["v"] = (normal(case["batch"], case["seq_k"], case["kv_heads"], dim) for _ in range(2))
        if case["backward"]:
            s["dout"] = normal(case["batch"], case["seq_q"], case["heads"], dim)
        return s
    if kind in ("decode", "append"):
        order = torch.randperm(case["batch"], generator=g, device=DEVICE)
        s["lens"] = torch.as_tensor(_lengths(case), device=DEVICE)[order].to(torch.int32)
        s["q"] = normal(case["batch"], case["tokens"], case["heads"], dim)
        s["k_cache"], s["v_cache"] = (normal(case["batch"], case["room"], case["kv_heads"], dim) for _ in range(2))
    if kind == "append":
        s["k"], s["v"] = (normal(case["batch"], case["tokens"], case["kv_heads"], dim) for _ in range(2))
    if kind == "rope":
        s["q"] = normal(case["batch"], case["seq"], case["heads"], dim)
        s["k"] = normal(case["batch"], case["seq"], case["kv_heads"], dim)
        s["positions"] = None
        if case["scattered"]:               # positions of packed sequences, in no order
            s["positions"] = case["start"] + torch.randint(0, max(case["seq"], 2), (case["batch"], case["seq"]), generator=g, device=DEVICE)
    if kind in ("rope", "append"):
        s["freqs"] = torch.as_tensor(_frequencies(case["rotary"]), device=DEVICE)
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _visible(case):
    """[seq_q, seq_k]: which keys a query sees."""
    pos = case["q_start"] + torch.arange(case["seq_q"], device=DEVICE)[:, None]
    key = torch.arange(case["seq_k"], device=DEVICE)[None, :]
    seen = torch.ones(case["seq_q"], case["seq_k"], dtype=torch.bool, device=DEVICE)
    if case["right"] >= 0:
        seen &= key <= pos + case["right"]
    if case["left"] >= 0:
        seen &= (key >= pos - case["left"]) | (key < case["sinks"])
    return seen


def _softmax(scores, hidden):
    """(P, row sums' logarithm) of scores in which `hidden` ones do not count; rows that see nothing: 0 and -inf."""
    scores = scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = (scores - top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p /= torch.where(total == 0, torch.ones_like(total), total)
    return p, (top + total.log()).squeeze(-1)


def _by_kv_head(x, kv_heads):
    """[B, S, H, D] -> float [B, kv_heads, H / kv_heads, S, D]"""
    b, s, h, d = x.shape
    return x.float().permute(0, 2, 1, 3).reshape(b, kv_heads, h // kv_heads, s, d)


def _rows(x, dtype):
    """[B, kv_heads, group, S, D] -> [B, S, H, D] of a type"""
    b, hk, g, s, d = x.shape
    return x.reshape(b, hk * g, s, d).permute(0, 2, 1, 3).to(dtype).contiguous()


def _plain_swa(s):
    case, hk = s["case"], s["case"]["kv_heads"]
    scale, dt = case["dim"] ** -0.5, s["q"].dtype
    q, k, v = _by_kv_head(s["q"], hk), _by_kv_head(s["k"], hk), _by_kv_head(s["v"], hk)
    hidden = ~_visible(case)
    p, lse = _softmax(torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(scale), hidden)
    out = torch.matmul(p, v)
    res = {"out": _rows(out, dt), "lse": lse.reshape(case["batch"], case["heads"], case["seq_q"])}
    if case["backward"]:
        do = _by_kv_head(s["dout"], hk)
        delta = (do * out).sum(dim=-1, keepdim=True)
        dv = torch.matmul(p.transpose(-1, -2), do).sum(dim=2, keepdim=True)
        ds = torch.matmul(do, v.transpose(-1, -2).contiguous()).sub_(delta).mul_(p).mul_(scale)
        del p
        dq = torch.matmul(ds, k)
        dk = torch.matmul(ds.transpose(-1, -2), q).sum(dim=2, keepdim=True)
        res |= {"dq": _rows(dq, dt), "dk": _rows(dk, dt), "dv": _rows(dv, dt)}
    return res


def _plain_decode(s):
    case, hk = s["case"], s["case"]["kv_heads"]
    q, k, v = _by_kv_head(s["q"], hk), _by_kv_head(s["k_cache"], hk), _by_kv_head(s["v_cache"], hk)
    pos = (s["lens"][:, None] - case["tokens"] + torch.arange(case["tokens"], device=DEVICE))[:, :, None]
    key = torch.arange(case["room"], device=DEVICE)
    seen = key <= pos
    if case["left"] >= 0:
        seen &= (key >= pos - case["left"]) | (key < case["sinks"])
    p, lse = _softmax(torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(case["dim"] ** -0.5), ~seen[:, None, None])
    return {"out": _rows(torch.matmul(p, v), s["q"].dtype), "lse": lse.reshape(case["batch"], case["heads"], case["tokens"])}


def _turn(x, pos, freqs, interleaved, sign):
    """Pairs of the first 2 * len(freqs) entries of x's heads turned by pos * freqs; pos [B, S] or [S]."""
    angle = (pos.double()[..., None] * freqs)[..., None, :]
    cos, sin = angle.cos().float(), sign * angle.sin().float()
    n = 2 * freqs.numel()
    f = x.float()
    if interleaved:
        a, b = f[..., 0:n:2], f[..., 1:n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = f[..., :n // 2], f[..., n // 2:n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, f[..., n:]), dim=-1).to(x.dtype)


def _plain_rope(s):
    case = s["case"]
    pos = s["positions"] if s["positions"] is not None else case["start"] + torch.arange(case["seq"], device=DEVICE)
    sign = -1.0 if case["backward"] else 1.0
    return {n: _turn(s[n], pos, s["freqs"], case["interleaved"], sign) for n in ("q", "k")}


def _plain_append(s):
    case = s["case"]
    pos = s["lens"].long()[:, None] - case["tokens"] + torch.arange(case["tokens"], device=DEVICE)
    q, k = (_turn(s[n], pos, s["freqs"], case["interleaved"], 1.0) for n in ("q", "k"))
    b, t = torch.nonzero((pos >= 0) & (pos < case["room"]), as_tuple=True)
    s["k_cache"][b, pos[b, t]] = k[b, t]
    s["v_cache"][b, pos[b, t]] = s["v"][b, t]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


PLAIN = {"swa": _plain_swa, "decode": _plain_decode, "rope": _plain_rope, "append": _plain_append}


# ---- the framework's operators -----------------------------------------------------------------------------------------


def _own_swa(s):
    import ultraattn_amd as ua
    case = s["case"]
    how = dict(window=(case["left"], case["right"]), sinks=case["sinks"], q_start=case["q_start"])
    out, lse = ua.swa_fwd(s["q"], s["k"], s["v"], **how)
    if not case["backward"]:
        return {"out": out, "lse": lse}
    dq, dk, dv = ua.swa_bwd(s["dout"], s["q"], s["k"], s["v"], out, lse, **how)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _own_decode(s):
    import ultraattn_amd as ua
    out, lse = ua.swa_decode(s["q"], s["k_cache"], s["v_cache"], s["lens"], window=s["case"]["left"], sinks=s["case"]["sinks"])
    return {"out": out, "lse": lse}


def _own_rope(s):
    import ultraattn_amd as ua
    case = s["case"]
    q, k = (ua.rope_bwd if case["backward"] else ua.rope_fwd)(s["q"], s["k"], s["freqs"], positions=s["positions"], start=case["start"],
                                                              interleaved=case["interleaved"])
    return {"q": q, "k": k}


def _own_append(s):
    import ultraattn_amd as ua
    q = ua.rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["lens"], s["freqs"], interleaved=s["case"]["interleaved"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


OWN = {"swa": _own_swa, "decode": _own_decode, "rope": _own_rope, "append": _own_append}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---- what a pass cannot do without, and what it has to give --------------------------------------------------------------


def _spans(case, pos, keys):
    """Of queries at `pos`: (first key of the window, end of the window, end of the sinks before it)."""
    left, right = case["left"], case.get("right", 0)
    hi = np.clip(pos + right + 1, 0, keys) if right >= 0 else np.full_like(pos, keys)
    lo = np.clip(pos - left, 0, hi) if left >= 0 else np.zeros_like(pos)
    return lo, hi, np.minimum(case["sinks"] if left >= 0 else 0, lo)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "swa":
        pos = case["q_start"] + np.arange(case["seq_q"], dtype=np.int64)
        lo, hi, sinks = _spans(case, pos, case["seq_k"])
        pairs = int((hi - lo + sinks).sum()) * case["batch"] * case["heads"]
        edge = np.zeros(case["seq_k"] + 1, dtype=np.int64)
        np.add.at(edge, lo, 1)
        np.add.at(edge, hi, -1)
        edge[0] += 1
        edge[int(sinks.max())] -= 1
        keys = int((np.cumsum(edge[:-1]) > 0).sum())
        q_bytes = case["batch"] * case["seq_q"] * case["heads"] * case["dim"] * e
        kv_bytes = case["batch"] * case["kv_heads"] * case["dim"] * e
        rows = case["batch"] * case["seq_q"] * case["heads"] * 4
        both = case["backward"]
        return {"bytes": q_bytes * (4 if both else 2) + kv_bytes * (2 * keys + (2 * case["seq_k"] if both else 0)) + rows,
                "flops": pairs * case["dim"] * (14 if both else 4)}
    if case["kind"] == "decode":
        total = pairs = 0
        for n in _lengths(case):
            pos = n - case["tokens"] + np.arange(case["tokens"])
            lo, hi, sinks = _spans(case, pos, int(n))
            pairs += int((hi - lo + sinks).sum())
            total += int(hi.max() - lo.min() + min(int(sinks.max()), int(lo.min())))
        rows = case["batch"] * case["tokens"] * case["heads"]
        return {"bytes": total * case["kv_heads"] * case["dim"] * 2 * e + rows * (2 * case["dim"] * e + 4),
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    heads = case["heads"] + case["kv_heads"]
    if case["kind"] == "rope":
        n = case["batch"] * case["seq"] * heads
        return {"bytes": 2 * n * case["dim"] * e + (case["batch"] * case["seq"] * 8 if case["scattered"] else 0), "flops": 3 * n * case["rotary"]}
    n = case["batch"] * case["tokens"]
    return {"bytes": 2 * n * (heads + case["kv_heads"]) * case["dim"] * e, "flops": 3 * n * heads * case["rotary"]}


def _exact_attention(q, k, v, seen, dout=None):
    """One key head's queries [G, S, D] in 64 bits: output, log of the row sums, and gradients by differentiating the definition."""
    q, k, v = (x.double().requires_grad_(dout is not None) for x in (q, k, v))
    scores = torch.einsum("gsd,td->gst", q, k) / math.sqrt(q.shape[-1])
    scores = torch.where(seen, scores, torch.full_like(scores[:1, :1, :1], -1e300))
    some = seen.any(dim=-1)
    p = torch.softmax(scores, dim=-1) * some[:, None]
    out = torch.einsum("gst,td->gsd", p, v)
    lse = torch.where(some, torch.logsumexp(scores.detach(), dim=-1), torch.full_like(out[..., 0].detach(), -math.inf))
    grads = torch.autograd.grad(out, (q, k, v), dout.double()) if dout is not None else ()
    return (out.detach(), lse, *grads)


def _exact_turn(x, pos, freqs, interleaved, back):
    """The pairs as complex numbers."""
    n = 2 * freqs.numel()
    z = x.double()
    pairs = z[..., :n].unflatten(-1, (n // 2, 2)) if interleaved else z[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2)
    angle = pos.double().unsqueeze(-1) * freqs
    turn = torch.polar(torch.ones_like(angle), -angle if back else angle).unsqueeze(-2)
    w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    w = w.flatten(-2) if interleaved else w.transpose(-1, -2).flatten(-2)
    return torch.cat((w, z[..., n:]), dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("swa", "decode"):
        k, v = (s["k"], s["v"]) if case["kind"] == "swa" else (s["k_cache"], s["v_cache"])
        group, back = case["heads"] // case["kv_heads"], case.get("backward", False)
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        lse = torch.empty(out.shape[0], out.shape[2], out.shape[1], dtype=torch.float64, device=DEVICE)
        res = {"out": out, "lse": lse}
        if back:
            res |= {"dq": torch.empty_like(out), "dk": torch.empty(k.shape, dtype=torch.float64, device=DEVICE),
                    "dv": torch.empty(k.shape, dtype=torch.float64, device=DEVICE)}
        key = torch.arange(k.shape[1], device=DEVICE)
        for b in range(case["batch"]):
            first = case["q_start"] if case["kind"] == "swa" else int(s["lens"][b]) - case["tokens"]
            back_by = (first + torch.arange(out.shape[1], device=DEVICE))[:, None] - key      # how far behind the query a key is
            far = (back_by > case["left"]) & (key >= case["sinks"]) if case["left"] >= 0 else torch.zeros_like(back_by, dtype=torch.bool)
            right = case.get("right", 0)
            seen = ~(far | (back_by < -right)) if right >= 0 else ~far
            for h in range(case["kv_heads"]):
                mine = slice(h * group, (h + 1) * group)
                got = _exact_attention(s["q"][b, :, mine].transpose(0, 1), k[b, :, h], v[b, :, h], seen,
                                       s["dout"][b, :, mine].transpose(0, 1) if back else None)
                out[b, :, mine], lse[b, mine] = got[0].transpose(0, 1), got[1]
                if back:
                    res["dq"][b, :, mine], res["dk"][b, :, h], res["dv"][b, :, h] = got[2].transpose(0, 1), got[3], got[4]
        return res
    if case["kind"] == "rope":
        pos = s["positions"] if s["positions"] is not None else torch.arange(case["start"], case["start"] + case["seq"], device=DEVICE)
        return {n: _exact_turn(s[n], pos, s["freqs"], case["interleaved"], case["backward"]) for n in ("q", "k")}
    pos = s["lens"].long()[:, None] + torch.arange(-case["tokens"], 0, device=DEVICE)
    res = {"q": _exact_turn(s["q"], pos, s["freqs"], case["interleaved"], False), "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
    k = _exact_turn(s["k"], pos, s["freqs"], case["interleaved"], False)
    for b in range(case["batch"]):
        for t in range(case["tokens"]):
            at = int(pos[b, t])
            if 0 <= at < case["room"]:
                res["k_cache"][b, at], res["v_cache"][b, at] = k[b, t], s["v"][b, t].double()
    return res
