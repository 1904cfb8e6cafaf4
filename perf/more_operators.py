"""A paged cache as a serving program uses it, as cases for timing: what the program has in hand before the call, the call, and what it
cannot do without.  With ``own`` a pass calls this framework's operators, otherwise it computes them in their plain form, elementary torch
operations in 32 bits.

The cache's rows lie in pages ``[n_pages, page, Hk, D]``; row r of sequence b is slot ``r % page`` of page ``table[b, r // page]``.  A step brings up to T
new tokens of every sequence, ``n_new[b]`` of them real, which follow its first ``lens[b] - n_new[b]`` rows.  They are a chain, or a tree of drafted tokens:
``parents[b, t]`` is the token before token t, or -1 where that is the last one of the cache.  Its position counts the tokens before it on its branch.

Families of cases (``kind``):

* ``append``  Q and K of the new tokens rotated by their positions, K and V written to their rows.
* ``decode``  the new tokens against the cache, which holds them already: each sees the cached rows and its own branch.
* ``keep``    after the draft's verification: the rows of the accepted branch are moved together, in all layers of a model.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CACHE_MAX = 64 * 16384 * 8 * 128         # elements of the largest key cache that is attended to
PAIRS_MAX = 16 * 64 * 32 * 8192          # scores, hidden ones too, of the largest decode
APPEND_MAX = 4 * 4096 * 48 * 128         # elements of the largest Q, K and V that are appended
KEEP_MAX = 16 * 48 * 128 * 8 * 128       # elements of the largest key cache of all layers that rows are moved in


def _append(dtype, dim, rotary, batch, tokens, heads, kv_heads, page, shortest, longest, tree, ragged, interleaved):
    return dict(kind="append", dtype=dtype, dim=dim, rotary=rotary, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, page=page,
                shortest=shortest, longest=longest, tree=tree, ragged=ragged, interleaved=interleaved)


def _decode(dtype, dim, batch, tokens, heads, kv_heads, page, shortest, longest, tree, ragged, left, sinks):
    return dict(kind="decode", dtype=dtype, dim=dim, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, page=page, shortest=shortest,
                longest=longest, tree=tree, ragged=ragged, left=left, sinks=sinks)


def _keep(dtype, dim, layers, batch, tokens, path, kv_heads, page, shortest, longest):
    return dict(kind="keep", dtype=dtype, dim=dim, layers=layers, batch=batch, tokens=tokens, path=path, kv_heads=kv_heads, page=page,
                shortest=shortest, longest=longest, ragged=True)


def listed():
    cases = [
        # one sequence answers, a token at a time
        ("append_one", _append("bf16", 128, 128, 1, 1, 32, 8, 16, 4000, 4000, False, False, False)),
        # trees of a serving batch, of different sizes, a part of each head rotated
        ("append_trees_fp16", _append("fp16", 64, 48, 32, 25, 14, 2, 32, 25, 1000, True, True, True)),
        # chunks of prompts on their way into the cache
        ("append_prompts", _append("bf16", 128, 128, 4, 4096, 32, 8, 64, 4096, 9000, False, False, False)),
        # one sequence answers
        ("decode_one", _decode("bf16", 128, 1, 1, 32, 8, 16, 4000, 4000, False, False, -1, 0)),
        # a serving batch: whole caches are read
        ("decode_batch_16k", _decode("bf16", 128, 64, 1, 32, 8, 16, 8192, 16384, False, False, -1, 0)),
        # one sequence verifies a tree
        ("tree_one", _decode("bf16", 128, 1, 26, 32, 8, 32, 2777, 2777, True, False, -1, 0)),
        # a batch verifies large trees, a wide product for every key head
        ("tree_batch_8k", _decode("bf16", 128, 16, 64, 32, 8, 64, 2048, 8192, True, False, -1, 0)),
        # young sequences among a batch, trees of different sizes, a window, pages of no power of two
        ("tree_ragged_fp16", _decode("fp16", 64, 9, 21, 14, 2, 24, 21, 1500, True, True, 299, 5)),
        # as many drafts as a tree may have, every query head on a key head of its own
        ("tree_largest", _decode("fp16", 128, 3, 256, 8, 8, 128, 700, 6000, True, True, -1, 0)),
        # one sequence's accepted branch, all layers of a model
        ("keep_one", _keep("bf16", 128, 32, 1, 26, 6, 8, 16, 1500, 1500)),
        # a serving batch's
        ("keep_batch_fp16", _keep("fp16", 64, 24, 48, 64, 9, 4, 32, 64, 700)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choices(("append", "decode", "keep"), (3, 6, 2))[0]
    dtype, dim = rng.choice(("bf16", "bf16", "fp16")), rng.choice((64, 128, 128))
    kv_heads, group = rng.choice((1, 2, 3, 5, 8)), rng.choice((1, 1, 2, 4, 7))
    page = rng.choice((1, 7, 16, 16, 24, 32, 64, 128, 256))
    tree = rng.random() < 0.6
    tokens = _log_int(rng, 1, 256) if tree else rng.choice((1, 1, 1, 2, 5))
    ragged = rng.random() < 0.5
    longest = tokens + _log_int(rng, 1, 32768)
    shortest = rng.randint(tokens, longest)
    if kind == "append":
        dtype = rng.choice((dtype, dtype, dtype, "fp32"))
        if not tree:
            tokens = _log_int(rng, 1, 4096)
            longest = tokens + _log_int(rng, 1, 8192)
            shortest = rng.randint(tokens, longest)
        return _append(dtype, dim, rng.choice((dim, dim, dim // 2, dim - 16, 20)), _log_int(rng, 1, 64), tokens, kv_heads * group, kv_heads, page, shortest,
                       longest, tree, ragged, rng.random() < 0.5)
    if kind == "keep":
        tokens = _log_int(rng, 2, 256)
        longest = tokens + _log_int(rng, 1, 1024)
        return _keep(dtype, dim, rng.choice((1, 8, 24, 32)), _log_int(rng, 1, 64), tokens, rng.randint(1, min(tokens, 16)), kv_heads, page,
                     rng.randint(tokens, longest), longest)
    left = _log_int(rng, 8, 4096) if rng.random() < 0.3 else -1
    return _decode(dtype, dim, _log_int(rng, 1, 96), tokens, kv_heads * group, kv_heads, page, shortest, longest, tree, ragged, left, rng.choice((0, 1, 4, 70)))


def draw(rng):
    while True:
        c = _draw_once(rng)
        cache = c["batch"] * c["longest"] * c["kv_heads"] * c["dim"]
        if c["kind"] == "append":
            fits = cache <= CACHE_MAX // 8 and c["batch"] * c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] <= APPEND_MAX // TYPES[c["dtype"]].itemsize
        elif c["kind"] == "keep":
            fits = cache * c["layers"] <= KEEP_MAX
        else:
            fits = cache <= CACHE_MAX // 2 and c["batch"] * c["tokens"] * c["heads"] * c["longest"] <= PAIRS_MAX // 2
        if fits:
            return c


def _lengths(case):
    """The cache lengths of a batch, with the new tokens, spread over the case's range."""
    return np.linspace(case["shortest"], case["longest"], case["batch"]).astype(np.int64)


def _counts(case):
    """The new tokens of every sequence."""
    t = np.full(case["batch"], case["tokens"], dtype=np.int64)
    return np.maximum(t - (np.arange(case["batch"]) * 5) % max(case["tokens"] // 2, 1), 1) if case["ragged"] else t


def _frequencies(rotary):
    return 10000.0 ** (-np.arange(0, rotary, 2, dtype=np.float64) / rotary)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt, dim, kind, batch, page = TYPES[case["dtype"]], case["dim"], case["kind"], case["batch"], case["page"]

    def normal(*shape):
        return torch.empty(*shape, dtype=dt, device=DEVICE).normal_(generator=g)

    s = dict(case=case)
    order = torch.randperm(batch, generator=g, device=DEVICE)
    lens, n_new = (torch.as_tensor(x, device=DEVICE)[order] for x in (_lengths(case), _counts(case)))
    most = -(-case["longest"] // page)
    pool = batch * most + 3
    table = torch.randperm(pool, generator=g, device=DEVICE)[:batch * most].reshape(batch, most)
    used = torch.arange(most, device=DEVICE) * page < lens[:, None]
    s["table"] = torch.where(used, table, torch.full_like(table, -1)).to(torch.int32)
    s["lens"] = lens.to(torch.int32)
    s["n_new"] = n_new.to(torch.int32) if case["ragged"] else None
    layers = (case["layers"],) if kind == "keep" else ()
    s["k_pages"], s["v_pages"] = (normal(*layers, pool, page, case["kv_heads"], dim) for _ in range(2))
    if kind == "keep":
        path = torch.rand(batch, case["tokens"], generator=g, device=DEVICE).argsort(dim=1)[:, :case["path"]]
        path = torch.minimum(path, n_new[:, None] - 1).sort(dim=1).values
        s["path"] = path.to(torch.int32)
        kept = torch.randint(1, case["path"] + 1, (batch,), generator=g, device=DEVICE)
        s["n_kept"] = torch.minimum(kept, n_new).to(torch.int32)
        return s
    s["parents"] = None
    if case["tree"]:                        # drafts grow from any of the tokens before them; some sequences have several first ones
        t = torch.arange(case["tokens"], device=DEVICE)
        s["parents"] = (torch.rand(batch, case["tokens"], generator=g, device=DEVICE) * (t + 0.5) - 0.5).floor().clamp(max=t - 1).to(torch.int32)
    s["q"] = normal(batch, case["tokens"], case["heads"], dim)
    if kind == "append":
        s["k"], s["v"] = (normal(batch, case["tokens"], case["kv_heads"], dim) for _ in range(2))
        s["freqs"] = torch.as_tensor(_frequencies(case["rotary"]), device=DEVICE)
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _twice(reach):
    return (torch.matmul(reach, reach) > 0).float()


def _branches(s):
    """[B, T, T]: 1 where token j is token t itself or before it on its branch."""
    case, t = s["case"], torch.arange(s["case"]["tokens"], device=DEVICE)
    if s["parents"] is None:
        return (t[:, None] >= t).float().expand(case["batch"], -1, -1)
    reach = (s["parents"].long()[:, :, None] == t).float() + torch.eye(case["tokens"], device=DEVICE)
    return _twice(_twice(_twice(_twice(_twice(_twice(_twice(_twice(reach))))))))        # branches of up to 256 tokens


def _step(s):
    """(first new row [B, 1], real tokens [B, T], branches [B, T, T], depths [B, T])"""
    case = s["case"]
    t = torch.arange(case["tokens"], device=DEVICE)
    n_new = s["n_new"].long() if s["n_new"] is not None else torch.full_like(s["lens"], case["tokens"]).long()
    base = (s["lens"].long() - n_new)[:, None]
    if s["parents"] is None:
        return base, t < n_new[:, None], None, t.expand(case["batch"], -1)
    branch = _branches(s)
    return base, t < n_new[:, None], branch, branch.sum(dim=-1).long() - 1


def _turn(x, pos, freqs, interleaved):
    """Pairs of the first 2 * len(freqs) entries of x's heads turned by pos * freqs; pos [B, S]."""
    angle = (pos.double()[..., None] * freqs)[..., None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    n = 2 * freqs.numel()
    f = x.float()
    if interleaved:
        a, b = f[..., 0:n:2], f[..., 1:n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = f[..., :n // 2], f[..., n // 2:n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, f[..., n:]), dim=-1).to(x.dtype)


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    base, real, _, depth = _step(s)
    q, k = (_turn(s[n], base + depth, s["freqs"], case["interleaved"]) for n in ("q", "k"))
    b, t = torch.nonzero(real, as_tuple=True)
    row = base[b, 0] + t
    at, slot = s["table"].long()[b, row // page], row % page
    s["k_pages"][at, slot] = k[b, t]
    s["v_pages"][at, slot] = s["v"][b, t]
    return {"q": q * real[..., None, None], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _rows_of(pages, table, kv_heads):
    """float [B, kv_heads, rows, D] of all rows that the table holds, zeros where it has no page"""
    x = pages.float()[table.long().clamp_min(0)] * (table >= 0)[:, :, None, None, None]
    b, n, page, h, d = x.shape
    return x.reshape(b, n * page, h, d).transpose(1, 2)


def _plain_decode(s):
    case, hk = s["case"], s["case"]["kv_heads"]
    base, real, branch, depth = _step(s)
    b, t, h, d = s["q"].shape
    k, v = _rows_of(s["k_pages"], s["table"], hk), _rows_of(s["v_pages"], s["table"], hk)
    row = torch.arange(k.shape[2], device=DEVICE).expand(b, -1)
    new = row - base                                                          # which of the new tokens a row is
    is_new = (new >= 0) & (new < t)
    at = new.clamp(0, t - 1)
    pos = torch.where(is_new, base + depth.gather(1, at), row)[:, None]       # of the rows
    mine = (base + depth)[:, :, None]                                         # of the queries
    if branch is None:
        seen = row[:, None] <= mine
    else:
        seen = torch.where(is_new[:, None], branch.gather(2, at[:, None].expand(-1, t, -1)) > 0, (new < 0)[:, None])
    if case["left"] >= 0:
        seen = seen & ((pos >= mine - case["left"]) | (pos < case["sinks"]))
    seen = seen & real[:, :, None]
    q = s["q"].float().permute(0, 2, 1, 3).reshape(b, hk, h // hk * t, d)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(d ** -0.5).reshape(b, hk, h // hk, t, -1)
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = (scores - top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p /= torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p.reshape(b, hk, h // hk * t, -1), v.contiguous())
    return {"out": out.reshape(b, h, t, d).permute(0, 2, 1, 3).to(s["q"].dtype).contiguous(), "lse": (top + total.log()).reshape(b, h, t)}


def _plain_keep(s):
    case, page = s["case"], s["case"]["page"]
    base = (s["lens"] - s["n_new"]).long()[:, None]
    b, i = torch.nonzero(torch.arange(case["path"], device=DEVICE) < s["n_kept"][:, None], as_tuple=True)
    source, to = (base + s["path"])[b, i], base[b, 0] + i
    table = s["table"].long()
    from_page, to_page = table[b, source // page], table[b, to // page]
    s["k_pages"][:, to_page, to % page] = s["k_pages"][:, from_page, source % page]
    s["v_pages"][:, to_page, to % page] = s["v_pages"][:, from_page, source % page]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


PLAIN = {"append": _plain_append, "decode": _plain_decode, "keep": _plain_keep}


# ---- the framework's operators -----------------------------------------------------------------------------------------


def _own_append(s):
    import ultraattn_amd as ua
    q = ua.paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["freqs"], n_new=s["n_new"], parents=s["parents"],
                        interleaved=s["case"]["interleaved"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_decode(s):
    import ultraattn_amd as ua
    out, lse = ua.paged_decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], n_new=s["n_new"], parents=s["parents"],
                               window=s["case"]["left"], sinks=s["case"]["sinks"])
    return {"out": out, "lse": lse}


def _own_keep(s):
    import ultraattn_amd as ua
    ua.paged_keep(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["n_new"], s["path"], s["n_kept"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


OWN = {"append": _own_append, "decode": _own_decode, "keep": _own_keep}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---- what a pass cannot do without, and what it has to give --------------------------------------------------------------


def work(case):
    e = TYPES[case["dtype"]].itemsize
    lens, n_new = _lengths(case), _counts(case)
    if case["kind"] == "append":
        n = int(n_new.sum())
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": 2 * n * (heads + case["kv_heads"]) * case["dim"] * e, "flops": 3 * n * heads * case["rotary"]}
    if case["kind"] == "keep":
        rows = int(np.minimum(case["path"] / 2, n_new).sum() * case["layers"]) * 2        # K and V, half a path on the average
        return {"bytes": 2 * rows * case["kv_heads"] * case["dim"] * e, "flops": 0}
    keys = pairs = 0
    for n, new in zip(lens.tolist(), n_new.tolist()):
        cached = n - new
        if case["left"] >= 0:                     # (a window's rows, as the first of the new tokens sees them)
            cached = min(cached, case["left"] + min(case["sinks"], max(cached - case["left"], 0)))
        keys += cached + new
        pairs += (cached + (1 if case["tree"] else (new + 1) / 2)) * new                 # of a branch at least the token itself
    rows = int(n_new.sum()) * case["heads"]
    return {"bytes": keys * case["kv_heads"] * case["dim"] * 2 * e + rows * (2 * case["dim"] * e + 4), "flops": 4 * int(pairs) * case["heads"] * case["dim"]}


def _branch_of(parents, t):
    """Tokens from t up to the first one of its branch."""
    found = [t]
    while 0 <= parents[found[-1]] < found[-1]:
        found.append(parents[found[-1]])
    return found


def _exact_append(case, s, lens, n_new, parents):
    res = {n: s[n].double() for n in ("k_pages", "v_pages")}
    n = case["rotary"]

    def turned(x, pos):                     # the pairs as complex numbers, x [T, H, D]
        z = x.double()
        pairs = z[..., :n].unflatten(-1, (n // 2, 2)) if case["interleaved"] else z[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2)
        angle = pos.double()[:, None] * s["freqs"]
        w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle).unsqueeze(-2))
        w = w.flatten(-2) if case["interleaved"] else w.transpose(-1, -2).flatten(-2)
        return torch.cat((w, z[..., n:]), dim=-1)

    q = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b in range(case["batch"]):
        m, first = n_new[b], lens[b] - n_new[b]
        depth = [len(_branch_of(parents[b], t)) - 1 for t in range(m)] if parents is not None else range(m)
        pos = first + torch.tensor(list(depth), device=DEVICE)
        row = first + torch.arange(m, device=DEVICE)
        at = s["table"][b].long()[row // case["page"]], row % case["page"]
        q[b, :m] = turned(s["q"][b, :m], pos)
        res["k_pages"][at] = turned(s["k"][b, :m], pos)
        res["v_pages"][at] = s["v"][b, :m].double()
    return {"q": q, **res}


def _exact_decode(case, s, lens, n_new, parents):
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    lse = torch.full((case["batch"], case["heads"], case["tokens"]), -math.inf, dtype=torch.float64, device=DEVICE)
    for b in range(case["batch"]):
        m, first = n_new[b], lens[b] - n_new[b]
        see = np.zeros((m, lens[b]), dtype=bool)
        for t in range(m):
            branch = _branch_of(parents[b], t) if parents is not None else list(range(t, -1, -1))
            pos = first + len(branch) - 1
            see[t, :first] = True
            see[t, [first + j for j in branch]] = True
            if case["left"] >= 0:
                far = np.arange(lens[b])
                far[[first + j for j in branch]] = [pos - i for i in range(len(branch))]
                see[t] &= (far >= pos - case["left"]) | (far < case["sinks"])
        see = torch.as_tensor(see, device=DEVICE)
        at = s["table"][b, :-(-lens[b] // case["page"])].long()
        k, v = (s[n][at].flatten(0, 1)[:lens[b]] for n in ("k_pages", "v_pages"))
        for h in range(case["kv_heads"]):
            mine = slice(h * group, (h + 1) * group)
            q = s["q"][b, :m, mine].double().transpose(0, 1)                  # [group, m, D]
            scores = (q @ k[:, h].double().T) / math.sqrt(case["dim"])
            scores = scores.masked_fill(~see, -math.inf)
            out[b, :m, mine] = (torch.softmax(scores, dim=-1) @ v[:, h].double()).transpose(0, 1)
            lse[b, mine, :m] = torch.logsumexp(scores, dim=-1)
    return {"out": out, "lse": lse}


def _exact_keep(case, s, lens, n_new):
    res = {}
    path, kept, table, page = s["path"].tolist(), s["n_kept"].tolist(), s["table"].tolist(), case["page"]
    for n in ("k_pages", "v_pages"):
        old, new = s[n].double(), s[n].double().clone()
        for b in range(case["batch"]):
            first = lens[b] - n_new[b]
            for i in range(kept[b]):
                source, to = first + path[b][i], first + i
                new[:, table[b][to // page], to % page] = old[:, table[b][source // page], source % page]
        res[n] = new
    return res


def exact(case, seed):
    s = prepare(case, seed)
    lens = s["lens"].tolist()
    n_new = s["n_new"].tolist() if s["n_new"] is not None else [case["tokens"]] * case["batch"]
    if case["kind"] == "keep":
        return _exact_keep(case, s, lens, n_new)
    parents = s["parents"].tolist() if s["parents"] is not None else None
    return (_exact_append if case["kind"] == "append" else _exact_decode)(case, s, lens, n_new, parents)
