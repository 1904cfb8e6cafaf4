"""New tokens' rows written to a paged cache with their rotary positions, against the definition.

Bounds: those of test_gpu_rope, and for fp16 2^-25 beside them: below 2^-14 fp16 holds multiples of 2^-24, so half a step is 2^-25 there, more than the 2^-11 of the
value that a rounding is elsewhere (3.46e-5 rounds to 581 * 2^-24, 2.76e-8 off, where 2^-11 of it and 2^-21 of its pair are 2.12e-8).
"""
import numpy as np
import pytest
import torch

import ultraattn_amd as ua
from tests.paged_util import branch, pools, trees
from tests.swa_util import DEV
from tests.test_gpu_rope import TYPES, rows, turn

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def expected(q, k, v, kp, vp, table, lens, n_new, parents, freqs, **how):
    """(q, its bound, K pool, its bound, V pool) in 64 bits; pools as they were where nothing is written."""
    b, t = q.shape[:2]
    page, n_pages, most = kp.shape[1], kp.shape[0], table.shape[1]
    pos = torch.zeros(b, t, dtype=torch.int64)
    to, real = [], np.zeros((b, t), dtype=bool)
    for i in range(b):
        n = min(max(n_new[i], 0), t) if n_new is not None else t
        base = min(max(int(lens[i]), 0), 2 ** 29) - n
        tree = parents[i] if parents is not None else None
        for j in range(t):
            pos[i, j] = base + (len(branch(tree, j)) - 1 if tree is not None else j)
            real[i, j] = j < n
            row = base + j
            if j < n and 0 <= row < most * page and 0 <= int(table[i, row // page]) < n_pages:
                to.append((i, j, int(table[i, row // page]), row % page))
    (yq, bq), (yk, bk) = turn(q, pos, freqs, **how), turn(k, pos, freqs, **how)
    if q.dtype == torch.float16:
        bq, bk = bq + 2.0 ** -25, bk + 2.0 ** -25
    yq[~real], bq[~real] = 0, 0
    ek, ev = kp.cpu().double().numpy(), vp.cpu().clone()
    eb = np.zeros_like(ek)
    for i, j, at, slot in to:
        ek[at, slot], eb[at, slot], ev[at, slot] = yk[i, j], bk[i, j], v[i, j].cpu()
    return yq, bq, ek, eb, ev


def within(got, want, bound):
    err = np.abs(got.cpu().double().numpy() - want)
    over = err > bound
    worst = [(float(want[i]), float(err[i]), float(bound[i])) for i in map(tuple, np.argwhere(over)[:5])]
    assert not worst, (int(over.sum()), worst)


def run(q, k, v, kp, vp, table, lens, freqs, n_new=None, parents=None, q_out=None, **how):
    lists = [x.tolist() if x is not None else None for x in (lens, n_new)]
    tree = None if parents is None else parents.expand(q.shape[0], q.shape[1]).tolist()
    yq, bq, ek, eb, ev = expected(q, k, v, kp, vp, table, lists[0], lists[1], tree, freqs, **how)
    out = ua.paged_append(q, k, v, kp, vp, table, lens, freqs, n_new, parents, q_out=q_out, **how)
    within(out, yq, bq)
    within(kp, ek, eb)                                         # (0 where nothing is written)
    same = torch.equal(vp.cpu(), ev)
    assert same
    return out


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("tokens,dim,rotary,page", [(1, 128, 128, 16), (5, 64, 48, 7), (23, 72, 20, 1), (70, 128, 64, 32), (256, 64, 64, 24)])
def test_rows(dtype, interleaved, tree, tokens, dim, rotary, page):
    kp, vp, table = pools(5, tokens + 60, page, 2, dim, dtype)
    q, k, v = rows(5, tokens, 4, dim, dtype), rows(5, tokens, 2, dim, dtype, 1), rows(5, tokens, 2, dim, dtype, 2)
    f = ua.rope_freqs(rotary, device=DEV)[0]
    n_new = ints([tokens, max(tokens // 2, 1), 0, tokens, 1])
    run(q, k, v, kp, vp, table, ints([tokens, tokens + 60, 9, tokens + 3, 44]), f, n_new, trees(5, tokens, bushy=0.4) if tree else None,
        interleaved=interleaved, scale=1.25)


@pytest.mark.parametrize("tree", [False, True])
def test_lengths_and_pages_that_do_not_fit(tree):
    kp, vp, table = pools(7, 64, 16, 2, 64, torch.bfloat16)
    q, k, v = rows(7, 9, 4, 64, torch.bfloat16), rows(7, 9, 2, 64, torch.bfloat16, 1), rows(7, 9, 2, 64, torch.bfloat16, 2)
    f = ua.rope_freqs(64, device=DEV)[0]
    table[1, 2], table[1, 3], table[6] = -1, kp.shape[0], -(2 ** 31)
    lens = ints([4, 64, 70, 2 ** 31 - 1, -3, 41, 30])
    before = kp.clone(), vp.clone()
    run(q, k, v, kp, vp, table, lens, f, None, trees(7, 9) if tree else None)
    assert not torch.equal(kp, before[0])
    run(q, k, v, kp, vp, table, lens, f, ints([9, 9, 12, 9, -2, 2 ** 31 - 1, 3]), trees(1, 9)[0] if tree else None)
    empty = kp[:0]
    out = ua.paged_append(q, k, v, empty, empty.clone(), table, lens, f)
    assert out.shape == q.shape and torch.isfinite(out).all()
    out = ua.paged_append(q, k, v, kp, vp, table[:, :0], lens, f)
    assert torch.isfinite(out).all()


def test_prompts_layouts_and_in_place():
    both = torch.randn(300, 2, 2, 16, 128, device=DEV).to(torch.float16)             # [pages, 2, H, page, D]
    kp, vp = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    table = torch.randperm(300, device=DEV).to(torch.int32).reshape(2, 150)
    qkv = rows(2, 2000, 8, 128, torch.float16)
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    f = ua.rope_freqs(96, device=DEV)[0]
    n_new = ints([2000, 1777])
    assert run(q, k, v, kp, vp, table, ints([2400, 1777]), f, n_new, q_out=q) is q
    assert (q[1, 1777:] == 0).all()
    one = rows(1, 1, 1, 4000, torch.float16).flatten()[1:1 + 40 * 64].view(2, 5, 4, 64)        # on no vector's boundary
    kp, vp, table = pools(2, 32, 16, 4, 64, torch.float16)
    run(one, one, one, kp, vp, table, ints([20, 6]), ua.rope_freqs(64, device=DEV)[0])


def test_pool_beyond_two_gigabytes():
    kp = torch.zeros(70_000, 16, 16, 128, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    table = ints([[69_999, 3]])
    q, k, v = rows(1, 3, 16, 128, torch.bfloat16), rows(1, 3, 16, 128, torch.bfloat16, 1), rows(1, 3, 16, 128, torch.bfloat16, 2)
    f = ua.rope_freqs(128, device=DEV)[0]
    ua.paged_append(q, k, v, kp, vp, table, ints([16]), f)
    assert torch.equal(vp[69_999, 13:], v[0]) and torch.equal(kp[69_999, 13:], ua.rope_fwd(q, k, f, start=13)[1][0])
    assert int(kp.count_nonzero()) <= k.numel() and int(vp.count_nonzero()) <= v.numel()


def test_agrees_with_the_contiguous_form():
    b, t, room = 3, 4, 50
    q, k, v = rows(b, t, 4, 64, torch.bfloat16), rows(b, t, 2, 64, torch.bfloat16, 1), rows(b, t, 2, 64, torch.bfloat16, 2)
    f, scale = ua.rope_freqs(64, scaling="yarn", factor=4.0, original_length=16, device=DEV)
    lens = ints([4, 50, 33])
    a, c = torch.zeros(2, b, room, 2, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, b, room, 2, 64, dtype=torch.bfloat16, device=DEV)
    one = ua.rope_append(q, k, v, a[0], a[1], lens, f, scale=scale)
    two = ua.paged_append(q, k, v, c[0], c[1], torch.arange(b, dtype=torch.int32, device=DEV)[:, None], lens, f, scale=scale)
    assert torch.equal(one, two) and torch.equal(a, c)


def test_refusals():
    kp, vp, table = pools(2, 64, 16, 2, 64, torch.bfloat16)
    q, k = rows(2, 3, 4, 64, torch.bfloat16), rows(2, 3, 2, 64, torch.bfloat16)
    lens, f = ints([10, 20]), ua.rope_freqs(64, device=DEV)[0]
    g = ua.paged_append
    bad = [lambda: g(q, k, k[:, :2], kp, vp, table, lens, f), lambda: g(q, k, k, kp, vp[:3], table, lens, f), lambda: g(q, k, k, kp, kp, table, lens, f),
           lambda: g(q, k, k, kp, kp[:, :, :, :], table, lens, f), lambda: g(q, k, k, kp[:1].expand(8, 16, 2, 64), vp[:8], table, lens, f),
           lambda: g(q, k, k, kp[..., :32], vp[..., :32], table, lens, f), lambda: g(q, k, k, kp.half(), vp.half(), table, lens, f),
           lambda: g(q, k, k, kp, vp, table.long(), lens, f), lambda: g(q, k, k, kp, vp, table[:1], lens, f), lambda: g(q, k, k, kp, vp, table, lens.long(), f),
           lambda: g(q, k, k, kp, vp, table, lens, f.float()), lambda: g(q, k, k, kp, vp, table, lens, f.cpu()), lambda: g(q, k, k, kp, vp, table, lens, f, lens[:1]),
           lambda: g(q, k, k, kp, vp, table, lens, f, None, trees(2, 4)), lambda: g(q, k, k, kp, vp, table, lens, f, scale=0.0),
           lambda: g(q, k, k, kp, vp, table, lens, f, q_out=q[:, :, :2]), lambda: g(q, k, k, kp, vp, table, lens, f, q_out=q.flip(1)[:, :, :1].expand(2, 3, 4, 64)),
           lambda: g(q, k, k, kp, vp, table, lens, ua.rope_freqs(128, device=DEV)[0]), lambda: g(q, k, k, kp[0], vp[0], table, lens, f),
           lambda: g(kp[:2, :3], kp[:2, :3], k, kp, vp, table, lens, f),
           lambda: g(rows(2, 257, 4, 64, torch.bfloat16), rows(2, 257, 2, 64, torch.bfloat16), rows(2, 257, 2, 64, torch.bfloat16), kp, vp, table, lens, f, None, trees(2, 257))]
    before = kp.clone()
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    assert torch.equal(kp, before)
