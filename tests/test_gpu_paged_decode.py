"""New tokens, chains and trees, against a paged cache, against the definition in 64 bits (bounds: swa_util)."""
import math

import pytest
import torch

import ultraattn_amd as ua
from tests.paged_util import pools, rows_of, trees, visible
from tests.swa_util import DEV, Reference, inputs

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def check(q, kp, vp, table, lens, n_new, parents, window, sinks, out, lse, scale=None):
    seen = visible(lens.tolist(), n_new.tolist() if n_new is not None else None, parents.tolist() if parents is not None else None, q.shape[1], table,
                   kp.shape[1], kp.shape[0], window, sinks)
    Reference(q, rows_of(kp, table), rows_of(vp, table), seen, scale).check(out=out, lse=lse)


def run(q, kp, vp, table, lens, n_new=None, parents=None, window=-1, sinks=0, scale=None):
    out, lse = ua.paged_decode(q, kp, vp, table, lens, n_new, parents, window, sinks, scale)
    check(q, kp, vp, table, lens, n_new, parents, window, sinks, out, lse, scale)
    return out, lse


def queries(batch, tokens, heads, dim, dtype, seed=0):
    return inputs(batch, tokens, 1, heads, 1, dim, dtype, seed)[0]


def spread(batch, least, most, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(least, most + 1, (batch,), generator=g)
    x[:3] = torch.tensor([least, most, (least + most) // 2])[:batch]
    return ints(x.tolist())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 8, 2), (3, 7, 1), (5, 14, 2), (40, 8, 2), (130, 3, 3)])
@pytest.mark.parametrize("page,rows,window,sinks", [(16, 16, -1, 0), (1, 33, -1, 0), (7, 500, -1, 0), (16, 500, 100, 5), (32, 900, 0, 0), (64, 900, 31, 70), (300, 300, -1, 0)])
def test_chains(dtype, dim, tokens, heads, kv_heads, page, rows, window, sinks):
    kp, vp, table = pools(4, rows, page, kv_heads, dim, dtype, rows + tokens)
    run(queries(4, tokens, heads, dim, dtype), kp, vp, table, spread(4, 0, rows), None, None, window, sinks)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 4, 1), (2, 8, 2), (9, 3, 3), (16, 14, 2), (32, 4, 4), (33, 1, 1), (64, 8, 2), (65, 4, 2), (256, 2, 1)])
@pytest.mark.parametrize("page,rows,window,sinks,bushy", [(16, 300, -1, 0, 1.0), (24, 700, 3, 2, 0.05), (128, 700, 40, 0, 1.0), (5, 260, 0, 261, 0.3)])
def test_trees(dtype, dim, tokens, heads, kv_heads, page, rows, window, sinks, bushy):
    kp, vp, table = pools(3, rows, page, kv_heads, dim, dtype, rows + tokens)
    run(queries(3, tokens, heads, dim, dtype), kp, vp, table, spread(3, tokens, rows), None, trees(3, tokens, tokens, bushy), window, sinks)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(6, 4, 2), (24, 8, 2), (70, 4, 2)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("window", [-1, 9])
def test_ragged_steps(tokens, heads, kv_heads, tree, window):
    """Steps of fewer tokens, of none, of more than there are; sequences shorter than their step, longer than their table, empty."""
    lens = ints([200, 37, 0, 5, tokens, 250, 100, -7, 2 ** 31 - 1])
    n_new = ints([tokens, 3, 0, tokens, tokens, tokens + 9, -4, 2, 2])
    kp, vp, table = pools(9, 240, 16, kv_heads, 64, torch.float16)
    q = queries(9, tokens, heads, 64, torch.float16)
    q[1, 3:] = torch.nan                                       # padding may hold anything
    out, lse = ua.paged_decode(q, kp, vp, table, lens, n_new, trees(9, tokens) if tree else None, window, 2)
    assert (out[1, 3:] == 0).all() and (lse[1, :, 3:] == -math.inf).all() and (out[2] == 0).all() and (lse[2] == -math.inf).all()
    check(torch.nan_to_num(q), kp, vp, table, lens, n_new, trees(9, tokens) if tree else None, window, 2, out, lse)


@pytest.mark.parametrize("tokens", [1, 5, 60])
def test_pages_that_are_not_there(tokens):
    kp, vp, table = pools(4, 400, 16, 2, 128, torch.bfloat16)
    q = queries(4, tokens, 4, 128, torch.bfloat16)
    lens = ints([400, 333, 400, 61])
    table[0, 3] = -1
    table[0, 7:9] = kp.shape[0]
    table[1, ::2] = 2 ** 31 - 1
    table[2] = -(2 ** 31)
    table[3, 4:] = -1
    for parents in (None, trees(4, tokens)):
        for window in (-1, 50):
            out, lse = run(q, kp, vp, table, lens, None, parents, window, 3)
            assert (out[2] == 0).all() and (lse[2] == -math.inf).all()


def test_parents_that_are_none():
    """Values outside 0 .. t - 1 say that a token follows the cache; nothing loops."""
    tokens = 40
    parents = trees(2, tokens).clone()
    parents[0, 5], parents[0, 6], parents[0, 7], parents[0, 8], parents[1, 0], parents[1, 39] = 5, 7, 39, 2 ** 31 - 1, 3, -(2 ** 31)
    kp, vp, table = pools(2, 150, 16, 2, 64, torch.bfloat16)
    for heads in (2, 8):
        run(queries(2, tokens, heads, 64, torch.bfloat16), kp, vp, table, ints([150, 60]), None, parents, 10, 1)


def test_one_tree_for_all_and_chains_as_trees():
    kp, vp, table = pools(3, 200, 16, 2, 64, torch.bfloat16)
    q = queries(3, 20, 4, 64, torch.bfloat16)
    lens = ints([200, 20, 99])
    one = trees(1, 20)[0]
    a = run(q, kp, vp, table, lens, None, one, 30, 2)
    b = run(q, kp, vp, table, lens, None, one.expand(3, 20).contiguous(), 30, 2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    chain = torch.arange(-1, 19, dtype=torch.int32, device=DEV)
    a, b = run(q, kp, vp, table, lens, None, chain, 30, 2), run(q, kp, vp, table, lens, None, None, 30, 2)
    assert (a[1] - b[1]).abs().max() < 1e-4


@pytest.mark.parametrize("tokens", [2, 50])
def test_nothing_that_no_token_sees_is_used(tokens):
    """NaN behind the lengths, in pages of nobody, before the windows, and in rows of pages that are not the sequence's."""
    kp, vp, table = pools(4, 300, 16, 2, 128, torch.bfloat16, spare=3)
    q = queries(4, tokens, 8, 128, torch.bfloat16)
    lens, window, sinks = ints([300, tokens, 133, 160]), 70, 3
    for parents in (None, trees(4, tokens, bushy=0.2)):
        want = run(q, kp, vp, table, lens, None, parents, window, sinks)
        seen = visible(lens.tolist(), None, parents.tolist() if parents is not None else None, tokens, table, 16, kp.shape[0], window, sinks).any(dim=2)[:, 0]
        k2, v2 = torch.full_like(kp, torch.nan), torch.full_like(vp, torch.inf)
        for b in range(4):
            for r in seen[b].nonzero()[:, 0].tolist():
                at = int(table[b, r // 16]), r % 16
                k2[at], v2[at] = kp[at], vp[at]
        t2 = table.clone()
        for b in range(4):
            t2[b, -(-int(lens[b]) // 16):] = 2 ** 30
        got = ua.paged_decode(q, k2, v2, t2, lens, None, parents, window, sinks)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_layouts_and_given_results():
    q = queries(3, 2, 12, 64, torch.bfloat16)
    lens = ints([64, 3, 40])
    both = torch.randn(20, 2, 4, 16, 64, device=DEV).to(torch.bfloat16)                # [pages, 2, H, page, D]
    kp, vp = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    table = torch.randperm(20, device=DEV).to(torch.int32)[:12].reshape(3, 4)
    out, lse = run(q[:, :, :8], kp, vp, table, lens, None, None, 20, 1)
    room, stat = torch.full_like(q, 7.0), torch.empty_like(lse)
    got = ua.paged_decode(q[:, :, :8], kp, vp, table, lens, window=20, sinks=1, out=room[:, :, 2:10], lse=stat)
    assert got[1] is stat and torch.equal(room[:, :, 2:10], out) and torch.equal(stat, lse) and (room[:, :, :2] == 7).all() and (room[:, :, 10:] == 7).all()
    wide = torch.full((3, 9), -5, dtype=torch.int32, device=DEV)
    wide[:, 2:6] = table
    got = ua.paged_decode(q[:, :, :8], kp, vp, wide[:, 2:6], lens, window=20, sinks=1)
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)
    mine = q[:, :, :8].clone()
    assert torch.equal(ua.paged_decode(mine, kp, vp, table, lens, window=20, sinks=1, out=mine)[0], out)
    assert ua.paged_decode(q[:0, :, :8], kp, vp, table[:0], lens[:0])[0].shape == (0, 2, 8, 64)
    assert ua.paged_decode(q[:, :0, :8], kp, vp, table, lens)[1].shape == (3, 8, 0)
    for nothing in ((kp[:0], vp[:0], table), (kp, vp, table[:, :0])):
        out, lse = ua.paged_decode(q[:, :, :8], *nothing, lens)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_contiguous_caches_and_shared_pages():
    b, room = 3, 500
    q, kc, vc, _ = inputs(b, 2, room, 8, 2, 128, torch.bfloat16)
    lens = ints([500, 7, 260])
    own = torch.arange(b, dtype=torch.int32, device=DEV)[:, None]
    got = run(q, kc, vc, own, lens, None, None, 100, 4)
    want = ua.swa_decode(q, kc, vc, lens, 100, 4)
    assert (got[0].float() - want[0].float()).abs().max() < 2e-2 and (got[1] - want[1]).abs().max() < 1e-4
    kp, vp, table = pools(3, 320, 32, 2, 128, torch.bfloat16)
    table[1:, :4] = table[0, :4]                                # a common beginning
    run(q, kp, vp, table, ints([320, 200, 129]))


def test_long_caches_in_parts():
    for tokens, heads, parents in ((1, 4, None), (30, 8, trees(1, 30))):
        kp, vp, table = pools(1, 70016, 64, 1, 128, torch.bfloat16)
        out, lse = ua.paged_decode(queries(1, tokens, heads, 128, torch.bfloat16), kp, vp, table, ints([70000]), None, parents)
        check(queries(1, tokens, heads, 128, torch.bfloat16), kp, vp, table, ints([70000]), None, parents, -1, 0, out, lse)
    # tables made for long sequences, of which these are short: most parts are empty
    kp, vp, table = pools(2, 320, 16, 2, 64, torch.float16)
    long = torch.full((2, 8192), -1, dtype=torch.int32, device=DEV)
    long[:, :20] = table
    for tokens in (1, 40):
        q = queries(2, tokens, 4, 64, torch.float16)
        out, lse = ua.paged_decode(q, kp, vp, long, ints([320, 41]))
        check(q, kp, vp, table, ints([320, 41]), None, None, -1, 0, out, lse)


@pytest.mark.parametrize("batch", [40, 64, 70])
@pytest.mark.parametrize("tokens,heads,kv_heads,tree", [(1, 8, 8, False), (5, 12, 6, True), (20, 16, 8, True), (70, 8, 4, False)])
def test_large_launches_take_the_longest_first(batch, tokens, heads, kv_heads, tree):
    """More workgroups than CUs: sequences are ranked by length up to 64 of them; equal and empty ones among them."""
    kp, vp, table = pools(batch, 330, 16, kv_heads, 64, torch.bfloat16)
    lens = spread(batch, 0, 330, batch)
    lens[5:15] = 200
    n_new = torch.minimum(torch.full_like(lens, tokens), lens)
    run(queries(batch, tokens, heads, 64, torch.bfloat16), kp, vp, table, lens, n_new, trees(batch, tokens) if tree else None)


def test_pools_beyond_two_gigabytes():
    pages, page = 70_000, 16
    kp = torch.zeros(pages, page, 16, 128, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    assert kp.numel() > 2 ** 31
    for tokens in (1, 20):
        q, k, v, _ = inputs(1, tokens, 208, 32, 16, 128, torch.bfloat16)
        table = torch.arange(pages - 13, pages, dtype=torch.int32, device=DEV).flip(0)[None]
        for i in range(13):
            kp[pages - 1 - i], vp[pages - 1 - i] = k[0, 16 * i:16 * i + 16], v[0, 16 * i:16 * i + 16]
        run(q, kp, vp, table, ints([208]))
    rows = pages * page                                         # one page of all rows
    long_k, long_v = kp.view(1, rows, 16, 128), vp.view(1, rows, 16, 128)
    long_k[:, -208:], long_v[:, -208:] = k, v
    out, lse = ua.paged_decode(q, long_k, long_v, ints([[0]]), ints([rows]), window=207 - 19, sinks=0)
    seen = torch.ones(20, 208, dtype=torch.bool, device=DEV).tril(188) & ~torch.ones(20, 208, dtype=torch.bool, device=DEV).tril(-1)
    Reference(q, k, v, seen).check(out=out, lse=lse)


def test_two_calls_at_once_and_on_another_stream():
    args = []
    for s in (0, 1):
        kp, vp, table = pools(2, 5000, 16, 2, 128, torch.bfloat16, s)
        args.append((queries(2, 9 + 10 * s, 8, 128, torch.bfloat16), kp, vp, table, ints([5000, 4000]), None, trees(2, 9 + 10 * s)))
    want = [run(*a) for a in args]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ua.paged_decode(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g[0], want[i][0]) and torch.equal(g[1], want[i][1]) for g in got[i])


def test_large_scores():
    """Scores that raise the reference in the middle of a walk, and equal ones."""
    for dtype in TYPES:
        for tokens in (2, 40):
            kp, vp, table = pools(2, 600, 16, 2, 128, dtype)
            q = queries(2, tokens, 4, 128, dtype) * 3
            rows = torch.arange(600, device=DEV)
            for b in range(2):
                kp[table[b].long()] *= 0.2
            where = table.long()[:, 300 // 16], 300 % 16
            kp[where] = (q[:, 0, :2] * 0.5).to(dtype)
            run(q, kp, vp, table, ints([600, 450]))
            kp.zero_()
            run(q, kp, vp, table, ints([600, 450]))
            assert rows.numel() == 600


def test_refusals():
    kp, vp, table = pools(2, 64, 16, 2, 64, torch.bfloat16)
    q, lens, many = queries(2, 3, 4, 64, torch.bfloat16), ints([10, 20]), queries(2, 257, 4, 64, torch.bfloat16)
    f = ua.paged_decode
    bad = [lambda: f(q, kp, vp[:, :8], table, lens), lambda: f(q, kp, vp, table.long(), lens), lambda: f(q, kp, vp, table[:1], lens), lambda: f(q, kp, vp, table[0], lens),
           lambda: f(q, kp, vp, table.cpu(), lens), lambda: f(q, kp, vp, table.t().contiguous().t(), lens), lambda: f(q, kp, vp, table, lens.long()),
           lambda: f(q, kp, vp, table, lens[:1]), lambda: f(q, kp, vp, table, lens.cpu()), lambda: f(q, kp, vp, table, lens, lens[:1]),
           lambda: f(q, kp, vp, table, lens, lens.float()), lambda: f(q, kp, vp, table, lens, None, trees(2, 4)), lambda: f(q, kp, vp, table, lens, None, trees(3, 3)),
           lambda: f(q, kp, vp, table, lens, None, trees(2, 3).long()), lambda: f(q, kp, vp, table, lens, None, trees(2, 3).cpu()),
           lambda: f(many, kp, vp, table, lens, None, trees(2, 257)), lambda: f(q, kp, vp, table, lens, window=-2), lambda: f(q, kp, vp, table, lens, sinks=-1),
           lambda: f(q.float(), kp.float(), vp.float(), table, lens), lambda: f(q[:, :, :3], kp, vp, table, lens), lambda: f(q, kp.half(), vp, table, lens),
           lambda: f(q, kp, vp.half(), table, lens), lambda: f(q[..., :32], kp[..., :32], vp[..., :32], table, lens), lambda: f(q, kp[..., :32], vp[..., :32], table, lens),
           lambda: f(q, kp, vp, table, lens, softmax_scale=0.0), lambda: f(q, kp, vp, table, lens, out=q[:, :, :2]),
           lambda: f(kp[:2, :3].repeat_interleave(2, 2), kp, vp, table, lens, out=kp[:2, :3].expand(2, 3, 2, 64)), lambda: f(q, kp[:, :0], vp[:, :0], table, lens),
           lambda: f(q, kp[0], vp[0], table, lens), lambda: f(q, kp, vp, table, lens, lse=torch.empty(2, 4, 2, device=DEV)),
           lambda: f(kp[:2, :3], kp, vp, table, lens, out=vp[:2, :3])]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(RuntimeError):                          # (strides of no whole 16 bytes)
        f(q, torch.zeros(8, 16, 2, 68, dtype=torch.bfloat16, device=DEV)[..., :64], vp[:8], table, lens)
