"""Rows of accepted branches moved together in a paged cache: exactly those, exactly as they were."""
import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def moved(pages, table, lens, n_new, path, kept):
    """Of [layers, n_pages, page, H, D] on the host: as if everything were read first."""
    old, new, page, room = pages.clone(), pages.clone(), pages.shape[2], table.shape[1] * pages.shape[2]
    there = lambda b, r: 0 <= r < room and 0 <= int(table[b, r // page]) < pages.shape[1]  # noqa: E731
    for b in range(len(lens)):
        n = max(n_new[b], 0)
        base = max(lens[b], 0) - n
        for i in range(min(max(kept[b], 0), len(path[b]), n)):
            source, to = base + path[b][i], base + i
            if i < path[b][i] < n and there(b, to) and there(b, source):
                new[:, int(table[b, to // page]), to % page] = old[:, int(table[b, source // page]), source % page]
    return new


def run(kp, vp, table, lens, n_new, path, kept):
    five = lambda x: x if x.dim() == 5 else x[None]  # noqa: E731
    many = n_new.tolist() if isinstance(n_new, torch.Tensor) else [n_new] * len(lens)
    want = [moved(five(x).cpu(), table.cpu(), lens.tolist(), many, path.tolist(), kept.tolist()) for x in (kp, vp)]
    assert ua.paged_keep(kp, vp, table, lens, n_new, path, kept) is None
    assert torch.equal(five(kp).cpu(), want[0]) and torch.equal(five(vp).cpu(), want[1])


def made(layers, batch, tokens, m, page, rows, kv_heads, dim, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    most = -(-rows // page)
    shape = (*([layers] if layers else []), batch * most + 2, page, kv_heads, dim)
    kp, vp = (torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2))
    table = torch.randperm(batch * most + 2, generator=g, device=DEV)[:batch * most].reshape(batch, most).to(torch.int32)
    path = torch.rand(batch, tokens, generator=g, device=DEV).argsort(1)[:, :m].sort(1).values.to(torch.int32)
    kept = torch.randint(0, m + 1, (batch,), generator=g, device=DEV).to(torch.int32)
    lens = torch.randint(tokens, rows + 1, (batch,), generator=g, device=DEV).to(torch.int32)
    return kp, vp, table, lens, path, kept


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("layers,batch,tokens,m,page,kv_heads,dim", [(None, 1, 2, 1, 16, 2, 128), (3, 5, 26, 6, 7, 2, 64), (2, 4, 64, 20, 16, 8, 128), (None, 3, 40, 40, 1, 3, 20),
                                                                     (1, 2, 700, 600, 64, 2, 64), (5, 9, 9, 9, 32, 1, 7)])
def test_branches(dtype, layers, batch, tokens, m, page, kv_heads, dim):
    kp, vp, table, lens, path, kept = made(layers, batch, tokens, m, page, tokens + 50, kv_heads, dim, dtype)
    run(kp, vp, table, lens, tokens, path, kept)
    run(kp, vp, table, lens, torch.full_like(lens, tokens), path, torch.full_like(kept, m))


def test_ragged_and_what_is_not_moved():
    kp, vp, table, _, path, _ = made(2, 8, 20, 8, 16, 100, 2, 64, torch.bfloat16)
    table[3, 2], table[4, 1], table[5] = -1, kp.shape[1], -(2 ** 31)
    lens = ints([100, 15, 5, 45, 40, 60, 0, -4])
    path[6:] = ints([[1, 2, 3, 4, 5, 6, 7, 8]])
    path[0] = ints([0, 1, 2, 9, 25, -3, 2 ** 31 - 1, 3])            # where they are already, no real token, below their place
    run(kp, vp, table, lens, ints([20, 12, 20, 20, 20, 20, 20, 2]), path, ints([8, 3, 8, 8, 8, 8, 8, 8]))
    run(kp, vp, table, lens, ints([0, -1, 2 ** 31 - 1, 7, 20, 20, 20, 20]), path, ints([8, 3, 2 ** 31 - 1, -8, 0, 8, 8, 8]))
    past = ints([130, 120, 101, 100, 100, 2 ** 31 - 1, 113, 99])   # lengths behind the table
    run(kp, vp, table, past, 20, path, torch.full_like(lens, 8))


def test_layouts_and_nothing_to_do():
    both = torch.randn(4, 30, 2, 3, 16, 64, device=DEV).to(torch.float16)               # [layers, pages, 2, H, page, D]
    kp, vp = both[:, :, 0].transpose(2, 3), both[:, :, 1].transpose(2, 3)
    table = torch.randperm(30, device=DEV).to(torch.int32).reshape(3, 10)
    lens, path, kept = ints([160, 20, 77]), ints([[0, 5, 6, 19], [1, 2, 3, 4], [3, 7, 8, 9]]), ints([4, 3, 4])
    run(kp, vp, table, lens, 20, path, kept)
    wide = torch.zeros(3, 9, dtype=torch.int32, device=DEV)
    wide[:, 2:6] = path
    run(kp, vp, table, lens, 20, wide[:, 2:6], kept)
    flat = torch.randn(2, 40 * 64 + 1, device=DEV).to(torch.float16)
    odd = [x[1:].view(5, 4, 2, 64) for x in flat]                                      # on no vector's boundary
    run(odd[0], odd[1], ints([[4, 0]]), ints([8]), 6, ints([[2, 5]]), ints([2]))
    before = both.clone()
    ua.paged_keep(kp, vp, table, lens, 20, path[:, :0], kept)
    ua.paged_keep(kp, vp, table, lens, 0, path, kept)
    ua.paged_keep(kp, vp, table[:0], lens[:0], 20, path[:0], kept[:0])
    ua.paged_keep(kp, vp, table[:, :0], lens, 20, path, kept)
    ua.paged_keep(kp[:, :0], vp[:, :0], table, lens, 20, path, kept)
    assert torch.equal(both, before)


def test_rows_beyond_two_gigabytes():
    kp = torch.zeros(70_000, 16, 16, 128, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    kp[69_999, 5], vp[69_999, 5] = 1.0, 2.0
    ua.paged_keep(kp, vp, ints([[69_998, 69_999]]), ints([24]), 20, ints([[17]]), ints([1]))         # row 4 takes row 21
    assert (kp[69_998, 4] == 1).all() and (vp[69_998, 4] == 2).all() and int(kp.count_nonzero()) == 2 * 16 * 128


def test_refusals():
    kp, vp, table, lens, path, kept = made(2, 2, 9, 3, 16, 60, 2, 64, torch.bfloat16)
    f = ua.paged_keep
    bad = [lambda: f(kp, vp[:1], table, lens, 9, path, kept), lambda: f(kp, kp, table, lens, 9, path, kept), lambda: f(kp, vp.half(), table, lens, 9, path, kept),
           lambda: f(kp[0, 0], vp[0, 0], table, lens, 9, path, kept), lambda: f(kp, vp, table.long(), lens, 9, path, kept), lambda: f(kp, vp, table[:1], lens, 9, path, kept),
           lambda: f(kp, vp, table, lens, None, path, kept), lambda: f(kp, vp, table, lens, -1, path, kept), lambda: f(kp, vp, table, lens, lens[:1], path, kept),
           lambda: f(kp, vp, table, lens, 9, path.long(), kept), lambda: f(kp, vp, table, lens, 9, path[:1], kept), lambda: f(kp, vp, table, lens, 9, path[0], kept),
           lambda: f(kp, vp, table, lens, 9, path, kept.long()), lambda: f(kp, vp, table, lens, 9, path, kept[:1]), lambda: f(kp, vp, table, lens.float(), 9, path, kept),
           lambda: f(kp[:1].expand(2, *kp.shape[1:]), vp, table, lens, 9, path, kept), lambda: f(kp.int(), vp.int(), table, lens, 9, path, kept),
           lambda: f(kp.cpu(), vp.cpu(), table, lens, 9, path, kept), lambda: f(kp, vp, table, lens[0], 9, path, kept)]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
