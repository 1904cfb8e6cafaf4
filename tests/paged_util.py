"""Paged caches for tests: pools with their rows in any order, and what a chain's or a tree's tokens see of them, by the definition, in Python loops."""
import torch

from tests.swa_util import DEV


def pools(batch, rows, page, kv_heads, dim, dtype, seed=0, spare=2):
    """(k_pages, v_pages, table) with random contents in all rows and pages in random order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    most = -(-rows // page)
    make = lambda: torch.randn(batch * most + spare, page, kv_heads, dim, generator=g, device=DEV).to(dtype)  # noqa: E731
    k, v = make(), make()
    table = torch.randperm(batch * most + spare, generator=g, device=DEV)[:batch * most].reshape(batch, most).to(torch.int32)
    return k, v, table


def rows_of(pages, table):
    """[B, rows, H, D] of the table's rows (of pages that are not there: of page 0)."""
    at = table.long()
    at = torch.where((at >= 0) & (at < pages.shape[0]), at, torch.zeros_like(at))
    return pages[at].flatten(1, 2)


def branch(parents, t):
    found = [t]
    while 0 <= parents[found[-1]] < found[-1]:
        found.append(parents[found[-1]])
    return found


def trees(batch, tokens, seed=0, bushy=1.0):
    """int32 [B, T]: the token before each, -1 for first ones; bushy near 0: long chains."""
    g = torch.Generator().manual_seed(seed)
    t = torch.arange(tokens)
    back = (torch.rand(batch, tokens, generator=g) * (t * bushy + 1)).floor()
    return (t - 1 - back).clamp_min(-1).to(torch.int32).to(DEV)


def visible(lens, n_new, parents, tokens, table, page, n_pages, window=-1, sinks=0):
    """[B, 1, T, rows]: which rows of the table a token sees."""
    rows = table.shape[1] * page
    seen = torch.zeros(len(lens), 1, tokens, rows, dtype=torch.bool)
    entries = table.tolist()
    lens = [min(max(n, 0), 2 ** 29) for n in lens]
    for b, n in enumerate(lens):
        real = min(max(n_new[b], 0), tokens) if n_new is not None else tokens
        base = n - real
        tree = None if parents is None else (parents[b] if isinstance(parents[0], list) else parents)
        there = torch.tensor([0 <= e < n_pages for e in entries[b]], dtype=torch.bool).repeat_interleave(page)
        for t in range(real):
            mine = branch(tree, t) if tree is not None else list(range(t, -1, -1))
            pos = base + len(mine) - 1
            # position of every row that is on the way: the cache's and the branch's
            where = {r: r for r in range(0, min(max(base, 0), rows))} if window >= 0 else None
            if where is None:
                seen[b, 0, t, :min(max(base, 0), rows)] = True
                for j in mine:
                    if 0 <= base + j < rows:
                        seen[b, 0, t, base + j] = True
            else:
                where.update({base + j: pos - i for i, j in enumerate(mine)})
                for r, at in where.items():
                    if 0 <= r < rows and (at >= pos - window or at < sinks):
                        seen[b, 0, t, r] = True
            seen[b, 0, t] &= there
    return seen.to(DEV)
