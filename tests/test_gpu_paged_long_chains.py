"""Chunks of prompts against a paged cache, tables much wider than the sequences, and references that rise several times in a walk, against the definition in 64 bits
(bounds: swa_util)."""
import pytest
import torch

import ultraattn_amd as ua
from tests.paged_util import pools, rows_of, trees, visible
from tests.swa_util import DEV, Reference, inputs

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def chain(lens, n_new, tokens, rows, window=-1, sinks=0):
    """[B, 1, T, rows] of a chain, all pages there."""
    base = (lens - n_new).long()[:, None, None]
    t, r = torch.arange(tokens, device=DEV)[None, :, None], torch.arange(rows, device=DEV)[None, None]
    seen = (r <= base + t) & (t < n_new[:, None, None])
    if window >= 0:
        seen &= (r >= base + t - window) | (r < sinks)
    return seen[:, None]


@pytest.mark.parametrize("dtype,dim,heads,kv_heads", [(torch.bfloat16, 128, 8, 2), (torch.float16, 64, 6, 2), (torch.bfloat16, 64, 1, 1), (torch.float16, 128, 3, 3)])
@pytest.mark.parametrize("tokens,rows", [(1000, 1000), (1111, 2500), (2048, 2100)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (299, 5), (1500, 130)])
def test_chunks_of_prompts(dtype, dim, heads, kv_heads, tokens, rows, window, sinks):
    kp, vp, table = pools(2, rows, 24, kv_heads, dim, dtype, tokens)
    q = inputs(2, tokens, 1, heads, 1, dim, dtype, tokens)[0]
    for lens, n_new in ((ints([rows, tokens]), None), (ints([rows - 7, tokens - 300]), ints([tokens - 1, tokens - 300]))):
        out, lse = ua.paged_decode(q, kp, vp, table, lens, n_new, None, window, sinks)
        real = n_new if n_new is not None else torch.full_like(lens, tokens)
        seen = chain(lens, real, tokens, table.shape[1] * 24, window, sinks)
        for b in range(2):
            Reference(q[b:b + 1], rows_of(kp, table[b:b + 1]), rows_of(vp, table[b:b + 1]), seen[b:b + 1]).check(out=out[b:b + 1], lse=lse[b:b + 1])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 8, 2), (5, 14, 2), (26, 8, 2), (120, 8, 8)])
@pytest.mark.parametrize("width", [8192, 131072])
def test_tables_wider_than_the_sequences(dtype, dim, tokens, heads, kv_heads, width):
    """As a server keeps them, as wide as the longest sequence allowed: the parts are made for that, most walks are shorter than them."""
    lens = ints([1500, 130, tokens, 777])
    kp, vp, narrow = pools(4, 1504, 16, kv_heads, dim, dtype, tokens)
    table = torch.full((4, width // 16), -1, dtype=torch.int32, device=DEV)
    table[:, :narrow.shape[1]] = narrow
    q = inputs(4, tokens, 1, heads, 1, dim, dtype, 3)[0]
    for parents in (None, trees(4, tokens, 2, 0.3)):
        out, lse = ua.paged_decode(q, kp, vp, table, lens, None, parents)
        seen = visible(lens.tolist(), None, parents.tolist() if parents is not None else None, tokens, narrow, 16, kp.shape[0])
        Reference(q, rows_of(kp, narrow), rows_of(vp, narrow), seen).check(out=out, lse=lse)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(2, 4, 2), (8, 8, 2), (32, 2, 2), (40, 4, 2), (70, 8, 4)])
def test_references_that_rise_in_a_walk(dtype, dim, tokens, heads, kv_heads):
    """Small keys, among them, at rising places and of rising size, copies of queries that share the key head: of every third token, of each query head in turn."""
    rows, group = 900, heads // kv_heads
    kp, vp, table = pools(2, rows, 16, kv_heads, dim, dtype, tokens)
    q = inputs(2, tokens, 1, heads, 1, dim, dtype, 5)[0] * 3
    kp *= 0.1
    chosen = list(range(0, tokens, 3))
    for n, t in enumerate(chosen):
        for again in range(3):                                     # three times in the walk, larger each time
            r = 20 + 290 * again + 7 * n
            at = table.long()[:, r // 16], r % 16
            kp[at] = (q[:, t].unflatten(1, (kv_heads, group))[:, :, (n + again) % group] * (0.1 + 0.2 * again)).to(dtype)
    for lens in (ints([900, 640]), ints([880, tokens])):
        out, lse = ua.paged_decode(q, kp, vp, table, lens)
        seen = chain(lens, torch.full_like(lens, tokens), tokens, table.shape[1] * 16)
        Reference(q, rows_of(kp, table), rows_of(vp, table), seen).check(out=out, lse=lse)
