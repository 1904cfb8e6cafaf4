"""Trees deeper than the window, of up to 32 rows of a key head and of more, in launches that fill the device and beside each other, against the definition in 64 bits
(bounds: swa_util) and, call for call, the same bits."""
import pytest
import torch

import ultraattn_amd as ua
from tests.paged_util import pools, rows_of, trees, visible
from tests.swa_util import DEV, Reference, inputs

pytestmark = pytest.mark.gpu


def made(batch, tokens, heads, kv_heads, dim, dtype, rows, bushy, seed):
    """Lengths of which the new tokens lie before, across and behind blocks of 32 and 64 keys; some sequences shorter than their tree."""
    kp, vp, table = pools(batch, rows, 16, kv_heads, dim, dtype, seed)
    lens = (torch.arange(batch, device=DEV) * 37 % (rows - tokens) + tokens).to(torch.int32)
    lens[1], lens[2], lens[3] = tokens, tokens // 2, rows
    return inputs(batch, tokens, 1, heads, 1, dim, dtype, seed)[0], kp, vp, table, lens, None, trees(batch, tokens, seed, bushy)


def check(args, window, sinks, out, lse):
    q, kp, vp, table, lens, _, parents = args
    seen = visible(lens.tolist(), None, parents.tolist(), q.shape[1], table, kp.shape[1], kp.shape[0], window, sinks)
    Reference(q, rows_of(kp, table), rows_of(vp, table), seen).check(out=out, lse=lse)


@pytest.mark.parametrize("window", [0, 1, 3, 7])
@pytest.mark.parametrize("sinks", [0, 70])
@pytest.mark.parametrize("batch,tokens,heads,kv_heads,dim,dtype,bushy", [(64, 9, 9, 3, 64, torch.bfloat16, 0.02), (70, 32, 8, 8, 128, torch.bfloat16, 0.05), (40, 16, 8, 8, 64, torch.float16, 0.2),
                                                                        (5, 32, 2, 2, 64, torch.float16, 0.0), (40, 20, 16, 8, 128, torch.bfloat16, 0.05), (20, 64, 4, 4, 64, torch.float16, 0.05),
                                                                        (9, 150, 4, 2, 64, torch.bfloat16, 0.01)])
def test_trees_deeper_than_the_window(window, sinks, batch, tokens, heads, kv_heads, dim, dtype, bushy):
    args = made(batch, tokens, heads, kv_heads, dim, dtype, 330, bushy, tokens)
    out, lse = ua.paged_decode(*args, window, sinks)
    check(args, window, sinks, out, lse)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    again = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                again.append(ua.paged_decode(*args, window, sinks))
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) and torch.equal(l, lse) for o, l in again)


def test_window_that_cuts_nothing():
    """As many steps as the deepest branch has: the same bits as with one more, which no branch reaches."""
    for tokens in (9, 32, 64, 100):
        args = made(5, tokens, 4, 4, 64, torch.bfloat16, 330, 0.0, 3)
        args = (*args[:4], torch.full_like(args[4], tokens), *args[5:])
        a, b = ua.paged_decode(*args, tokens - 1, 0), ua.paged_decode(*args, tokens + 7, 0)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
