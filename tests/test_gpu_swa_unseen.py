"""NaN and infinity in keys, values and query rows that a tile of 128 rows (in a decode the rows of a key head) does not see: nothing of them
reaches the tile, whatever blocks of 64 (32) keys its walk is made of."""
import math

import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, Reference, inputs, visible

pytestmark = pytest.mark.gpu
KINDS = [(torch.bfloat16, 128), (torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 64)]


def poison(x, hidden):
    """x [B, S, H, D] with NaN and infinities in the rows `hidden` [S]."""
    bad = torch.tensor([math.nan, math.inf, -math.inf], device=DEV, dtype=x.dtype)
    fill = bad[torch.arange(x[:, hidden].numel(), device=DEV) % 3].view(x[:, hidden].shape)
    y = x.clone()
    y[:, hidden] = fill
    return y


# windows whose ends lie inside blocks: of one tile, of several, behind sinks that end inside a block, between them, beyond the keys
PLACES = [(300, 700, (60, 0), 0, 250), (300, 700, (60, 0), 5, 250), (40, 500, (33, 0), 70, 217), (1, 300, (20, 0), 2, 150), (130, 900, (100, 37), 3, 333),
          (128, 2000, (10, 0), 4, 1000), (300, 200, (10, 0), 0, 100), (300, 200, (10, 0), 3, -50), (200, 300, (0, 0), 0, 77)]


@pytest.mark.parametrize("dtype,dim", KINDS)
@pytest.mark.parametrize("seq_q,seq_k,window,sinks,start", PLACES)
def test_keys_and_rows_that_nothing_sees(dtype, dim, seq_q, seq_k, window, sinks, start):
    q, k, v, do = inputs(2, seq_q, seq_k, 4, 2, dim, dtype, 3)
    seen = visible(seq_q, seq_k, window, sinks, start)
    keys, rows = ~seen.any(0), ~seen.any(1)
    assert keys.any() or rows.any()
    ref = Reference(q, k, v, seen, dout=do)
    qb, kb, vb, dob = poison(q, rows), poison(k, keys), poison(v, keys), poison(do, rows)
    how = dict(window=window, sinks=sinks, q_start=start)
    out, lse = ua.swa_fwd(qb, kb, vb, **how)
    ref.check(out=out, lse=lse)
    dq, dk, dv = ua.swa_bwd(dob, qb, kb, vb, out, lse, **how)
    ref.check(dq=dq, dk=dk, dv=dv)
    assert not dk[:, keys].any() and not dv[:, keys].any() and not dq[:, rows].any()


@pytest.mark.parametrize("dtype,dim", KINDS)
@pytest.mark.parametrize("sinks", [0, 5])
def test_keys_that_another_tile_sees(dtype, dim, sinks):
    """Rows 128 .. 255 see the keys 380 and 400; the first tile's walk ends at 377, the last one's begins at 446, in the block of 384."""
    q, k, v, _ = inputs(1, 300, 700, 2, 2, dim, dtype)
    how = dict(window=(60, 0), sinks=sinks, q_start=250)
    ref = Reference(q, k, v, visible(300, 700, (60, 0), sinks, 250))
    kb, vb = k.clone(), v.clone()
    kb[:, [380, 400]] = math.nan
    vb[:, [380, 400]] = math.inf
    out, lse = ua.swa_fwd(q, kb, vb, **how)
    for rows in (slice(0, 128), slice(256, 300)):
        err = (out[:, rows].double() - ref.out[:, rows]).abs()
        assert (err <= ref.out_bound[:, rows]).all() and ((lse[..., rows] - ref.lse[..., rows]).abs() <= ref.lse_bound[..., rows]).all()
    assert torch.isnan(lse[..., 150:191]).all()                       # rows that see the keys say so


@pytest.mark.parametrize("dtype,dim", KINDS)
@pytest.mark.parametrize("tokens,heads", [(1, 8), (3, 14), (9, 12)])
@pytest.mark.parametrize("window,sinks", [(100, 0), (77, 5), (0, 1), (200, 40), (-1, 0)])
def test_rows_of_a_cache_that_no_token_sees(dtype, dim, tokens, heads, window, sinks):
    """Rows that left the window, and rows behind the length."""
    room = 700
    q, kc, vc, _ = inputs(3, tokens, room, heads, 2, dim, dtype, tokens)
    lens = torch.tensor([431, 90, 700], dtype=torch.int32, device=DEV)
    pos = (lens.long()[:, None] - tokens + torch.arange(tokens, device=DEV))[:, :, None]
    key = torch.arange(room, device=DEV)
    seen = key <= pos
    if window >= 0:
        seen &= (key >= pos - window) | (key < sinks)
    ref = Reference(q, kc, vc, seen[:, None])
    kb, vb = kc.clone(), vc.clone()
    for b in range(3):
        hidden = ~seen[b].any(0)
        kb[b:b + 1], vb[b:b + 1] = poison(kc[b:b + 1], hidden), poison(vc[b:b + 1], hidden)
    out, lse = ua.swa_decode(q, kb, vb, lens, window, sinks)
    ref.check(out=out, lse=lse)
