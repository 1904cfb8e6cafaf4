"""Results that share memory with an operand of another type are refused; results beside it in one allocation are not."""
import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, inputs

pytestmark = pytest.mark.gpu


def views(seq=16, heads=4, dim=64, extra=64):
    """One allocation as rows [1, seq, heads, dim] of bf16 with `extra` bytes behind them, and as bytes."""
    n = 2 * seq * heads * dim
    raw = torch.zeros(n + extra, dtype=torch.uint8, device=DEV)
    return raw, raw[:n].view(torch.bfloat16).view(1, seq, heads, dim)


def test_lse():
    seq, heads = 16, 4
    raw, x = views(extra=4 * seq * heads)
    stat = lambda at: raw[at:at + 4 * seq * heads].view(torch.float32).view(1, heads, seq)  # noqa: E731
    q, k, v, do = inputs(1, seq, seq, heads, heads, 64, torch.bfloat16)
    x.copy_(q)
    want = ua.swa_fwd(q, k, v)
    behind, inside = stat(x.numel() * 2), [stat(0), stat(x.numel() * 2 - 4)]
    got = ua.swa_fwd(x, k, v, lse=behind)
    assert torch.equal(got[0], want[0]) and torch.equal(behind, want[1])
    lens = torch.full((1,), seq, dtype=torch.int32, device=DEV)
    for l in inside:
        for args in ((x, k, v), (q, x, v), (q, k, x)):
            with pytest.raises(ValueError, match="overlap"):
                ua.swa_fwd(*args, lse=l)
            with pytest.raises(ValueError, match="overlap"):
                ua.swa_decode(*args, lens, lse=l)
        with pytest.raises(ValueError, match="overlap"):
            ua.swa_fwd(q, k, v, out=x, lse=l)
        with pytest.raises(ValueError, match="overlap"):
            ua.swa_decode(q, k, v, lens, out=x, lse=l)
        for name in ("dq", "dk", "dv"):
            l.copy_(want[1])
            with pytest.raises(ValueError, match="overlap"):
                ua.swa_bwd(do, q, k, v, want[0], l, **{name: x})
            with pytest.raises(ValueError, match="overlap"):
                ua.swa_bwd(do, q, k, v, None, want[1], softmax_d=l, **{name: x})
    # heads of which every second belongs to a result: its gaps are rows of 128 bytes, a statistic of 32 floats fits one
    wide = torch.zeros(1, 32, 2, 64, dtype=torch.bfloat16, device=DEV)
    q, k, v, _ = inputs(1, 32, 32, 1, 1, 64, torch.bfloat16)
    gap = wide[0, 3, 1].view(torch.float32).view(1, 1, 32)
    got = ua.swa_fwd(q, k, v, out=wide[:, :, :1], lse=gap)
    want = ua.swa_fwd(q, k, v)
    assert torch.equal(got[0], want[0]) and torch.equal(gap, want[1])
    with pytest.raises(ValueError, match="overlap"):
        ua.swa_fwd(q, k, v, out=wide[:, :, :1], lse=wide[0, 3, 0].view(torch.float32).view(1, 1, 32))


def test_lengths_positions_frequencies():
    raw, x = views()
    q, k, v, _ = inputs(1, 16, 16, 4, 4, 64, torch.bfloat16)
    freqs = raw[:8 * 32].view(torch.float64)
    positions = raw[-64 - 128:-64].view(torch.int64)
    lens = raw[1024:1028].view(torch.int32)
    real = ua.rope_freqs(64, device=DEV)[0]
    new = torch.ones(1, dtype=torch.int32, device=DEV)
    one = [t[:, :1].contiguous() for t in (q, k, v)]
    bad = [lambda: ua.rope_fwd(q, k, freqs, q_out=x), lambda: ua.rope_fwd(q, k, freqs, k_out=x), lambda: ua.rope_fwd(q, k, real, positions, q_out=x),
           lambda: ua.rope_fwd(x, k, real, positions, q_out=x), lambda: ua.rope_bwd(q, k, real, positions, dk_out=x),
           lambda: ua.rope_append(*one, x, v.clone(), lens, real), lambda: ua.rope_append(*one, k.clone(), x, lens, real),
           lambda: ua.rope_append(*one, x, v.clone(), new, freqs), lambda: ua.rope_append(*one, k, v, lens, real, q_out=x[:, 2:3]),
           lambda: ua.swa_decode(q, k, v, lens, out=x)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError, match="overlap"):
            call()
            pytest.fail(f"call {i} was taken")
