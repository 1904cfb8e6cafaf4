"""Results given to sliding windows and rotary positions: their operand's own memory or none of it; parts of one packed row are apart."""
import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV

pytestmark = pytest.mark.gpu


def rows(h, s=40, b=2, d=64):
    return torch.randn(b, s, h, d, device=DEV, dtype=torch.float32, generator=torch.Generator(device=DEV).manual_seed(h)).to(torch.bfloat16)


def test_shifted_and_restrided_results_are_refused():
    long, k = rows(4, 41), rows(4)
    q, shifted = long[:, :40], long[:, 1:]
    other = rows(4, 4)                                                  # 4 tokens x 4 heads: its transpose is a view of the same shape
    turned = other.transpose(1, 2)
    f, _ = ua.rope_freqs(64, device=DEV)
    lens = torch.tensor([40, 40], dtype=torch.int32, device=DEV)
    out, lse = ua.swa_fwd(q, k, k)
    calls = [lambda: ua.swa_fwd(q, k, k, out=shifted), lambda: ua.swa_fwd(k, q, k, out=shifted), lambda: ua.swa_fwd(other, other.clone(), other.clone(), out=turned),
             lambda: ua.swa_decode(q, k, k, lens, out=shifted), lambda: ua.rope_fwd(q, None, f, q_out=shifted), lambda: ua.rope_fwd(k, q, f, k_out=shifted),
             lambda: ua.rope_fwd(q, k, f, k_out=shifted), lambda: ua.rope_fwd(other, None, f, q_out=turned),
             lambda: ua.swa_bwd(k, k, k, q, out, lse, dv=shifted), lambda: ua.swa_bwd(k, k, k, k, out, lse, dk=q, dv=shifted),
             lambda: ua.rope_append(q[:, :2], k[:, :2], k[:, :2], k, rows(4), lens, f),
             lambda: ua.rope_append(k[:, :2], k[:, :2], k[:, :2], q, shifted, lens, f)]
    for call in calls:
        with pytest.raises(ValueError):
            call()


def test_in_place_and_packed_results_are_taken():
    f, _ = ua.rope_freqs(64, device=DEV)
    pack = rows(8)
    q, k, v = pack[:, :, :4], pack[:, :, 4:6], pack[:, :, 6:]
    want = ua.rope_fwd(q, k, f)
    ua.rope_fwd(q, k, f, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    out, lse = ua.swa_fwd(q, k, v)
    grads = torch.empty_like(pack)
    dq, dk, dv = grads[:, :, :4], grads[:, :, 4:6], grads[:, :, 6:]
    want = ua.swa_bwd(out, q, k, v, out, lse)
    ua.swa_bwd(out, q, k, v, out, lse, dq=dq, dk=dk, dv=dv)
    assert all(torch.equal(x, y) for x, y in zip(want, (dq, dk, dv)))
    ua.swa_fwd(q, k, v, out=q)
    assert torch.equal(q, out)
