"""Rotations whose results go past the caches (more than 128 MiB), all types and layouts, against the same rows turned in smaller calls and sampled rows
against the definition; and rows whose offsets pass 2^31 elements."""
import pytest
import torch

import ultraattn_amd as ua
from tests.test_gpu_rope import DEV, check, positions, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,seq", [(torch.bfloat16, 8500), (torch.float16, 8500), (torch.float32, 4250)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [128, 40])
def test_results_beyond_the_caches(dtype, seq, interleaved, rotary):
    q, k = rows(2, seq, 28, 128, dtype), rows(2, seq, 4, 128, dtype, 1)
    assert (q.numel() + k.numel()) * q.element_size() > 128 << 20
    f = ua.rope_freqs(rotary, device=DEV)[0]
    how = dict(interleaved=interleaved, scale=1.25)
    for back, run in ((False, ua.rope_fwd), (True, ua.rope_bwd)):
        qo, ko = run(q, k, f, start=11, **how)
        for s in range(0, seq, 1000):                                    # (results of a call: at most 33 MB)
            part = slice(s, min(s + 1000, seq))
            qp, kp = run(q[:, part], k[:, part], f, start=11 + s, **how)
            assert torch.equal(qp, qo[:, part]) and torch.equal(kp, ko[:, part])
        at = torch.tensor([0, 1, 777, seq - 1], device=DEV)
        check(qo[:, at, ::9], q[:, at, ::9], 11 + at.expand(2, 4), f, back=back, **how)
    x, y = q.clone(), k.clone()
    ua.rope_fwd(x, y, f, start=11, q_out=x, k_out=y, **how)              # in place
    want = ua.rope_fwd(q, k, f, start=11, **how)
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_rows_beyond_two_to_the_31_elements():
    """A view whose last batch, and one whose last head, begins behind 2^31 elements."""
    f = ua.rope_freqs(64, device=DEV)[0]
    room = torch.zeros(2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device=DEV)
    x = rows(2, 50, 2, 64, torch.bfloat16)
    want = ua.rope_fwd(x, None, f)[0]
    for strides in ((2 ** 31, 128, 64, 1), (6400, 128, 2 ** 31, 1)):
        far = room.as_strided(x.shape, strides)
        far.copy_(x)
        assert torch.equal(ua.rope_fwd(far, None, f)[0], want)
        ua.rope_fwd(far, None, f, q_out=far)
        assert torch.equal(far, want)
    lens = torch.tensor([50, 50], dtype=torch.int32, device=DEV)
    caches = [room.as_strided(x.shape, (2 ** 31, 128, 64, 1)), torch.zeros_like(x)]
    for kc, vc in (caches, caches[::-1]):
        ua.rope_append(x, x, x, kc, vc, lens, f)
        assert torch.equal(kc, want) and torch.equal(vc, x)
