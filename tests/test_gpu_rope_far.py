"""The farthest positions that are turned exactly, and those refused."""
import pytest
import torch

import ultraattn_amd as ua
from tests.test_gpu_rope import DEV, check, positions, rows

pytestmark = pytest.mark.gpu


def test_farthest_positions():
    f, q = ua.rope_freqs(128, device=DEV)[0], rows(2, 64, 2, 128, torch.float32)
    for start in (2 ** 53 - 64, -(2 ** 53)):
        check(ua.rope_fwd(q, None, f, start=start)[0], q, positions(2, 64, start), f)
        check(ua.rope_bwd(q, None, f, positions=positions(2, 64, start))[0], q, positions(2, 64, start), f, back=True)
    for start in (2 ** 53 - 63, -(2 ** 53) - 1, 2 ** 63 - 1):
        with pytest.raises(ValueError, match="2\\^53"):
            ua.rope_fwd(q, None, f, start=start)
