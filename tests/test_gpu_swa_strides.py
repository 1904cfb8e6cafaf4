"""Tokens that lie far apart: up to the limit they are taken, beyond it the tensor is named."""
import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, inputs

pytestmark = pytest.mark.gpu
MOST = 4194296                                                        # the largest multiple of 8 up to the limit


def apart(x, stride):
    """x [1, S, H, D] with its tokens `stride` elements apart."""
    far = torch.empty((x.shape[1] - 1) * stride + x[0, 0].numel(), dtype=x.dtype, device=DEV).as_strided(x.shape, (stride, stride, x.shape[3], 1))
    return far.copy_(x)


@pytest.mark.parametrize("which", range(4))
def test_limit(which):
    args = list(inputs(1, 100, 100, 2, 2, 64, torch.bfloat16))
    q, k, v, do = args
    out, lse = ua.swa_fwd(q, k, v, (30, 0), 2)
    want = ua.swa_bwd(do, q, k, v, out, lse, (30, 0), 2)
    lens = torch.full((1,), 100, dtype=torch.int32, device=DEV)
    dec = ua.swa_decode(q[:, -2:].contiguous(), k, v, lens, 30, 2)
    x = args[which]
    args[which] = apart(x, MOST)
    q, k, v, do = args
    assert torch.equal(ua.swa_fwd(q, k, v, (30, 0), 2)[0], out)
    assert all(torch.equal(a, b) for a, b in zip(ua.swa_bwd(do, q, k, v, out, lse, (30, 0), 2), want))
    assert torch.equal(ua.swa_decode(q[:, -2:], k, v, lens, 30, 2)[0], dec[0])
    args[which] = apart(x[:, :2], MOST + 8)
    q, k, v, do = (a[:, :2] for a in args)
    name = ("q", "k", "v", "dout")[which]
    if which in (1, 2):
        with pytest.raises(ValueError, match=f"^{name}: its tokens lie {MOST + 8} elements apart"):
            ua.swa_fwd(q, k, v)
        with pytest.raises(ValueError, match=f"^{name}_cache: its tokens lie"):
            ua.swa_decode(q, k, v, lens)
    else:
        ua.swa_fwd(q, k, v)                                            # the forward does not walk it
    with pytest.raises(ValueError, match=f"^{name}: its tokens lie"):
        ua.swa_bwd(do, q, k, v, out[:, :2], lse[..., :2].contiguous())
    ua.swa_fwd(*(a[:, 1:2] for a in (q, k, v)))                        # of one token there is no stride
