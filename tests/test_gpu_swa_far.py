"""Rows of queries, keys, values and gradients whose offsets pass 2^31 elements: the last batch or the last head of a strided view."""
import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def room():
    yield torch.zeros(2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device=DEV)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("far_head", [False, True])
def test_forward_and_backward(room, dim, far_head):
    q, k, v, do = inputs(2, 200, 200, 2, 2, dim, torch.bfloat16)
    how = dict(window=(70, 0), sinks=3)
    out, lse = ua.swa_fwd(q, k, v, **how)
    want = (out, *ua.swa_bwd(do, q, k, v, out, lse, **how))
    strides = (400 * dim, 2 * dim, 2 ** 31, 1) if far_head else (2 ** 31, 2 * dim, dim, 1)

    def far(x):
        y = room.as_strided(x.shape, strides)
        y.copy_(x)
        return y

    for i in range(4):                                                    # one operand at a time lies far out
        args = [q, k, v, do]
        args[i] = far(args[i])
        a, b, c, d = args
        got = ua.swa_fwd(a, b, c, **how)
        assert torch.equal(got[0], out) and torch.equal(got[1], lse)
        assert all(torch.equal(x, y) for x, y in zip(ua.swa_bwd(d, a, b, c, out, lse, **how), want[1:]))
    at = far(out)
    assert all(torch.equal(x, y) for x, y in zip(ua.swa_bwd(do, q, k, v, at, lse, **how), want[1:]))
    at.zero_()
    assert torch.equal(ua.swa_fwd(q, k, v, out=at, **how)[0], out)
    for i, name in enumerate(("dq", "dk", "dv"), 1):                      # and one result
        at.zero_()
        got = ua.swa_bwd(do, q, k, v, out, lse, **how, **{name: at})
        assert all(torch.equal(x, y) for x, y in zip(got, want[1:]))
