"""fp16 holds values below 6e-5 with fewer bits and none below 3e-8: probabilities of long rows lie there."""
import math

import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV

pytestmark = pytest.mark.gpu


def one_and_many(seq_q, seq_k, dim, below):
    """Keys of which the first scores `below` (a factor of P) above all others; its value is 0, the others' are 1."""
    q = torch.zeros(1, seq_q, 1, dim, device=DEV, dtype=torch.float16)
    k = torch.zeros(1, seq_k, 1, dim, device=DEV, dtype=torch.float16)
    v = torch.ones(1, seq_k, 1, dim, device=DEV, dtype=torch.float16)
    q[..., 0] = 8.0
    k[0, 0, 0, 0] = math.log(below) * dim ** 0.5 / 8
    v[0, 0] = 0
    s = 8.0 * k[0, 0, 0, 0].double().item() * dim ** -0.5
    rest = (seq_k - 1) * math.exp(-s)
    return q, k, v, rest / (1 + rest)


# The exact row is rest / (1 + rest).  Half a step of the result, of P (both 2^-11), scores and sums in 32 bits (70000 * 2^-24 = 2^-8 at most, of
# which a sum over parts has less): 2^-10 + 2^-8 of the value; the result's own last place; and P held to 2^-32 of the largest.
def close(got, want, seq_k=70000):
    return ((got.double() - want).abs() <= (2.0 ** -10 + 2.0 ** -8) * want + 2.0 ** -25 + seq_k * 2.0 ** -32).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("below", [2.0 ** 16, 2.0 ** 26, 2.0 ** 27])
def test_many_keys_far_below_the_largest_decode(dim, below):
    q, k, v, want = one_and_many(1, 70000, dim, below)
    for batch, heads in ((1, 1), (40, 8)):                             # in parts, and whole
        many = [x.expand(batch, x.shape[1], heads, dim) for x in (q, k, v)]
        out, _ = ua.swa_decode(*many, torch.full((batch,), 70000, dtype=torch.int32, device=DEV))
        assert close(out, want), (batch, out.flatten()[:4], want)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("below", [2.0 ** 16, 2.0 ** 26, 2.0 ** 27])
def test_many_keys_far_below_the_largest_forward(dim, below):
    q, k, v, want = one_and_many(130, 70000, dim, below)
    out, _ = ua.swa_fwd(q, k, v, (-1, -1))
    assert close(out, want), (out.flatten()[:4], want)
