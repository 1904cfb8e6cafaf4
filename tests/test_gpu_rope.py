"""Rotary positions against their definition; angles are reduced exactly, as integers.

Bounds: an output is rounded once, by half a step of its type.  What comes before is 32 bits: the angle in half turns (|x| <= 1, off by 2^-25,
times pi), sine and cosine (two steps of 2^-24), three roundings of products and sums of 2^-24 each, together under 3.4 * 2^-23 of
scale * (|a| + |b|); 2^-21 is allowed.
"""
import itertools

import numpy as np
import pytest
import torch

import ultraattn_amd as ua

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


TWO_PI = int("6283185307179586476925286766559005768394338798750211641949889184615632812572417997256069650684234136")   # * 10^99


def reduced(pos, freqs):
    """pos * freq modulo 2 pi as float64: both are rationals, so the product and its remainder are exact but for 2 pi's 99 decimals."""
    out = np.empty((pos.size, len(freqs)))
    for j, f in enumerate(float(x) for x in freqs):
        m, d = f.as_integer_ratio()
        for i, p in enumerate(pos.reshape(-1).tolist()):
            rest = (p * m * 10 ** 99) % (TWO_PI * d)
            out[i, j] = rest * 10 ** 20 // (d * 10 ** 99) / 1e20
    return out.reshape(*pos.shape, len(freqs))


def turn(x, pos, freqs, interleaved=False, scale=1.0, back=False):
    """(turned, bound) as float64 numpy, pos [B, S]."""
    f, n = x.detach().cpu().double().numpy(), len(freqs)
    angle = reduced(pos.cpu().numpy(), freqs.cpu().numpy())[:, :, None]
    c, s = np.cos(angle), np.sin(angle)
    s = -s if back else s
    one, two = (np.s_[..., 0:2 * n:2], np.s_[..., 1:2 * n:2]) if interleaved else (np.s_[..., :n], np.s_[..., n:2 * n])
    y, size = f.copy(), np.zeros_like(f)
    y[one], y[two] = scale * (f[one] * c - f[two] * s), scale * (f[two] * c + f[one] * s)
    size[one] = size[two] = scale * (np.abs(f[one]) + np.abs(f[two]))
    return y, torch.finfo(x.dtype).eps / 2 * np.abs(y) * (1 + 2e-6) + 2.0 ** -21 * size


def check(got, x, pos, freqs, **how):
    y, bound = turn(x, pos, freqs, **how)
    err = np.abs(got.detach().cpu().double().numpy() - y)
    assert (err <= bound).all(), (float((err - bound).max()), np.argwhere(err > bound)[:3])


def rows(b, s, h, d, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(b, s, h, d, generator=g, device=DEV).to(dtype)


def positions(b, s, start=0):
    return start + torch.arange(s, device=DEV).expand(b, s)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
# whole heads, parts of them that vectors of 8, 4, 2 and 1 elements fit, one pair, the largest head
@pytest.mark.parametrize("dim,rotary", [(128, 128), (64, 32), (128, 48), (72, 40), (40, 20), (66, 12), (9, 6), (128, 2), (512, 512)])
def test_layouts(dtype, interleaved, dim, rotary):
    q, k = rows(2, 5, 3, dim, dtype), rows(2, 5, 2, dim, dtype, 1)
    f = ua.rope_freqs(rotary, device=DEV)[0]
    for back, run in ((False, ua.rope_fwd), (True, ua.rope_bwd)):
        qo, ko = run(q, k, f, start=3, interleaved=interleaved, scale=1.25)
        check(qo, q, positions(2, 5, 3), f, interleaved=interleaved, scale=1.25, back=back)
        check(ko, k, positions(2, 5, 3), f, interleaved=interleaved, scale=1.25, back=back)
        assert torch.equal(qo[..., rotary:], q[..., rotary:]) and torch.equal(ko[..., rotary:], k[..., rotary:])


@pytest.mark.parametrize("b,s,h,hk", [(1, 1, 1, 0), (1, 1, 32, 8), (3, 333, 7, 1), (1, 4097, 5, 5), (2, 2500, 16, 2)])
def test_sizes(b, s, h, hk):
    q, k = rows(b, s, h, 64, torch.bfloat16), rows(b, s, hk, 64, torch.bfloat16, 1) if hk else None
    f = ua.rope_freqs(64, device=DEV)[0]
    qo, ko = ua.rope_fwd(q, k, f, start=17)
    check(qo, q, positions(b, s, 17), f)
    if hk:
        check(ko, k, positions(b, s, 17), f)
    else:
        assert ko is None


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions_in_any_order_far_and_negative(kind):
    f = ua.rope_freqs(128, device=DEV)[0]
    q = rows(2, 64, 2, 128, torch.float32)
    g = torch.Generator().manual_seed(5)
    pos = torch.randint(-(2 ** 31), 2 ** 31 - 1, (2, 64), generator=g)
    pos[0, :3] = torch.tensor([0, 2 ** 31 - 1, -(2 ** 31)])
    if kind == torch.int64:
        pos[1] *= 2 ** 14                                                # up to 2^45
    check(ua.rope_fwd(q, None, f, positions=pos.to(DEV, kind))[0], q, pos, f)
    wide = torch.zeros(64, 4, 2, dtype=kind, device=DEV)                  # strided [B, S], and one row for all
    wide[:, 1] = pos.T.to(DEV, kind)
    check(ua.rope_fwd(q, None, f, positions=wide[:, 1].T)[0], q, pos, f)
    check(ua.rope_fwd(q, None, f, positions=wide[:, 1, 0])[0], q, pos[:1].expand(2, 64), f)
    check(ua.rope_fwd(q, None, f, start=2 ** 40)[0], q, positions(2, 64, 2 ** 40), f)


def test_views_and_in_place():
    f = ua.rope_freqs(32, device=DEV)[0]
    qkv = rows(2, 37, 10, 64, torch.float16)
    want = {i: turn(x, positions(2, 37), f) for i, x in enumerate((qkv[:, :, :6], qkv[:, :, 6:8]))}
    before = qkv.clone()
    q, k = qkv[:, :, :6], qkv[:, :, 6:8]
    qo, ko = ua.rope_fwd(q, k, f, q_out=q, k_out=k)                       # into the projection's own output
    assert qo is q and ko is k and torch.equal(qkv[:, :, 8:], before[:, :, 8:])
    for i, x in enumerate((q, k)):
        assert (np.abs(x.cpu().double().numpy() - want[i][0]) <= want[i][1]).all()
    heads_first = rows(2, 6, 37, 64, torch.float16).transpose(1, 2)
    check(ua.rope_fwd(heads_first, None, f)[0], heads_first, positions(2, 37), f)
    flat = rows(1, 1, 1, 4000, torch.float16).flatten()
    odd = flat[1:1 + 3 * 5 * 4 * 64].view(3, 5, 4, 64)                    # not on any vector's boundary
    check(ua.rope_fwd(odd, None, f)[0], odd, positions(3, 5), f)
    one = rows(2, 37, 1, 64, torch.float16).expand(2, 37, 6, 64)          # a broadcast input; the result is not
    check(ua.rope_fwd(one, None, f)[0], one, positions(2, 37), f)
    into = torch.full((2, 40, 6, 64), 7.0, dtype=torch.float16, device=DEV)
    ua.rope_fwd(one, None, f, q_out=into[:, 1:38])
    check(into[:, 1:38], one, positions(2, 37), f)
    assert (into[:, :1] == 7).all() and (into[:, 38:] == 7).all()
    empty = rows(2, 0, 6, 64, torch.float16)
    assert ua.rope_fwd(empty, None, f)[0].shape == empty.shape


@pytest.mark.parametrize("rotary,interleaved,partner", [(16, False, 11), (20, False, 13), (20, True, 2), (6, True, 2), (6, False, None)])
def test_infinities_stay_in_their_pair(rotary, interleaved, partner):
    f = ua.rope_freqs(rotary, device=DEV)[0]
    q = rows(1, 4, 1, 32, torch.bfloat16)
    at = 3 if partner is not None else 7                              # (behind the pairs: alone)
    q[0, 2, 0, at] = torch.inf
    got = ua.rope_fwd(q, None, f, start=1, interleaved=interleaved)[0]
    bad = ~torch.isfinite(got)
    assert bad[0, 2, 0, at] and (partner is None or bad[0, 2, 0, partner]) and bad.sum() == (1 if partner is None else 2)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 20), (64, 12), (64, 6), (128, 36), (48, 46)])
def test_parts_that_no_vector_divides_in_place_and_not(dim, rotary, interleaved):
    q, k = rows(2, 40, 3, dim, torch.float16), rows(2, 40, 2, dim, torch.float16, 1)
    f = ua.rope_freqs(rotary, device=DEV)[0]
    qo, ko = ua.rope_fwd(q, k, f, start=9, interleaved=interleaved)
    check(qo, q, positions(2, 40, 9), f, interleaved=interleaved)
    check(ko, k, positions(2, 40, 9), f, interleaved=interleaved)
    x = q.clone()
    ua.rope_fwd(x, None, f, start=9, interleaved=interleaved, q_out=x)
    assert torch.equal(x, qo)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_the_formula_and_differences(interleaved):
    """The turn is linear: differences with a step of 1 are exact up to the roundings of 32 bits."""
    f, scale = ua.rope_freqs(48, scaling="yarn", factor=4.0, original_length=100, device=DEV)
    x, g, d = (rows(2, 9, 3, 64, torch.float32, i) for i in range(3))
    how = dict(interleaved=interleaved, scale=scale, start=50)
    dx = ua.rope_bwd(g, None, f, **how)[0]
    check(dx, g, positions(2, 9, 50), f, interleaved=interleaved, scale=scale, back=True)
    up, down = (ua.rope_fwd(x + e * d, None, f, **how)[0].double() for e in (1, -1))
    along, want = ((up - down) / 2 * g).sum().item(), (dx.double() * d).sum().item()
    # 3456 products of entries of size about 1, each off by under 2^-21 * 4
    assert abs(along - want) <= 3456 * 2.0 ** -19, (along, want)


@pytest.mark.parametrize("dtype,interleaved,tokens", itertools.product(TYPES, [False, True], [1, 3]))
def test_append(dtype, interleaved, tokens):
    """Every row of the caches but the new ones stays as it is, bit for bit."""
    b, room, hk, dim = 7, 20, 2, 64
    lens = torch.tensor([0, 1, 2, 20, 21, 23, 11], dtype=torch.int32, device=DEV)
    q, k, v = rows(b, tokens, 6, dim, dtype), rows(b, tokens, hk, dim, dtype, 1), rows(b, tokens, hk, dim, dtype, 2)
    store = rows(2, b, room + 2, hk * dim, dtype, 3).view(2, b, room + 2, hk, dim)
    before = store.clone()
    kc, vc = store[0, :, 1:-1], store[1, :, 1:-1]
    f = ua.rope_freqs(32, device=DEV)[0]
    qo = ua.rope_append(q, k, v, kc, vc, lens, f, interleaved=interleaved, scale=1.5)
    pos = lens.long()[:, None] - tokens + torch.arange(tokens, device=DEV)
    check(qo, q, pos, f, interleaved=interleaved, scale=1.5)
    turned, bound = turn(k, pos, f, interleaved=interleaved, scale=1.5)
    for i in range(b):
        for t in range(tokens):
            at = int(pos[i, t])
            if 0 <= at < room:
                assert (np.abs(kc[i, at].cpu().double().numpy() - turned[i, t]) <= bound[i, t]).all()
                assert torch.equal(vc[i, at], v[i, t])
                kc[i, at], vc[i, at] = before[0, i, at + 1], before[1, i, at + 1]
    assert torch.equal(store, before)


def test_append_in_place_q_and_no_room():
    f = ua.rope_freqs(64, device=DEV)[0]
    q, k = rows(2, 1, 4, 64, torch.bfloat16), rows(2, 1, 2, 64, torch.bfloat16, 1)
    none = torch.empty(2, 0, 2, 64, dtype=torch.bfloat16, device=DEV)
    lens = torch.tensor([5, 9], dtype=torch.int32, device=DEV)
    x = q.clone()
    assert ua.rope_append(x, k, k, none, none, lens, f, q_out=x) is x
    check(x, q, lens.long()[:, None] - 1, f)


def test_refusals():
    f = ua.rope_freqs(64, device=DEV)[0]
    q, k = rows(2, 4, 4, 64, torch.bfloat16), rows(2, 4, 2, 64, torch.bfloat16)
    lens, cache = torch.ones(2, dtype=torch.int32, device=DEV), rows(2, 8, 2, 64, torch.bfloat16)
    bad = [lambda: ua.rope_fwd(q, k.half(), f), lambda: ua.rope_fwd(q, k[:, :3], f), lambda: ua.rope_fwd(q, k[..., :32], f),
           lambda: ua.rope_fwd(q, k, f.float()), lambda: ua.rope_fwd(q, k, f.cpu()), lambda: ua.rope_fwd(q, k, torch.cat([f, f])),
           lambda: ua.rope_fwd(q, k, f[::2]), lambda: ua.rope_fwd(q, k, f, positions=torch.zeros(3, dtype=torch.int32, device=DEV)),
           lambda: ua.rope_fwd(q, k, f, positions=torch.zeros(4, device=DEV)), lambda: ua.rope_fwd(q, k, f, positions=torch.zeros(4, dtype=torch.int32)),
           lambda: ua.rope_fwd(q, k, f, scale=0.0), lambda: ua.rope_fwd(q, k, f, scale=float("inf")),
           lambda: ua.rope_fwd(q.transpose(2, 3), None, f), lambda: ua.rope_fwd(q[0], None, f), lambda: ua.rope_fwd(q.double(), None, f),
           lambda: ua.rope_fwd(q, None, f, k_out=k), lambda: ua.rope_fwd(q, k, f, q_out=k), lambda: ua.rope_fwd(q, k, f, q_out=q.half()),
           lambda: ua.rope_fwd(q, k, f, q_out=q[:, :, :1].expand(2, 4, 4, 64)), lambda: ua.rope_append(q, k, k, cache, cache[:, :3], lens, f),
           lambda: ua.rope_append(q, k, k, cache, cache, lens.long(), f), lambda: ua.rope_append(q, k, k, cache, cache, lens[:1], f),
           lambda: ua.rope_append(q, k, k[:, :1], cache, cache, lens, f), lambda: ua.rope_append(q, k, k, cache[:1].expand(2, 8, 2, 64), cache, lens, f),
           lambda: ua.rope_append(q, k, k, cache, cache, lens.cpu(), f)]
    same = rows(2, 4, 4, 64, torch.bfloat16, 7)
    bad += [lambda: ua.rope_fwd(q, same, f, q_out=same), lambda: ua.rope_fwd(q, same, f, k_out=q), lambda: ua.rope_fwd(q, same, f, q_out=q, k_out=q),
            lambda: ua.rope_append(q, k, k, cache, cache, lens, f)]
    before = q.clone(), k.clone(), cache.clone()
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    assert all(torch.equal(x, y) for x, y in zip(before, (q, k, cache)))


def test_captured_and_on_another_stream():
    f = ua.rope_freqs(64, device=DEV)[0]
    q, k = rows(2, 50, 4, 64, torch.bfloat16), rows(2, 50, 2, 64, torch.bfloat16, 1)
    ua.rope_fwd(q, k, f)
    torch.cuda.synchronize()
    pos = torch.zeros(2, 50, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = ua.rope_fwd(q, k, f, positions=pos)
    for start in (0, 70, 5):
        pos.copy_(positions(2, 50, start))
        q.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        check(qo, q, pos, f)
        check(ko, k, pos, f)
        assert torch.equal(qo, ua.rope_fwd(q, k, f, start=start)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ua.rope_fwd(q, None, f, positions=pos)[0]
    side.synchronize()
    assert torch.equal(got, qo)
