"""New tokens against a cache, against the definition in 64 bits (bounds: swa_util), and a serving step with rotary positions."""
import math

import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, Reference, inputs

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def visible(lens, tokens, room, window, sinks):
    pos = (lens.long()[:, None] - tokens + torch.arange(tokens, device=DEV))[:, :, None]
    key = torch.arange(room, device=DEV)
    seen = (key <= pos) & (key < lens.long()[:, None, None])
    if window >= 0:
        seen &= (key >= pos - window) | (key < sinks)
    return seen[:, None]


def run(q, kc, vc, lens, window=-1, sinks=0, scale=None):
    out, lse = ua.swa_decode(q, kc, vc, lens, window, sinks, scale)
    Reference(q, kc, vc, visible(lens, q.shape[1], kc.shape[1], window, sinks), scale).check(out=out, lse=lse)
    return out, lse


def lengths(room, batch, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, room + 1, (batch,), generator=g)
    lens[:3] = torch.tensor([0, 1, room])[:batch]
    return lens.to(DEV, torch.int32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 5])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (7, 1), (40, 2)])
@pytest.mark.parametrize("room,window,sinks", [(1, -1, 0), (33, -1, 0), (500, -1, 0), (500, 0, 0), (500, 100, 5), (500, 31, 70), (3000, 1000, 4)])
def test_lengths_and_windows(dtype, dim, tokens, heads, kv_heads, room, window, sinks):
    q, kc, vc, _ = inputs(5, tokens, room, heads, kv_heads, dim, dtype, room + tokens)
    run(q, kc, vc, lengths(room, 5), window, sinks)


def test_many_tokens_and_long_caches():
    q, kc, vc, _ = inputs(2, 40, 900, 6, 2, 64, torch.float16)
    run(q, kc, vc, torch.tensor([900, 41], dtype=torch.int32, device=DEV), 100, 3)
    q, kc, vc, _ = inputs(1, 1, 70001, 4, 1, 128, torch.bfloat16)
    run(q, kc, vc, torch.tensor([70000], dtype=torch.int32, device=DEV))
    q, kc, vc, _ = inputs(70, 1, 700, 8, 8, 64, torch.bfloat16)
    run(q, kc, vc, lengths(700, 70))


def test_cache_beyond_two_gigabytes():
    """Rows of the last head lie behind offsets of 32 bits, in bytes and in elements."""
    room = 1_100_000
    kc = torch.zeros(1, room, 16, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    assert kc.numel() > 2 ** 31
    q, k, v, _ = inputs(1, 1, 200, 16, 16, 128, torch.bfloat16)
    kc[:, -200:], vc[:, -200:] = k, v
    lens = torch.tensor([room], dtype=torch.int32, device=DEV)
    out, lse = ua.swa_decode(q, kc, vc, lens, 199)
    seen = torch.ones(1, 200, dtype=torch.bool, device=DEV)
    Reference(q, k, v, seen).check(out=out, lse=lse)
    out, lse = ua.swa_decode(q, kc, vc, lens)
    S = torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double()) * 128 ** -0.5
    want = torch.logsumexp(torch.cat([S, torch.zeros_like(S[..., :1]) + math.log(room - 200)], -1), -1)
    assert (lse.double() - want).abs().max() < 1e-4                   # (1.1 million terms of 32 bits in 256 sums or more: 4300 * 2^-24 each)


def test_nothing_behind_the_lengths_is_read():
    q, kc, vc, _ = inputs(6, 2, 300, 8, 2, 128, torch.bfloat16)
    lens = torch.tensor([0, 1, 31, 32, 133, 299], dtype=torch.int32, device=DEV)
    want = run(q, kc, vc, lens, 50, 3)
    for b, n in enumerate(lens.tolist()):
        kc[b, n:], vc[b, n:] = torch.nan, torch.inf
    got = ua.swa_decode(q, kc, vc, lens, 50, 3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (got[0][0] == 0).all() and (got[1][0] == -math.inf).all() and (got[1][1, :, 0] == -math.inf).all()


def test_lengths_outside_the_cache():
    q, kc, vc, _ = inputs(4, 1, 100, 2, 2, 64, torch.float16)
    lens = torch.tensor([-5, 130, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32, device=DEV)
    out, lse = ua.swa_decode(q, kc, vc, lens, 50, 2)
    assert (lse[[0, 3]] == -math.inf).all() and (out[[0, 3]] == 0).all()
    key = torch.arange(100, device=DEV)
    Reference(q[1:2], kc[1:2], vc[1:2], ((key >= 79) | (key < 2))[None]).check(out=out[1:2], lse=lse[1:2])
    Reference(q[2:3], kc[2:3], vc[2:3], (key < 2)[None]).check(out=out[2:3], lse=lse[2:3])


def test_views_strides_and_given_results():
    store = inputs(3, 1, 64, 1, 1, 64, torch.bfloat16)[1]
    kv = torch.randn(3, 2, 4, 64, 64, device=DEV).to(torch.bfloat16)          # [B, 2, H, room, D], as some caches lie
    kc, vc = kv[:, 0].transpose(1, 2), kv[:, 1].transpose(1, 2)
    q = inputs(3, 2, 1, 12, 1, 64, torch.bfloat16)[0]
    lens = torch.tensor([64, 3, 40], dtype=torch.int32, device=DEV)
    out, lse = run(q[:, :, :8], kc, vc, lens, 20, 1)
    room = torch.full_like(q, 7.0)
    stat = torch.empty_like(lse)
    got = ua.swa_decode(q[:, :, :8], kc, vc, lens, 20, 1, out=room[:, :, 2:10], lse=stat)
    assert got[1] is stat and torch.equal(room[:, :, 2:10], out) and torch.equal(stat, lse) and (room[:, :, :2] == 7).all() and (room[:, :, 10:] == 7).all()
    run(q, store.expand(3, 64, 4, 64), store.expand(3, 64, 4, 64), lens, 20, 1)
    empty = inputs(3, 2, 0, 8, 4, 64, torch.bfloat16)
    out, lse = ua.swa_decode(q[:, :, :8], empty[1], empty[2], lens)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert ua.swa_decode(q[:0, :, :8], kc[:0], vc[:0], lens[:0])[0].shape == (0, 2, 8, 64)
    assert ua.swa_decode(q[:, :0, :8], kc, vc, lens)[1].shape == (3, 8, 0)


def test_agrees_with_the_prompt_form():
    q, kc, vc, _ = inputs(1, 4, 777, 8, 2, 128, torch.bfloat16)
    lens = torch.tensor([777], dtype=torch.int32, device=DEV)
    a, b = run(q, kc, vc, lens, 300, 4), ua.swa_fwd(q, kc, vc, (300, 0), 4)
    Reference(q, kc, vc, visible(lens, 4, 777, 300, 4)).check(out=b[0], lse=b[1])
    assert (a[1] - b[1]).abs().max() < 1e-4


@pytest.mark.parametrize("interleaved", [False, True])
def test_serving_steps_equal_the_prompt(interleaved):
    """rope_append and swa_decode, token by token and by threes, captured once and replayed, against rope_fwd and swa_fwd of the whole sequence."""
    b, steps, hq, hk, dim, window, sinks = 2, 24, 4, 2, 64, 9, 2
    q, k, v, _ = inputs(b, steps, steps, hq, hk, dim, torch.float16)
    f, scale = ua.rope_freqs(dim // 2, scaling="yarn", factor=2.0, original_length=16, device=DEV)
    qr, kr = ua.rope_fwd(q, k, f, interleaved=interleaved, scale=scale)
    whole = ua.swa_fwd(qr, kr, v, (window, 0), sinks)
    ref = Reference(qr, kr, v, torch.stack([visible(torch.tensor([steps], device=DEV), steps, steps, window, sinks)[0, 0]])[0])
    ref.check(out=whole[0], lse=whole[1])
    for tokens in (1, 3):
        kc, vc = torch.full((2, b, steps, hk, dim), torch.nan, dtype=torch.float16, device=DEV)
        lens = torch.zeros(b, dtype=torch.int32, device=DEV)
        sq, sk, sv = (torch.zeros(b, tokens, h, dim, dtype=torch.float16, device=DEV) for h in (hq, hk, hk))

        def step():
            lens.add_(tokens)
            turned = ua.rope_append(sq, sk, sv, kc, vc, lens, f, interleaved=interleaved, scale=scale)
            return ua.swa_decode(turned, kc, vc, lens, window, sinks)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = step()
        lens.zero_()
        kc.fill_(torch.nan)
        vc.fill_(torch.nan)
        got = []
        for i in range(0, steps, tokens):
            for x, y in ((sq, q), (sk, k), (sv, v)):
                x.copy_(y[:, i:i + tokens])
            graph.replay()
            got.append((out.clone(), lse.clone()))
            torch.cuda.synchronize()
        assert torch.equal(kc, kr) and torch.equal(vc, v)
        ref.check(out=torch.cat([g[0] for g in got], 1), lse=torch.cat([g[1] for g in got], 2))


def test_two_calls_at_once():
    args = [inputs(1, 1, 5000, 8, 2, 128, torch.bfloat16, s)[:3] for s in (0, 1)]
    lens = torch.tensor([5000], dtype=torch.int32, device=DEV)
    want = [run(*a, lens) for a in args]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ua.swa_decode(*args[i], lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g[0], want[i][0]) and torch.equal(g[1], want[i][1]) for g in got[i])


def test_refusals():
    q, kc, vc, _ = inputs(2, 1, 16, 4, 2, 64, torch.bfloat16)
    lens = torch.ones(2, dtype=torch.int32, device=DEV)
    bad = [lambda: ua.swa_decode(q, kc, vc[:, :8], lens), lambda: ua.swa_decode(q, kc, vc, lens.long()), lambda: ua.swa_decode(q, kc, vc, lens[:1]),
           lambda: ua.swa_decode(q, kc, vc, lens.cpu()), lambda: ua.swa_decode(q, kc, vc, lens, -2), lambda: ua.swa_decode(q, kc, vc, lens, 3, -1),
           lambda: ua.swa_decode(q.float(), kc.float(), vc.float(), lens), lambda: ua.swa_decode(q[:, :, :3], kc, vc, lens),
           lambda: ua.swa_decode(q, kc.half(), vc, lens), lambda: ua.swa_decode(q, kc, vc, lens, out=q[:, :, :2]), lambda: ua.swa_decode(q[:1], kc, vc, lens),
           lambda: ua.swa_decode(q, kc, vc, lens, softmax_scale=0.0), lambda: ua.swa_decode(q, kc, vc, lens[None]),
           lambda: ua.swa_decode(q, kc, vc, torch.ones(4, dtype=torch.int32, device=DEV)[::2])]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
