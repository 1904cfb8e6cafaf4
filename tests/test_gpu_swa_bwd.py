"""Sliding-window attention, backward, against the formula in 64 bits (bounds: swa_util), and against differences of the definition."""
import math

import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, Reference, inputs, visible

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def run(q, k, v, do, window=(-1, 0), sinks=0, q_start=None, k_start=0, scale=None, **more):
    how = (window, sinks, scale, q_start, k_start)
    out, lse = ua.swa_fwd(q, k, v, *how)
    dq, dk, dv = ua.swa_bwd(do, q, k, v, out, lse, *how, **more)
    Reference(q, k, v, visible(q.shape[1], k.shape[1], window, sinks, q_start, k_start), scale, do).check(out=out, lse=lse, dq=dq, dk=dk, dv=dv)
    return out, lse, dq, dk, dv


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seq_q,seq_k", [(1, 1), (1, 65), (31, 64), (64, 63), (100, 100), (128, 128), (129, 257), (300, 1000), (513, 511)])
@pytest.mark.parametrize("window,sinks", [((-1, 0), 0), ((20, 0), 3), ((64, 7), 65), ((0, 0), 0), ((130, -1), 1), ((-1, -1), 0)])
def test_lengths_and_windows(dtype, dim, seq_q, seq_k, window, sinks):
    q, k, v, do = inputs(2, seq_q, seq_k, 4, 2, dim, dtype, seq_q + seq_k)
    run(q, k, v, do, window, sinks)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (7, 1), (6, 3), (16, 2)])
def test_shared_key_heads(heads, kv_heads):
    q, k, v, do = inputs(1, 200, 333, heads, kv_heads, 64, torch.bfloat16)
    run(q, k, v, do, (70, 0), 2)


@pytest.mark.parametrize("q_start,k_start", [(5000, 0), (-1000, 0), (150, 0), (400, 300), (390, 10), (2 ** 40 + 100, 2 ** 40), (-3, 0)])
@pytest.mark.parametrize("window,sinks", [((100, 0), 0), ((100, 0), 20), ((100, 50), 20), ((-1, 0), 0)])
def test_shards(q_start, k_start, window, sinks):
    q, k, v, do = inputs(1, 260, 300, 2, 1, 128, torch.bfloat16)
    run(q, k, v, do, window, sinks, q_start, k_start)


def test_no_keys_no_rows_no_batch():
    for b, sq, sk in ((2, 5, 0), (2, 0, 7), (0, 5, 7), (1, 0, 0)):
        q, k, v, do = inputs(b, sq, sk, 4, 2, 64, torch.bfloat16)
        out, lse = ua.swa_fwd(q, k, v, (3, 0))
        dq, dk, dv = ua.swa_bwd(do, q, k, v, out, lse, (3, 0))
        assert dq.shape == q.shape and dk.shape == k.shape and dv.shape == v.shape
        assert not dq.any() and not dk.any() and not dv.any()


# columns of the sinks cut alone (many heads), all columns and rows cut (few lines); more sinks than a tile
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("seq_q,seq_k,heads,window,sinks", [(2000, 2000, 2, (100, 0), 5), (1500, 1500, 48, (128, 0), 4), (1500, 1500, 32, (100, 0), 200),
                                                            (3, 3000, 2, (-1, 0), 0), (1800, 200, 2, (-1, -1), 0), (2000, 70, 40, (64, 0), 70)])
def test_cut_walks(dtype, dim, seq_q, seq_k, heads, window, sinks):
    q, k, v, do = inputs(1, seq_q, seq_k, heads, heads // 2, dim, dtype)
    first = run(q, k, v, do, window, sinks)
    again = run(q, k, v, do, window, sinks)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_shards_add_up():
    """A ring's step: global statistics, partial gradients of the queries added, keys' gradients of their own shard."""
    q, k, v, do = inputs(1, 512, 1024, 4, 4, 128, torch.bfloat16)
    how = dict(window=(300, 0), sinks=10, q_start=512)
    chunks = [(i, k[:, i:i + 256].contiguous(), v[:, i:i + 256].contiguous()) for i in range(0, 1024, 256)]
    parts = [ua.swa_fwd(q, kc, vc, k_start=i, **how) for i, kc, vc in chunks]
    out, lse = ua.merge_partials([p[0] for p in parts], [p[1] for p in parts])
    delta = ua.softmax_delta(out, do)
    grads = [ua.swa_bwd(do, q, kc, vc, None, lse, k_start=i, softmax_d=delta, **how) for i, kc, vc in chunks]
    ref = Reference(q, k, v, visible(512, 1024, (300, 0), 10, 512), dout=do)
    for b in ("dq_bound", "dk_bound", "dv_bound"):
        setattr(ref, b, 6 * getattr(ref, b))                          # rows rounded in every part and merged: twice the forward's; four roundings of dq
    ref.check(dq=ua.grad_sum([g[0] for g in grads]), dk=torch.cat([g[1] for g in grads], 1), dv=torch.cat([g[2] for g in grads], 1))


def test_views_broadcast_and_given_results():
    qkv = inputs(2, 150, 150, 8, 8, 64, torch.float16)[0]
    do = inputs(2, 150, 150, 4, 4, 64, torch.float16, 2)[0]
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    out, lse, dq, dk, dv = run(q, k, v, do, (33, 0), 2)
    room = torch.full_like(qkv, 7.0)                                 # the projection's gradient, in place
    got = ua.swa_bwd(do, q, k, v, out, lse, (33, 0), 2, dq=room[:, :, :4], dk=room[:, :, 4:6], dv=room[:, :, 6:])
    assert torch.equal(room, torch.cat([dq, dk, dv], 2)) and all(torch.equal(x, y) for x, y in zip(got, (dq, dk, dv)))
    one = inputs(2, 150, 150, 1, 1, 64, torch.float16)
    broad = [x.expand(2, 150, 4, 64) for x in (one[1], one[2])]       # the gradient of an expanded input is of its expanded shape
    full = run(q, *broad, do.expand(2, 150, 4, 64), (33, 0), 2)
    dense = run(q, *(x.contiguous() for x in broad), do, (33, 0), 2)
    assert all(torch.equal(x, y) for x, y in zip(full, dense))
    flat = torch.ones(1, 1, 1, 64, dtype=torch.float16, device=DEV).expand(2, 150, 4, 64)      # what sum().backward() hands over
    run(q, k, v, flat, (33, 0), 2)


def test_softmax_d_given():
    q, k, v, do = inputs(2, 200, 200, 4, 2, 64, torch.bfloat16)
    out, lse, dq, dk, dv = run(q, k, v, do, (33, 0), 2)
    delta = (out.float() * do.float()).sum(-1).transpose(1, 2).contiguous()
    got = ua.swa_bwd(do, q, k, v, None, lse, (33, 0), 2, softmax_d=delta)
    Reference(q, k, v, visible(200, 200, (33, 0), 2), dout=do).check(dq=got[0], dk=got[1], dv=got[2])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_delta_of_rows_of_few_keys_is_not_the_rounded_output_s(dtype, dim):
    """Rows of up to 8 keys: dS must not carry the rounding of O.  In a row of one key dS = dP - delta = 0, so dQ is what is left of it."""
    q, k, v, do = inputs(2, 400, 300, 6, 3, dim, dtype)
    for window, sinks, start in (((0, 0), 0, None), ((0, 0), 1, -50), ((7, 0), 3, 100)):
        out, lse = ua.swa_fwd(q, k, v, window, sinks, None, start)
        dq = ua.swa_bwd(do, q, k, v, out, lse, window, sinks, None, start)[0]
        n = visible(400, 300, window, sinks, start).sum(-1)
        one = (n == 1).nonzero()[:, 0]
        if window[0] == 0:
            # |dP - delta| is the difference of two dot products in 32 bits, each off by (dim + 4) 2^-24 of its terms' sum, and of P = 1 by 2^-20
            K = k.double().repeat_interleave(2, dim=2)
            terms = (do.double().abs().sum(-1) * v.double().abs().max())[:, one]
            assert (dq.double()[:, one].abs().amax(-1) <= dim ** -0.5 * (2 * (dim + 4) * 2.0 ** -24 + 2.0 ** -20) * terms * K.abs().max()).all()
            assert len(one) >= 50


def test_delta_of_a_shard_takes_the_whole_rows_output():
    """A shard in which rows have few keys, statistics of the whole: delta must not be made of the shard's keys."""
    q, k, v, do = inputs(1, 64, 300, 2, 2, 128, torch.bfloat16)
    out, lse = ua.swa_fwd(q, k, v, (299, 0), q_start=290)
    ref = Reference(q, k, v, visible(64, 300, (299, 0), 0, 290), dout=do)
    ref.check(out=out, lse=lse)
    parts = [ua.swa_bwd(do, q, k[:, i:j].contiguous(), v[:, i:j].contiguous(), out, lse, (299, 0), q_start=290, k_start=i) for i, j in ((0, 290), (290, 300))]
    for b in ("dq_bound", "dk_bound", "dv_bound"):
        setattr(ref, b, 3 * getattr(ref, b))                          # dq is rounded in either part and once more
    ref.check(dq=ua.grad_sum([g[0] for g in parts]), dk=torch.cat([g[1] for g in parts], 1), dv=torch.cat([g[2] for g in parts], 1))


@pytest.mark.parametrize("window,sinks,q_start", [((10, 0), 2, None), ((5, 5), 0, 3)])
def test_against_differences(window, sinks, q_start):
    """The directional derivative of sum(out * do), by central differences of the definition in 64 bits, at the same inputs."""
    q, k, v, do = inputs(1, 40, 50, 4, 2, 64, torch.float16)
    _, _, dq, dk, dv = run(q, k, v, do, window, sinks, q_start)
    seen = visible(40, 50, window, sinks, q_start)
    g = torch.Generator(device=DEV).manual_seed(9)

    def value(*x):
        return (Reference(x[0], x[1], x[2], seen, 64 ** -0.5).out * do.double()).sum().item()

    ref = Reference(q, k, v, seen, dout=do)
    base = [x.double() for x in (q, k, v)]
    for i, (grad, name) in enumerate(((dq, "dq"), (dk, "dk"), (dv, "dv"))):
        d = torch.randn(base[i].shape, generator=g, device=DEV, dtype=torch.float64)
        step = 1e-4
        moved = [value(*[x + s * step * d if j == i else x for j, x in enumerate(base)]) for s in (1, -1)]
        along, got = (moved[0] - moved[1]) / (2 * step), (grad.double() * d).sum().item()
        # the gradient's own bound, and the differences' error: under 1e-6 of the gradient's size (step^2 = 1e-8 times the third derivative)
        room = (getattr(ref, name + "_bound") * d.abs()).sum().item() + 1e-6 * (grad.double().abs() * d.abs()).sum().item()
        assert abs(along - got) <= room, (name, along, got, room)


@pytest.mark.parametrize("std", [0.05, 4.0])
def test_small_and_large_scores(std):
    for dtype in TYPES:
        q, k, v, do = inputs(1, 300, 400, 2, 2, 64, dtype, std=std)
        run(q, k, v, (do.float() / std).to(dtype), (100, 0), 3, scale=0.2)


def test_captured_while_eager_calls_go_on():
    q, k, v, do = inputs(1, 1000, 1000, 2, 1, 64, torch.bfloat16)
    want = run(q, k, v, do, (100, 0), 4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = ua.swa_fwd(q, k, v, (100, 0), 4)
        res = (out, lse, *ua.swa_bwd(do, q, k, v, out, lse, (100, 0), 4))
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.replay()
        eager = run(q, k, v, do, (100, 0), 4)                         # at the same time, with a workspace of its own
        torch.cuda.synchronize()
        for x, y, w in zip(res, eager, want):
            assert torch.equal(x, w) and torch.equal(y, w)
            x.zero_()


def test_refusals():
    q, k, v, do = inputs(2, 16, 16, 4, 2, 64, torch.bfloat16)
    out, lse = ua.swa_fwd(q, k, v)
    bad = [lambda: ua.swa_bwd(do[:, :8], q, k, v, out, lse), lambda: ua.swa_bwd(do.half(), q, k, v, out, lse), lambda: ua.swa_bwd(do, q, k, v, None, lse),
           lambda: ua.swa_bwd(do, q, k, v, out[:, :8], lse), lambda: ua.swa_bwd(do, q, k, v, out, lse.double()),
           lambda: ua.swa_bwd(do, q, k, v, out, lse.transpose(1, 2)), lambda: ua.swa_bwd(do, q, k, v, out, lse, dq=k),
           lambda: ua.swa_bwd(do, q, k, v, out, lse, dk=q), lambda: ua.swa_bwd(do, q, k, v, out, lse, dk=k[:, :, :1].expand_as(k)),
           lambda: ua.swa_bwd(do, q, k, v, None, lse, softmax_d=lse[:, :2]), lambda: ua.swa_bwd(do, q, k, v, out, lse, softmax_scale=-1.0),
           lambda: ua.swa_bwd(do, q, k, v, out, lse, (-3, 0)), lambda: ua.swa_bwd(do, q, k, v, out.cpu(), lse), lambda: ua.swa_bwd(do, q, k, v, out, lse.cpu())]
    bad += [lambda: ua.swa_bwd(do, q, k, v, out, lse, dq=q), lambda: ua.swa_bwd(do, q, k, v, out, lse, dq=do), lambda: ua.swa_bwd(do, q, k, v, out, lse, dk=k),
            lambda: ua.swa_bwd(do, q, k, v, out, lse, dk=out[:, :, :2], dv=out[:, :, :2])]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    assert math.isfinite(lse[0, 0, 0].item())
