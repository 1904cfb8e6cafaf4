"""Sliding-window attention, forward, against its definition in 64 bits (bounds: swa_util)."""
import math

import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, Reference, inputs, visible

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def run(q, k, v, window=(-1, 0), sinks=0, q_start=None, k_start=0, scale=None, **more):
    out, lse = ua.swa_fwd(q, k, v, window, sinks, scale, q_start, k_start, **more)
    Reference(q, k, v, visible(q.shape[1], k.shape[1], window, sinks, q_start, k_start), scale).check(out=out, lse=lse)
    return out, lse


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seq_q,seq_k", [(1, 1), (1, 65), (31, 64), (64, 63), (100, 100), (128, 128), (129, 257), (300, 1000), (513, 511)])
@pytest.mark.parametrize("window,sinks", [((-1, 0), 0), ((20, 0), 3), ((64, 7), 65), ((0, 0), 0), ((130, -1), 1), ((-1, -1), 0)])
def test_lengths_and_windows(dtype, dim, seq_q, seq_k, window, sinks):
    q, k, v, _ = inputs(2, seq_q, seq_k, 4, 2, dim, dtype, seq_q + seq_k)
    run(q, k, v, window, sinks)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (7, 1), (6, 3), (16, 2)])
def test_shared_key_heads(heads, kv_heads):
    q, k, v, _ = inputs(1, 200, 333, heads, kv_heads, 64, torch.bfloat16)
    run(q, k, v, (70, 0), 2)


# the keys far before, far behind, half beside the queries; a shard that holds the end of the sinks; positions beyond 32 bits
@pytest.mark.parametrize("q_start,k_start", [(5000, 0), (-1000, 0), (150, 0), (400, 300), (390, 10), (2 ** 40 + 100, 2 ** 40), (2 ** 60, -2 ** 60), (-3, 0)])
@pytest.mark.parametrize("window,sinks", [((100, 0), 0), ((100, 0), 20), ((100, 50), 20), ((-1, 0), 0), ((2 ** 40, 2 ** 35), 4)])
def test_shards(q_start, k_start, window, sinks):
    q, k, v, _ = inputs(1, 260, 300, 2, 1, 128, torch.bfloat16)
    run(q, k, v, window, sinks, q_start, k_start)


def test_rows_and_keys_that_nothing_sees():
    q, k, v, _ = inputs(2, 300, 200, 3, 3, 64, torch.float16)
    out, lse = run(q, k, v, (10, 0), 0, q_start=100)                # rows from 110 on see nothing
    assert (out[:, 110:] == 0).all() and (lse[..., 110:] == -math.inf).all() and torch.isfinite(lse[..., :110]).all()
    out, lse = run(q, k, v, (10, 0), 0, q_start=-50)                # nor do the first 50
    assert (lse[..., :50] == -math.inf).all() and torch.isfinite(lse[..., 50:260]).all()


def test_no_keys_no_rows_no_batch():
    q, k, v, _ = inputs(2, 5, 0, 4, 2, 64, torch.bfloat16)
    out, lse = ua.swa_fwd(q, k, v, (3, 0))
    assert (out == 0).all() and (lse == -math.inf).all()
    for b, s in ((0, 7), (2, 0)):
        q, k, v, _ = inputs(b, s, 9, 4, 2, 64, torch.bfloat16)
        out, lse = ua.swa_fwd(q, k, v, (3, 0))
        assert out.shape == q.shape and lse.shape == (b, 4, s)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_grow_along_the_row_and_rows_that_begin_low(dtype, dim):
    """References have to be raised, again and again; and a first block far below zero must not vanish."""
    q, k, v, _ = inputs(1, 256, 1500, 2, 2, dim, dtype, std=0.5)
    grow = torch.linspace(-6, 6, 1500, device=DEV)[None, :, None, None] * torch.ones(dim, device=DEV) / dim ** 0.5
    k = (k.float() * 0.1 + grow * 2).to(dtype)
    q = (q.float() * 0.1 + 3.0).to(dtype)
    for window, start in (((-1, 0), None), ((700, 0), None), ((-1, -1), None), ((40, 0), 0)):
        run(q, k, v, window, 5, start)
        run(q, k.flip(1), v, window, 5, start)


def test_infinite_scores_and_nan():
    q, k, v, _ = inputs(1, 130, 300, 1, 1, 64, torch.bfloat16)
    k[0, 10, 0] = torch.nan                                         # keys that rows from 100 on do not see, nor their tile
    v[0, 11, 0] = torch.inf
    out, lse = ua.swa_fwd(q, k, v, (60, 0), q_start=150)
    ref = Reference(q, torch.nan_to_num(k), torch.nan_to_num(v, posinf=1.0), visible(130, 300, (60, 0), q_start=150))
    ref.check(out=out, lse=lse)
    out, lse = ua.swa_fwd(q, k, v, (60, 0), q_start=0)
    assert torch.isnan(out[0, 10:71]).all() and torch.isnan(lse[0, 0, 10:71]).all()        # rows that see it say so
    assert torch.isfinite(lse[0, 0, :10]).all() and torch.isfinite(lse[0, 0, 71:]).all()


def test_views_strides_broadcast_and_given_results():
    qkv = inputs(2, 150, 150, 8, 8, 64, torch.float16)[0]
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]          # one projection's output
    out, lse = run(q, k, v, (33, 0), 2)
    room = torch.full((2, 160, 4, 64), 7.0, dtype=torch.float16, device=DEV)
    stat = torch.empty_like(lse)
    got = ua.swa_fwd(q, k, v, (33, 0), 2, out=room[:, 3:153], lse=stat)
    assert got[1] is stat and torch.equal(room[:, 3:153], out) and torch.equal(stat, lse)
    assert (room[:, :3] == 7).all() and (room[:, 153:] == 7).all()
    q, k = inputs(2, 4, 2, 150, 150, 64, torch.float16)[:2]         # [B, H, S, D] tensors
    run(q.transpose(1, 2), k.transpose(1, 2), k.transpose(1, 2), (33, 0), 2)
    one = inputs(2, 150, 150, 1, 1, 64, torch.float16)
    run(inputs(2, 150, 150, 6, 1, 64, torch.float16, 5)[0], one[1].expand(2, 150, 6, 64), one[2].expand(2, 150, 6, 64), (33, 0), 2)
    same = inputs(1, 150, 150, 2, 2, 64, torch.float16)
    run(same[0].expand(3, 150, 2, 64), same[1].expand(3, 150, 2, 64), same[2].expand(3, 150, 2, 64), (33, 0), 2)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("seq_q,seq_k,window,sinks", [(3, 5000, (-1, 0), 0), (200, 4100, (3000, 0), 100), (130, 2000, (-1, -1), 0), (1, 1025, (-1, 0), 0)])
def test_few_rows_and_many_keys(dtype, dim, seq_q, seq_k, window, sinks):
    """Cut into parts; one head or a sequence of its own gives the same as among others up to rounding."""
    q, k, v, _ = inputs(2, seq_q, seq_k, 4, 2, dim, dtype)
    run(q, k, v, window, sinks)
    run(q, k, v, window, sinks, q_start=40)                         # parts in which some rows see nothing


def test_out_in_place_of_q():
    for seq_k in (200, 5000):                                        # whole, and cut into parts
        q, k, v, _ = inputs(1, 150, seq_k, 2, 2, 64, torch.bfloat16)
        want = ua.swa_fwd(q, k, v)[0]
        x = q.clone()
        assert ua.swa_fwd(x, k, v, out=x)[0] is x and torch.equal(x, want)


def test_larger_grids():
    q, k, v, _ = inputs(3, 1111, 1111, 24, 8, 128, torch.bfloat16)
    run(q, k, v, (256, 0), 4)


def test_shards_merge_to_the_whole():
    q, k, v, _ = inputs(1, 512, 1024, 4, 4, 128, torch.bfloat16)
    how = dict(window=(300, 0), sinks=10, q_start=512)
    parts = [ua.swa_fwd(q, k[:, i:i + 256].contiguous(), v[:, i:i + 256].contiguous(), k_start=i, **how) for i in range(0, 1024, 256)]
    out, lse = ua.merge_partials([p[0] for p in parts], [p[1] for p in parts])
    ref = Reference(q, k, v, visible(512, 1024, (300, 0), 10, 512))
    ref.out_bound = 2 * ref.out_bound                                # every part's rows are rounded, and their merge
    ref.check(out=out, lse=lse)


def test_captured_other_stream_and_two_graphs():
    """Replays in turn and on two streams at once: cut calls have workspaces of their own."""
    q, k, v, _ = inputs(1, 100, 4000, 2, 2, 64, torch.bfloat16)
    q2, k2, v2, _ = inputs(1, 100, 4000, 2, 2, 64, torch.bfloat16, 1)
    want, want2 = run(q, k, v, (-1, 0)), run(q2, k2, v2, (-1, 0))
    graphs = []
    for args in ((q, k, v), (q2, k2, v2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = ua.swa_fwd(*args)
        graphs.append((g, res))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (g, _res), s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_g, res), w in zip(graphs, (want, want2)):
            assert torch.equal(res[0], w[0]) and torch.equal(res[1], w[1])
            res[0].zero_()
        assert torch.equal(ua.swa_fwd(q, k, v)[0], want[0])
    with torch.cuda.stream(streams[0]):
        got = ua.swa_fwd(q, k, v)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0])


def test_refusals():
    q, k, v, _ = inputs(2, 16, 16, 4, 2, 64, torch.bfloat16)
    wide = inputs(2, 16, 16, 4, 2, 128, torch.bfloat16)[1]
    bad = [lambda: ua.swa_fwd(q, k, v[:, :8]), lambda: ua.swa_fwd(q, k[:1], v[:1]), lambda: ua.swa_fwd(q, k.half(), v), lambda: ua.swa_fwd(q.float(), k.float(), v.float()),
           lambda: ua.swa_fwd(q, wide, wide), lambda: ua.swa_fwd(q[:, :, :3], k, v), lambda: ua.swa_fwd(q[..., :32], k[..., :32], v[..., :32]),
           lambda: ua.swa_fwd(q, k, v, (-2, 0)), lambda: ua.swa_fwd(q, k, v, (0, -2)), lambda: ua.swa_fwd(q, k, v, (0, 0), -1),
           lambda: ua.swa_fwd(q, k, v, softmax_scale=0.0), lambda: ua.swa_fwd(q, k, v, softmax_scale=math.nan), lambda: ua.swa_fwd(q, k, v, q_start=2 ** 61),
           lambda: ua.swa_fwd(q, k, v, out=q[:, :8]), lambda: ua.swa_fwd(q, k, v, out=q[:, :, :1].expand(2, 16, 4, 64)),
           lambda: ua.swa_fwd(q, k, v, lse=torch.empty(2, 16, 4, device=DEV)), lambda: ua.swa_fwd(q, k, v, lse=torch.empty(2, 4, 16)),
           lambda: ua.swa_fwd(q, k.cpu(), v), lambda: ua.swa_fwd(q.cpu(), k.cpu(), v.cpu()), lambda: ua.swa_fwd(q[:, :, 0], k, v),
           lambda: ua.swa_fwd(q.transpose(2, 3), k, v), lambda: ua.swa_fwd(q, k[:, :, :0], v[:, :, :0])]
    bad += [lambda: ua.swa_fwd(q, k.repeat(1, 1, 2, 1), q, out=q)]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was taken")
    flat = torch.zeros(2 * 16 * 4 * 64 + 8, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="aligned"):
        ua.swa_fwd(flat[1:1 + q.numel()].view_as(q), k, v)
    rows = torch.zeros(2, 16, 4 * 68, dtype=torch.bfloat16, device=DEV).unflatten(2, (4, 68))[..., :64]
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ua.swa_fwd(rows, k, v)
