"""Results over shards of the keys, joined: merges, updates, sums and deltas for the types and head sizes of sliding-window attention."""
import math

import pytest
import torch

import ultraattn_amd as ua
from tests.swa_util import DEV, Reference, inputs, visible

pytestmark = pytest.mark.gpu
KINDS = [(torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 64), (torch.bfloat16, 128)]
NEW = KINDS[:3]
E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def parts_of(dtype, dim, n=4, q_len=512, k_len=1024, heads=4, kv_heads=2):
    q, k, v, do = inputs(1, q_len, k_len, heads, kv_heads, dim, dtype)
    how = dict(window=(300, 0), sinks=10, q_start=k_len - q_len)
    step = k_len // n
    chunks = [(i, k[:, i:i + step].contiguous(), v[:, i:i + step].contiguous()) for i in range(0, k_len, step)]
    return q, k, v, do, how, chunks, [ua.swa_fwd(q, kc, vc, k_start=i, **how) for i, kc, vc in chunks]


@pytest.mark.parametrize("dtype,dim", KINDS)
def test_shards_merge_to_the_whole(dtype, dim):
    q, k, v, _, how, _, parts = parts_of(dtype, dim)
    ref = Reference(q, k, v, visible(512, 1024, (300, 0), 10, 512))
    ref.out_bound = 2 * ref.out_bound                                # every part's rows are rounded, and their merge
    out, lse = ua.merge_partials([p[0] for p in parts], [p[1] for p in parts])
    assert out.dtype == dtype
    ref.check(out=out, lse=lse)
    run = (None, None)
    for p in parts:
        run = ua.update_out_and_lse(*run, *p)
    assert run[0].dtype == torch.float32                              # as the reference's running output
    ref.lse_bound = ref.lse_bound + 4 * 8 * E * ref.lse.abs().clamp_min(1).nan_to_num(posinf=1, neginf=1)
    ref.check(out=run[0].to(dtype), lse=run[1].squeeze(-1).transpose(1, 2))


@pytest.mark.parametrize("dtype,dim", KINDS)
def test_shards_add_up(dtype, dim):
    """A ring's step: global statistics, partial gradients of the queries added, keys' gradients of their own shard."""
    q, k, v, do, how, chunks, parts = parts_of(dtype, dim)
    out, lse = ua.merge_partials([p[0] for p in parts], [p[1] for p in parts])
    delta = ua.softmax_delta(out, do)
    grads = [ua.swa_bwd(do, q, kc, vc, None, lse, k_start=i, softmax_d=delta, **how) for i, kc, vc in chunks]
    ref = Reference(q, k, v, visible(512, 1024, (300, 0), 10, 512), dout=do)
    for b in ("dq_bound", "dk_bound", "dv_bound"):
        setattr(ref, b, 6 * getattr(ref, b))                          # rows rounded in every part and merged: twice the forward's; four roundings of dq
    ref.check(dq=ua.grad_sum([g[0] for g in grads]), dk=torch.cat([g[1] for g in grads], 1), dv=torch.cat([g[2] for g in grads], 1))


def random_parts(n, shape, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    outs = [torch.randn(*shape, generator=g, device=DEV).to(dtype) for _ in range(n)]
    lses = [torch.rand(shape[0], shape[2], shape[1], generator=g, device=DEV) * 20 - 10 for _ in range(n)]
    return outs, lses


def exact_merge(outs, lses):
    l = torch.stack([x.double() for x in lses])
    total = torch.logsumexp(l, 0)
    w = torch.exp(l - torch.where(total == -math.inf, torch.zeros_like(total), total)).transpose(2, 3)[..., None]
    rows = [torch.where(x > 0, x * o.double(), torch.zeros_like(o.double())) for x, o in zip(w, outs)]
    return sum(rows), sum(r.abs() for r in rows), total


# a weight is off by 4 e |lse_p - LSE| (two roundings of the exponent, each of up to 2 |x| e) + 4 e, |lse_p - LSE| <= 24; sums of 16 terms 16 e
WEIGHTS = (4 * 24 + 4 + 16) * E


@pytest.mark.parametrize("dtype,dim", NEW)
@pytest.mark.parametrize("n,shape", [(1, (1, 1, 1)), (2, (2, 7, 3)), (5, (1, 300, 9)), (16, (3, 33, 300))])
def test_merge_of_any_parts(dtype, dim, n, shape):
    outs, lses = random_parts(n, (*shape, dim), dtype, n)
    for i in range(n):                                                # rows without keys hold anything, among them all parts' of one row
        lses[i][:, :, i::5] = -math.inf
        outs[i].transpose(1, 2)[lses[i] == -math.inf] = math.nan
        lses[i][0, 0, 0] = -math.inf
    want, size, total = exact_merge(outs, lses)
    out, lse = ua.merge_partials(outs, lses)
    assert ((out.double() - want).abs() <= half_step(dtype) * want.abs() + WEIGHTS * size + 2.0 ** -25).all()
    none = total == -math.inf
    assert (lse[none] == -math.inf).all() and none.any() and ((lse - total).abs()[~none] <= (16 + 8 * 24) * E).all()
    given = torch.full_like(out, 7), torch.empty_like(lse)
    got = ua.merge_partials(outs, lses, out=given[0], lse=given[1])
    assert got[0] is given[0] and got[1] is given[1] and torch.equal(got[0], out) and torch.equal(got[1], lse)
    first = outs[0].clone(), lses[0].clone()
    got = ua.merge_partials([first[0], *outs[1:]], [first[1], *lses[1:]], out=first[0], lse=first[1])       # in place of the first part
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)


def test_merge_keeps_nan():
    outs, lses = random_parts(3, (1, 40, 2, 64), torch.float16)
    outs[1][0, 5, 1] = math.nan
    lses[2][0, 0, 7] = math.nan
    out, lse = ua.merge_partials(outs, lses)
    assert torch.isnan(out[0, 5, 1]).all() and torch.isnan(out[0, 7, 0]).all() and torch.isnan(lse[0, 0, 7])
    bad = torch.zeros(1, 40, 2, dtype=torch.bool, device=DEV)
    bad[0, 5, 1] = bad[0, 7, 0] = True
    assert torch.isfinite(out[~bad]).all()


@pytest.mark.parametrize("dtype,dim", NEW)
def test_update_of_slices_in_place(dtype, dim):
    (out, blk), (lse, blk_lse) = random_parts(2, (2, 50, 6, dim), dtype, 4)
    lse[0, 0, 30], blk_lse[0, 0, 31], lse[1, 2, 40], blk_lse[1, 2, 40] = (-math.inf,) * 4
    part, part_lse = blk[:, 20:].contiguous(), blk_lse[..., 20:].contiguous()
    want, size, total = exact_merge([out[:, 20:], part], [lse[..., 20:], part_lse])
    run, run_lse = out.clone(), lse.transpose(1, 2).unsqueeze(-1).contiguous()
    got, got_lse = ua.update_out_and_lse(run, run_lse, part, part_lse, slice_=(slice(None), slice(20, None)))
    assert got is run and got_lse is run_lse and got.dtype == dtype
    assert torch.equal(run[:, :20], out[:, :20]) and torch.equal(run_lse[:, :20, :, 0].transpose(1, 2), lse[..., :20])
    assert ((run[:, 20:].double() - want).abs() <= half_step(dtype) * want.abs() + WEIGHTS * size + 2.0 ** -25).all()
    now = run_lse[:, 20:, :, 0].transpose(1, 2)
    some = total > -math.inf
    assert (now[~some] == -math.inf).all() and ((now - total).abs()[some] <= (16 + 8 * 24) * E).all()
    f32, _ = ua.update_out_and_lse(out[:, 20:], lse.transpose(1, 2).unsqueeze(-1)[:, 20:], part, part_lse)       # strided views into new fp32 rows
    assert f32.dtype == torch.float32 and ((f32.double() - want).abs() <= WEIGHTS * size + 2.0 ** -149).all()
    again, _ = ua.update_out_and_lse(f32, lse.transpose(1, 2).unsqueeze(-1)[:, 20:].contiguous(), f32, part_lse)  # fp32 on both sides
    assert ((again.double() - want).abs() <= 3 * WEIGHTS * (size + want.abs())).all()


@pytest.mark.parametrize("dtype,dim", NEW)
@pytest.mark.parametrize("n", [1, 3, 16])
def test_sums(dtype, dim, n):
    parts, _ = random_parts(n, (2, 31, 5, dim), dtype, n)
    want, size = sum(p.double() for p in parts) * 0.5, sum(p.double().abs() for p in parts)
    room = torch.full((2, 40, 10, dim), 7.0, dtype=dtype, device=DEV)
    out = room[:, 4:35, ::2]
    got = ua.grad_sum(parts, out=out, scale=0.5)
    assert got is out and ((got.double() - want).abs() <= half_step(dtype) * want.abs() + 17 * E * size + 2.0 ** -25).all()
    assert (room[:, :4] == 7).all() and (room[:, 35:] == 7).all() and (room[:, :, 1::2] == 7).all()
    wide = [p.float() / 3 for p in parts]
    want = sum(p.double() for p in wide)
    for into in (None, torch.empty(2, 31, 5, dim, dtype=torch.float16, device=DEV)):
        got = ua.grad_sum(wide, out=into)
        assert got.dtype == (torch.bfloat16 if into is None else torch.float16)
        assert ((got.double() - want).abs() <= half_step(got.dtype) * want.abs() + 17 * E * size + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype,dim", NEW)
def test_delta(dtype, dim):
    (wide, do), _ = random_parts(2, (2, 37, 10, dim), dtype, 5)
    out, do = wide[:, :, ::2], do[:, :, :5]
    want, size = (out.double() * do.double()).sum(-1).transpose(1, 2), (out.double() * do.double()).abs().sum(-1).transpose(1, 2)
    given = torch.empty(2, 5, 37, device=DEV)
    assert ua.softmax_delta(out, do, given) is given
    assert ((given - want).abs() <= (dim + 4) * E * size).all() and torch.equal(ua.softmax_delta(out, do), given)


def test_captured_on_another_stream():
    q, k, v, do, how, chunks, parts = parts_of(torch.float16, 64)
    outs, lses = [p[0] for p in parts], [p[1] for p in parts]
    want = ua.merge_partials(outs, lses)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = ua.merge_partials(outs, lses)
        delta = ua.softmax_delta(res[0], do)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1]) and torch.equal(delta, ua.softmax_delta(want[0], do))
        res[0].zero_()


def test_nothing_to_join():
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        outs, lses = random_parts(2, shape, torch.float16)
        out, lse = ua.merge_partials(outs, lses)
        assert out.shape == shape and lse.shape == (shape[0], 2, shape[1])
        assert ua.grad_sum(outs).shape == shape and ua.softmax_delta(outs[0], outs[1]).numel() == 0
        assert ua.update_out_and_lse(outs[0], lses[0].transpose(1, 2).unsqueeze(-1), outs[1], lses[1])[0].shape == shape


def test_refusals():
    outs, lses = random_parts(2, (1, 16, 2, 64), torch.float16)
    a, b = outs
    wide = random_parts(1, (1, 16, 2, 128), torch.float16)[0][0]
    run = lses[0].transpose(1, 2).unsqueeze(-1).contiguous()
    bad = [lambda: ua.merge_partials([a, b.bfloat16()], lses), lambda: ua.merge_partials([a, wide], lses), lambda: ua.merge_partials([a, b[:, :8]], lses),
           lambda: ua.merge_partials(outs, [lses[0], lses[1].double()]), lambda: ua.merge_partials(outs, lses, out=a.bfloat16()), lambda: ua.merge_partials([a.cpu(), b], lses),
           lambda: ua.merge_partials([a] * 17, [lses[0]] * 17), lambda: ua.merge_partials([a, b], [lses[0].cpu(), lses[1]]),
           lambda: ua.merge_partials([a[..., :32].contiguous()] * 2, lses), lambda: ua.merge_partials([a.float(), b.float()], lses),
           lambda: ua.grad_sum([a, b.bfloat16()]), lambda: ua.grad_sum([a, b], out=a.bfloat16()), lambda: ua.grad_sum([a[..., :32].contiguous()]),
           lambda: ua.grad_sum([a, b], out=torch.empty(1, 16, 2, 128, dtype=torch.float16, device=DEV)), lambda: ua.grad_sum([a, b], out=a.float()),
           lambda: ua.softmax_delta(a, b.bfloat16()), lambda: ua.softmax_delta(a, wide), lambda: ua.softmax_delta(a, b, torch.empty(1, 16, 2, device=DEV)),
           lambda: ua.update_out_and_lse(a, run, b.bfloat16(), lses[1]), lambda: ua.update_out_and_lse(a, run, wide, lses[1]),
           lambda: ua.update_out_and_lse(a, run, b, lses[1].cpu()), lambda: ua.update_out_and_lse(a, run.half(), b, lses[1])]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was taken")


def test_results_over_operands_are_refused():
    (a, b), (la, lb) = random_parts(2, (1, 16, 2, 64), torch.float16)
    run = la.transpose(1, 2).unsqueeze(-1).contiguous()
    flat = torch.zeros(3 * a.numel(), dtype=torch.float16, device=DEV)
    view = lambda at, like=a: flat[at:at + like.numel()].view(like.shape)  # noqa: E731
    stat = lambda at: flat[at:at + 2 * la.numel()].view(torch.float32).view(la.shape)  # noqa: E731
    wide = flat[:2 * a.numel()].view(torch.float32).view(a.shape)
    bad = [lambda: ua.merge_partials([view(0), b], [la, lb], out=view(64)), lambda: ua.merge_partials([a, b], [la, lb], out=view(0), lse=stat(128)),
           lambda: ua.merge_partials([a, b], [stat(0), lb], lse=stat(2)), lambda: ua.merge_partials([view(0), b], [la, lb], lse=stat(128)),
           lambda: ua.merge_partials([a, b], [stat(0), lb], out=view(0)), lambda: ua.grad_sum([view(0), b], out=view(64)), lambda: ua.grad_sum([wide], out=view(0)),
           lambda: ua.grad_sum([a, b], out=a[:, :1].expand_as(a)), lambda: ua.softmax_delta(view(0), b, stat(0)),
           lambda: ua.update_out_and_lse(view(0), run, view(64), lb, slice_=(slice(None),)), lambda: ua.update_out_and_lse(a[:, :1].expand_as(a), run, b, lb, slice_=(slice(None),)),
           lambda: ua.update_out_and_lse(a, run[:, :1].expand_as(run), b, lb, slice_=(slice(None),)), lambda: ua.update_out_and_lse(a, run, a, lb, slice_=(slice(None),))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError, match="overlap"):
            call()
            pytest.fail(f"call {i} was taken")
    beside = ua.merge_partials([view(0), view(a.numel())], [la, lb], out=view(2 * a.numel()))
    assert torch.equal(beside[0], ua.merge_partials([view(0).clone(), view(a.numel()).clone()], [la, lb])[0])
    same = a.clone()
    assert torch.equal(ua.grad_sum([same, b], out=same), ua.grad_sum([a, b]))
