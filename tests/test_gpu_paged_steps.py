"""A paged cache as a serving program runs it: a prompt, drafts verified as trees, the accepted branches kept, one captured step replayed, against causal attention of what
was accepted, in 64 bits (bounds: swa_util)."""
import pytest
import torch

import ultraattn_amd as ua
from tests.paged_util import branch, trees
from tests.swa_util import DEV, Reference, inputs

pytestmark = pytest.mark.gpu


def test_drafts_verified_and_kept():
    batch, heads, kv_heads, dim, page, tokens, prompt, layers, window, sinks = 3, 8, 2, 64, 16, 13, 37, 2, 40, 2
    dtype, room, keep = torch.bfloat16, 160, 6
    freqs, scale = ua.rope_freqs(48, device=DEV)
    kp, vp = torch.full((2, layers, 40, page, kv_heads, dim), torch.nan, dtype=dtype, device=DEV)
    table = torch.randperm(40, device=DEV)[:batch * (room // page)].reshape(batch, -1).to(torch.int32)
    lens = torch.full((batch,), prompt, dtype=torch.int32, device=DEV)
    kept_q, kept_k, kept_v = ([[[] for _ in range(batch)] for _ in range(layers)] for _ in range(3))
    kept_out, kept_lse = ([[[] for _ in range(batch)] for _ in range(layers)] for _ in range(2))

    for layer in range(layers):                                                     # the prompt
        q, k, v, _ = inputs(batch, prompt, prompt, heads, kv_heads, dim, dtype, 100 + layer)
        turned = ua.paged_append(q, k, v, kp[layer], vp[layer], table, lens, freqs, scale=scale)
        out, lse = ua.paged_decode(turned, kp[layer], vp[layer], table, lens, window=window, sinks=sinks)
        for b in range(batch):
            for store, x in ((kept_q, q), (kept_k, k), (kept_v, v), (kept_out, out), (kept_lse, lse.transpose(1, 2))):
                store[layer][b].append(x[b])

    # the step's own buffers, and the step, captured before anything is in them
    n_new, n_kept = (torch.zeros(batch, dtype=torch.int32, device=DEV) for _ in range(2))
    parents, path = torch.full((batch, tokens), -1, dtype=torch.int32, device=DEV), torch.zeros(batch, keep, dtype=torch.int32, device=DEV)
    sq = torch.zeros(layers, batch, tokens, heads, dim, dtype=dtype, device=DEV)
    sk, sv = (torch.zeros(layers, batch, tokens, kv_heads, dim, dtype=dtype, device=DEV) for _ in range(2))

    def verify():
        lens.add_(n_new)
        return [ua.paged_decode(ua.paged_append(sq[n], sk[n], sv[n], kp[n], vp[n], table, lens, freqs, n_new, parents, scale=scale), kp[n], vp[n], table, lens, n_new,
                                parents, window, sinks) for n in range(layers)]

    def accept():
        ua.paged_keep(kp, vp, table, lens, n_new, path, n_kept)
        lens.add_(n_kept - n_new)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0], stream=stream):
        results = verify()
    with torch.cuda.graph(graphs[1], stream=stream):
        accept()

    g = torch.Generator().manual_seed(7)
    for step in range(8):
        tree = trees(batch, tokens, step, (0.1, 1.0, 0.4)[step % 3])
        count = [tokens, 1 + step, 5 + step % 4]
        parents.copy_(tree)
        n_new.copy_(torch.tensor(count, dtype=torch.int32))
        for n in range(layers):
            q, k, v, _ = inputs(batch, tokens, tokens, heads, kv_heads, dim, dtype, 10 * step + n)
            for x, y in ((sq[n], q), (sk[n], k), (sv[n], v)):
                x.copy_(y)
        base = lens.tolist()
        graphs[0].replay()
        got = [(o.clone(), l.clone()) for o, l in results]
        torch.cuda.synchronize()
        lens.sub_(n_new)                                                            # the same step once more, without the graph
        again = verify()
        assert all(torch.equal(a[0], c[0]) and torch.equal(a[1], c[1]) for a, c in zip(again, got))
        for b in range(batch):
            leaf = int(torch.randint(0, count[b], (1,), generator=g))
            way = branch(tree[b].tolist(), leaf)[::-1][:keep]
            path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
            n_kept[b] = len(way)
            for n in range(layers):
                for store, x in ((kept_q, sq[n]), (kept_k, sk[n]), (kept_v, sv[n]), (kept_out, got[n][0]), (kept_lse, got[n][1].transpose(1, 2))):
                    store[n][b].append(x[b, way])
        graphs[1].replay()
        torch.cuda.synchronize()
        assert lens.tolist() == [x + y for x, y in zip(base, n_kept.tolist())]

    for n in range(layers):
        for b in range(batch):
            q, k, v, out, lse = (torch.cat(x[n][b])[None] for x in (kept_q, kept_k, kept_v, kept_out, kept_lse))
            qr, kr = ua.rope_fwd(q, k, freqs, scale=scale)
            total = q.shape[1]
            rows = torch.arange(total, device=DEV)
            at = table[b].long()[rows // page], rows % page
            assert total == int(lens[b]) and torch.equal(kp[n][at], kr[0]) and torch.equal(vp[n][at], v[0])
            back = rows[:, None] - rows
            seen = (back >= 0) & ((back <= window) | (rows < sinks))
            Reference(qr, kr, v, seen).check(out=out, lse=lse.transpose(1, 2))


@pytest.mark.parametrize("tree", [False, True])
def test_first_calls_captured_and_replayed(tree):
    """Replays over new lengths, tables and trees, with eager work between them, equal the eager calls."""
    batch, tokens, heads, kv_heads, dim, page, most = 2, 9, 8, 2, 128, 16, 64
    kp, vp = (torch.randn(batch * most, page, kv_heads, dim, device=DEV).to(torch.float16) for _ in range(2))
    q = torch.randn(batch, tokens, heads, dim, device=DEV).to(torch.float16)
    lens, n_new = torch.full((batch,), tokens, dtype=torch.int32, device=DEV), torch.full((batch,), tokens, dtype=torch.int32, device=DEV)
    table = torch.zeros(batch, most, dtype=torch.int32, device=DEV)
    parents = torch.full((batch, tokens), -1, dtype=torch.int32, device=DEV) if tree else None
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, results = [], []
    for _ in range(2):                                                              # two graphs: their workspaces are apart
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            results.append(ua.paged_decode(q, kp, vp, table, lens, n_new, parents))
        graphs.append(graph)
    for i in range(5):
        g = torch.Generator().manual_seed(i)
        table.copy_(torch.randperm(batch * most, generator=g).reshape(batch, most).to(torch.int32))
        lens.copy_(torch.randint(tokens, most * page + 1, (batch,), generator=g).to(torch.int32))
        n_new.copy_(torch.randint(0, tokens + 1, (batch,), generator=g).to(torch.int32))
        if tree:
            parents.copy_(trees(batch, tokens, i))
        want = ua.paged_decode(q, kp, vp, table, lens, n_new, parents)
        torch.cuda.synchronize()
        for graph, got in zip(graphs, results):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
