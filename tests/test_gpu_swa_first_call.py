"""The very first calls of a process, captured into a graph, replayed and compared with eager calls."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
import ultraattn_amd as ua
mk = lambda s, h: torch.randn(2, s, h, 64, device="cuda").to(torch.float16)
q, k, v, do = mk(700, 4), mk(700, 2), mk(700, 2), mk(700, 4)
f = ua.rope_freqs(64, device="cuda")[0]
tq, tk, tv = mk(1, 4), mk(1, 2), mk(1, 2)
kc, vc = torch.zeros(2, 2, 900, 2, 64, dtype=torch.float16, device="cuda")
lens = torch.tensor([5, 801], dtype=torch.int32, device="cuda")

def everything():
    qr, kr = ua.rope_fwd(q, k, f)
    out, lse = ua.swa_fwd(qr, kr, v, (200, 0), 4)
    dq, dk, dv = ua.swa_bwd(do, qr, kr, v, out, lse, (200, 0), 4)
    dq, dk = ua.rope_bwd(dq, dk, f, dq_out=dq, dk_out=dk)
    turned = ua.rope_append(tq, tk, tv, kc, vc, lens, f)
    return (out, lse, dq, dk, dv, turned, *ua.swa_decode(turned, kc, vc, lens, 200, 4))

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = everything()
for _ in range(3):
    q.normal_(); tk.normal_()
    graph.replay()
    torch.cuda.synchronize()
    kept = [x.clone() for x in got]
    for x, y in zip(kept, everything()):
        assert torch.equal(x, y)
print("captured first")
"""


def test_first_calls_of_a_process_are_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr
