"""A process whose first call of each row operator is inside a graph capture:
the calls set up nothing that a capture forbids.  (A process of its own, since
any earlier call would have loaded the kernels.)"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch
import pz_sampling as pz
torch.manual_seed(1)
x = torch.randn(4, 50000, device="cuda")
o, g1, g2 = (torch.empty_like(x) for _ in range(3))
ids = torch.arange(12, device="cuda", dtype=torch.int32).view(4, 3).contiguous()
t = torch.randn(4, 3, device="cuda")
loss, loss2 = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
st = torch.empty(4, 4, device="cuda")
h = torch.randn(200, 64, device="cuda")
w = torch.randint(-9, 9, (1000, 64), device="cuda", dtype=torch.int8)
ws = torch.ones(1000, device="cuda")
q = torch.empty(200, 64, dtype=torch.int8, device="cuda")
qs = torch.empty(200, device="cuda")
few, many = torch.empty(3, 1000, device="cuda"), torch.empty(200, 1000, device="cuda")


def calls():
    pz.process_logits(x, o)
    pz.distill_forward(x, ids, t, loss, st)
    pz.distill_backward(x, ids, t, st, g1)
    pz.distill_loss_grad(x, ids, t, loss2, g2)
    pz.lm_head_i8(h, w, ws, many, q, qs)
    pz.lm_head_i8(h[:3], w, ws, few, q[:3], qs[:3])


torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
g.replay()
torch.cuda.synchronize()
first = [v.clone() for v in (o, loss, g1, loss2, g2, many, few)]
calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(first, (o, loss, g1, loss2, g2, many, few)))
assert torch.equal(o, x) and torch.equal(many[:3], few)
print("captured first")
"""


def test_first_calls_inside_a_capture(cuda):
    lib = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-zero_b200")
    r = subprocess.run([sys.executable, "-c", SCRIPT, lib], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]
