"""Operators whose first call of a process happens inside a stream capture, and
calls from several threads at once (each in a process of its own, so that
nothing has been called before)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SETUP = """
import sys, threading
sys.path.insert(0, sys.argv[1])
import torch
from gotransformers_b200 import moe
torch.manual_seed(1)
bf = torch.bfloat16
x = torch.randn(500, 256, device="cuda").to(bf)
dy = torch.randn(500, 264, device="cuda").to(bf)
w3 = torch.randn(3, 264, 256, device="cuda").to(bf)
w, b = torch.randn(256, device="cuda"), torch.randn(256, device="cuda")
counts = torch.tensor([200, 0, 300], device="cuda")
def everything(x=x, dy=dy):
    y, mean, rstd = moe.layer_norm(x, w, b)
    back = moe.layer_norm_backward(x, x, mean, rstd, w, residual_gradients=y)
    d = moe.dropout(x, 0.3, 5, 1, residual=y)
    e = moe.dropout_backward(x, 0.3, 5, 1)
    p = moe.grouped_product(x, w3, counts)
    q = moe.grouped_product_input_gradients(dy, w3, counts)
    r = moe.grouped_product_weight_gradients(dy, x, counts, dtype=torch.float32)
    s = moe.grouped_product(x.float(), w3.float(), counts)
    return (y, mean, rstd) + back + (d, e, p, q, r, s)
"""

CAPTURED = SETUP + """
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = everything()
graph.replay()
torch.cuda.synchronize()
ref = everything()
assert all(torch.equal(a, b) for a, b in zip(out, ref))
moe.check_operators()
print("done")
"""

THREADS = SETUP + """
results, errors = {}, []
def work(i):
    try:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                results[i] = everything()
        s.synchronize()
    except Exception as e:
        errors.append(e)
torch.cuda.synchronize()
threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not errors, errors
ref = everything()
torch.cuda.synchronize()
for r in results.values():
    assert all(torch.equal(a, b) for a, b in zip(r, ref))
moe.check_operators()
print("done")
"""


@pytest.mark.parametrize("script", [CAPTURED, THREADS], ids=["captured", "threads"])
def test_first_calls(script):
    r = subprocess.run([sys.executable, "-c", script, ROOT], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]
