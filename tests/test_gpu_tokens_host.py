"""Host side of the token-table and dropout operators on a GPU: threads,
streams, autograd's bookkeeping."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_first_calls_of_several_threads(cuda):
    """Each thread's first call is among the process's first ones; a token
    outside the table is reported to one of them."""
    code = """
import threading
import torch
from t3st_b200 import kernels, nn

table = torch.randn(50, 64, device="cuda")
tok = torch.arange(40, device="cuda")
torch.cuda.synchronize()
start, outs = threading.Barrier(8), [None] * 8

def work(i):
    start.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        w = table.clone().requires_grad_()
        for _ in range(20):
            y = nn.embedding(tok, w, p=0.2, seed=i)
            y.backward(torch.ones_like(y))
        torch.cuda.current_stream().synchronize()
        outs[i] = (y.detach(), w.grad)

threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
[t.start() for t in threads], [t.join() for t in threads]
for i, (y, g) in enumerate(outs):
    w = table.clone().requires_grad_()
    want = nn.embedding(tok, w, p=0.2, seed=i)
    assert torch.equal(y, want)
    want = torch.autograd.grad(want, w, torch.ones_like(want))[0]
    total = torch.zeros_like(want)
    for _ in range(20):
        total += want
    assert torch.equal(g, total)

nn.embedding(tok + 20, table)
torch.cuda.synchronize()
seen = []

def look():
    start.wait()
    try:
        kernels.check_tokens("cuda")
    except IndexError:
        seen.append(1)

threads = [threading.Thread(target=look) for i in range(8)]
[t.start() for t in threads], [t.join() for t in threads]
assert len(seen) == 1, seen
print("right")
"""
    out = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "right", out.stderr
