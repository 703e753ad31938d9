"""Host side of the token-table and dropout operators on a GPU: threads,
streams, autograd's bookkeeping, empty batches."""

import os
import subprocess
import sys

import pytest
import torch

from t3st_b200 import kernels, nn

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


@pytest.mark.parametrize("tokens,vocab,dim", [((0,), 6, 8), ((0,), 6, 5), ((0,), 0, 8), ((0, 3), 6, 8),
                                              ((2, 0), 6, 8), ((0,), 6, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_backward_of_an_empty_batch(cuda, tokens, vocab, dim, in_place):
    """The gradient that sum() sends back is expanded: its strides are zero."""
    w = torch.randn(vocab, dim, device=cuda).requires_grad_()
    if in_place:
        w.grad = torch.ones_like(w)
    y = nn.embedding(torch.zeros(tokens, dtype=torch.int64, device=cuda), w, 2.0, p=0.1, seed=1,
                     grad_in_place=in_place)
    y.sum().backward()
    assert y.shape == (*tokens, dim) and w.grad.shape == w.shape
    assert torch.equal(w.grad, torch.ones_like(w) if in_place else torch.zeros_like(w))


def test_second_derivative_of_an_empty_batch(cuda):
    w = torch.randn(6, 8, device=cuda).requires_grad_()
    dy = torch.zeros(0, 8, device=cuda).requires_grad_()
    y = nn.embedding(torch.zeros(0, dtype=torch.int64, device=cuda), w)
    (dw,) = torch.autograd.grad(y, w, dy, create_graph=True)
    dw.sum().backward()
    assert dy.grad.shape == (0, 8) and torch.equal(dw, torch.zeros_like(w))


def test_rows_of_empty_matrices_lie_anywhere(cuda):
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    dy = torch.zeros(1, 1, device=cuda).expand(0, 8)
    assert dy.shape == (0, 8) and dy.stride() == (0, 0)
    grad = kernels.embedding_grad(none, dy, torch.ones(5, 8, device=cuda))
    assert not grad.any()


@pytest.mark.parametrize("tokens", [(), (3,), (2, 3), (1, 2, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_backward_of_a_table_without_columns(cuda, tokens, in_place):
    w = torch.empty(6, 0, device=cuda, requires_grad=True)
    if in_place:
        w.grad = torch.empty(6, 0, device=cuda)
    y = nn.embedding(torch.zeros(tokens, dtype=torch.int64, device=cuda), w, grad_in_place=in_place)
    y.sum().backward()
    assert y.shape == (*tokens, 0) and w.grad.shape == (6, 0)


def test_autograd_sees_that_buffers_are_written(cuda):
    """A buffer that a graph has saved and that a call then overwrites: its
    backward raises, as after any in-place operation, instead of using the new
    values."""
    table = torch.randn(6, 8, device=cuda)
    tok = torch.arange(4, device=cuda)
    calls = {
        "embedding": lambda b: kernels.embedding(tok, table, b),
        "dropout": lambda b: kernels.dropout(table[:4], b, 0.5),
        "dropout in place": lambda b: kernels.dropout(b, b, 0.5),
        "grad": lambda b: kernels.embedding_grad(tok, table[:4], b),
        "grad added": lambda b: kernels.embedding_grad(tok, table[:4], b, accumulate=True),
    }
    for name, write in calls.items():
        buf = torch.randn(4, 8, device=cuda)
        w = torch.ones(4, 8, device=cuda, requires_grad=True)
        y, want = (buf * w).sum(), buf.clone()
        y.backward(retain_graph=True)
        assert torch.equal(w.grad, want)
        before = buf._version
        assert write(buf) is buf
        assert buf._version == before + 1, name
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    w = table.clone().requires_grad_()
    w.grad = torch.zeros_like(w)
    v = torch.ones_like(w).requires_grad_()
    y = (w.grad * v).sum()
    nn.embedding(tok, w, grad_in_place=True).sum().backward()
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    assert not nn.dropout(table, 0.5)._version and not nn.embedding(tok, w)._version


def test_buffers_of_inference_mode_are_written_as_before(cuda):
    table = torch.randn(6, 8, device=cuda)
    tok = torch.arange(4, device=cuda)
    with torch.inference_mode():
        out = kernels.embedding(tok, table, torch.empty(4, 8, device=cuda))
    assert torch.equal(kernels.dropout(out, out, 0.0), table[:4])


@pytest.mark.parametrize("caller", ["default", "forward", "third"])
@pytest.mark.parametrize("tied", [False, True])
def test_in_place_rows_are_ordered_behind_and_before_the_accumulator(cuda, caller, tied):
    """The weight's accumulator was made on the default stream, the lookup runs
    on another one, where its backward is held up: what follows backward() on
    its caller's stream, and a dense gradient of the same weight (tied to a
    second use), come after the rows."""
    gen = torch.Generator().manual_seed(4)
    tok = torch.randint(0, 40, (300,), generator=gen).cuda()
    dy = torch.randint(-8, 9, (300, 64), generator=gen).float().cuda()
    dense = torch.randint(-8, 9, (40, 64), generator=gen).float().cuda()
    w = torch.randn(40, 64, generator=gen).cuda().requires_grad_()
    want = torch.zeros_like(w).index_add_(0, tok, dy)  # whole numbers: exact in any order
    if tied:
        want = want + dense
    main, side, third = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()
    w.grad = torch.zeros_like(w)
    other = w * dense  # makes the accumulator
    side.wait_stream(main)
    with torch.cuda.stream(side):
        out = nn.embedding(tok, w, grad_in_place=True)
        out.register_hook(lambda g: torch.cuda._sleep(100_000_000))  # about 50 ms, in the backward
        loss = (out * dy).sum()
    main.wait_stream(side)
    if tied:
        loss = loss + other.sum()
    stream = {"default": main, "forward": side, "third": third}[caller]
    stream.wait_stream(main)
    with torch.cuda.stream(stream):
        for _ in range(2):
            loss.backward(retain_graph=True)
        got = w.grad.clone()
    torch.cuda.synchronize()
    assert torch.equal(got, 2 * want) and torch.equal(w.grad, 2 * want)


def test_captured_in_place_backward_beside_an_eager_graph_is_refused(cuda):
    """Ordering a capture behind an eager graph's stream is not possible: the
    call raises, and the process goes on."""
    code = """
import torch
from t3st_b200 import nn

w = torch.randn(10, 8, device="cuda").requires_grad_()
tok = torch.arange(5, device="cuda")
w.grad = torch.zeros_like(w)
eager = nn.embedding(tok, w, grad_in_place=True)  # alive: its accumulator is the default stream's
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
dy = torch.ones(5, 8, device="cuda")
said = ""
with torch.cuda.graph(graph):
    try:
        nn.embedding(tok, w, grad_in_place=True).backward(dy)
    except RuntimeError as e:
        said = str(e)
assert "made outside the capture" in said, said
del eager
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    nn.embedding(tok, w, grad_in_place=True).backward(dy)
w.grad.zero_()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(w.grad[:5], dy) and not w.grad[5:].any()
print("refused")
"""
    out = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "refused", out.stderr


def test_masks_of_a_rank(cuda):
    x = torch.randn(1000, device=cuda)
    for rank, base in ((0, 0), (1, 1 << 63), (3, 3 << 62), (6, 3 << 61)):
        rng = nn.CounterRng(seed=5, rank=rank, device=cuda)
        rng.advance()
        want = nn.dropout(x, 0.3, seed=5, offset=base + (1 << 32) + 2)
        assert torch.equal(nn.dropout(x, 0.3, seed=rng, offset=2), want)


def test_autograd_grad_of_an_in_place_weight(cuda):
    """torch.autograd.grad asks for the gradient: it gets a dense one, and .grad
    stays as it was.  backward(inputs=...) adds in place only to its inputs."""
    tok = torch.randint(0, 20, (60,), generator=torch.Generator().manual_seed(5)).cuda()
    w = torch.randn(20, 24, device=cuda).requires_grad_()
    x = torch.randn(60, 24, device=cuda).requires_grad_()
    dy = torch.randn(60, 24, device=cuda).requires_grad_()
    kw = dict(padding_idx=3, p=0.3, seed=8, offset=9)
    want = torch.autograd.grad(nn.embedding(tok, w, 2.0, **kw), w, dy)[0].detach()
    w.grad = torch.ones_like(w)
    y = nn.embedding(tok, w, 2.0, grad_in_place=True, **kw) + x
    (dw,) = torch.autograd.grad(y, w, dy, retain_graph=True)
    assert torch.equal(dw, want) and (w.grad == 1).all()
    dw, dx = torch.autograd.grad(y, [w, x], dy, retain_graph=True)
    assert torch.equal(dw, want) and torch.equal(dx, dy) and (w.grad == 1).all()
    (dw,) = torch.autograd.grad(y, w, dy, create_graph=True)
    (ddy,) = torch.autograd.grad(dw, dy, torch.ones_like(w))
    ones = torch.ones_like(w)
    ones[3] = 0
    assert torch.equal(ddy, nn.embedding(tok, ones, 2.0, **kw))
    y.backward(dy, inputs=[x], retain_graph=True)
    assert (w.grad == 1).all()
    grad = w.grad
    y.backward(dy, inputs=[w], retain_graph=True)
    assert w.grad is grad and torch.equal(grad, want + 1)
    y.backward(dy)
    assert w.grad is grad and torch.equal(grad, want + 1 + want)


def test_hooks_see_an_in_place_weights_gradient(cuda):
    """A hook on the weight's gradient, or on its accumulation, needs the dense
    gradient: it gets it, with the result that a dense gradient gives."""
    tok = torch.randint(0, 20, (60,), generator=torch.Generator().manual_seed(5)).cuda()
    w = torch.randn(20, 24, device=cuda).requires_grad_()
    dy = torch.randn(60, 24, device=cuda)
    want = torch.autograd.grad(nn.embedding(tok, w, 2.0), w, dy)[0]

    def backward():
        w.grad = torch.ones_like(w)
        nn.embedding(tok, w, 2.0, grad_in_place=True).backward(dy)
        return w.grad

    assert torch.equal(backward(), want + 1)
    hook = w.register_hook(lambda g: g * 2)
    assert torch.equal(backward(), want * 2 + 1)
    hook.remove()
    seen = []
    hook = w.register_post_accumulate_grad_hook(lambda p: seen.append(p.grad.clone()))
    assert torch.equal(backward(), want + 1) and len(seen) == 1 and torch.equal(seen[0], want + 1)
    hook.remove()
    accumulator = w.view_as(w).grad_fn.next_functions[0][0]
    hook = accumulator.register_prehook(lambda g: (g[0] * 4,))
    assert torch.equal(backward(), want * 4 + 1)
    hook.remove()
    assert torch.equal(backward(), want + 1) and len(seen) == 1


def test_optimizer_in_the_backward_pass(cuda):
    """Steps taken by hooks on accumulation happen with grad_in_place too."""
    from t3st_b200 import DFCAdamW

    tok = torch.randint(0, 50, (90,), generator=torch.Generator().manual_seed(5)).cuda()
    finals = []
    for in_place in (False, True):
        torch.manual_seed(0)
        emb = nn.Embedding(50, 16, grad_in_place=in_place, device=cuda)
        opt = DFCAdamW(emb.parameters(), lr=1e-2)
        emb.weight.grad = torch.zeros_like(emb.weight)

        def step(p):
            opt.step()
            opt.zero_grad(set_to_none=False)

        emb.weight.register_post_accumulate_grad_hook(step)
        before = emb.weight.detach().clone()
        for _ in range(3):
            emb(tok).square().sum().backward()
        assert not torch.equal(before, emb.weight)
        finals.append(emb.weight.detach().clone())
    assert torch.equal(*finals)
