"""The table's gradient along each form of its sort and its joins: one cluster
with one, two, four and eight items a thread, count / scan / scatter with one
to four passes, runs over many blocks; int32 and int64 tokens.

Tolerance as in test_gpu_tokens.py: m + 4 FP32 half steps of the sum of the
absolute terms for a row of m terms, and the rounding to the output type."""

import numpy as np
import pytest
import torch

from oracle import tokens as T
from t3st_b200 import kernels

pytestmark = pytest.mark.gpu

HALF32 = 2.0 ** -24


def draw(kind, n, vocab, seed):
    g = np.random.default_rng(seed)
    if kind == "equal":
        return np.full(n, vocab - 1)
    if kind == "distinct":
        return g.permutation(vocab)[np.arange(n) % vocab]
    ids = np.floor(vocab * g.random(n) ** 4).astype(np.int64)
    if kind == "padded":
        ids[n // 2:] = min(1, vocab - 1)
    return ids


def check(tok, vocab, dim, *, dtype=torch.float32, accumulate=False, **kw):
    """Both widths of tokens; the rows that occur against the oracle, the others
    zero or as they were; returns the gradient."""
    n = len(tok)
    dy = torch.randn(n, dim, generator=torch.Generator().manual_seed(n + dim)).to(dtype).cuda()
    rows = np.unique(tok)
    want, mag, terms = T.embedding_grad(np.searchsorted(rows, tok), dy.double().cpu().numpy(), len(rows), **kw)
    base = 3.0 if accumulate else 0.0
    bound = HALF32 * ((terms[:, None] + 4) * (mag + base) + np.abs(want + base))
    grads = []
    for width in (torch.int64, torch.int32):
        grad = torch.full((vocab, dim), 3.0, device="cuda")
        t = torch.from_numpy(tok).to(width).cuda()
        kernels.embedding_grad(t, dy, grad, accumulate=accumulate, **kw)
        named = torch.from_numpy(rows).cuda()
        got = grad[named].double().cpu().numpy()
        bad = ~(np.abs(got - (want + base)) <= bound)
        assert not bad.any(), (int(bad.sum()), got[bad][:4], (want + base)[bad][:4])
        rest = torch.ones(vocab, dtype=torch.bool, device="cuda")
        rest[named] = False
        assert (grad[rest] == base).all()
        grads.append(grad)
    assert torch.equal(*grads)
    return grads[0]


# CTAs and items a thread: 1 x 1, 2 x 1, 16 x 1, 16 x 2, 16 x 4, 16 x 8, then the other kernels
COUNTS = [1024, 1025, 16384, 16385, 32768, 32769, 65535, 65536, 65537, 131071, 131072, 131073]


@pytest.mark.parametrize("n", COUNTS)
@pytest.mark.parametrize("kind", ["skewed", "equal", "distinct"])
@pytest.mark.parametrize("vocab", [400, 30000])
def test_each_form_of_the_sort(cuda, n, kind, vocab):
    tok = draw(kind, n, vocab, n)
    check(tok, vocab, 8, accumulate=kind == "skewed")


@pytest.mark.parametrize("n", [3, 256, 257, 512])
@pytest.mark.parametrize("kind", ["skewed", "equal", "distinct"])
def test_few_tokens_of_either_width(cuda, n, kind):
    check(draw(kind, n, 700, n), 700, 40)
    check(draw(kind, n, 700, n), 700, 33, accumulate=True)


@pytest.mark.parametrize("n", [5000, 100000, 131073, 140000])
@pytest.mark.parametrize("vocab", [1, 511, 512, 262143, 262144, (1 << 27) + 3])
def test_passes_of_the_sort(cuda, n, vocab):
    """One to four passes: the last one leaves the order in either buffer."""
    tok = draw("skewed", n, vocab, n)
    tok[:: max(1, n // 50)] = vocab - 1
    check(tok, vocab, 1)


@pytest.mark.parametrize("n,dim", [(20000, 512), (70000, 64), (20000, 513), (140000, 40)])
@pytest.mark.parametrize("kind", ["equal", "padded"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_runs_over_many_blocks(cuda, n, dim, kind, accumulate):
    """Up to 625 blocks in one run: more than a join looks at in one round."""
    check(draw(kind, n, 200, n), 200, dim, accumulate=accumulate)
    check(draw(kind, n, 200, n), 200, dim, dtype=torch.bfloat16, accumulate=accumulate, scale=0.5,
          p=0.1, seed=3, offset=4)


@pytest.mark.parametrize("n", [100, 40000, 100000, 140000])
def test_padding_and_tokens_outside_of_either_width(cuda, n):
    tok = draw("padded", n, 300, n)
    tok[::9] = 300
    tok[1::9] = -5
    dy = torch.randn(n, 8, generator=torch.Generator().manual_seed(1)).cuda()
    want, mag, terms = T.embedding_grad(tok, dy.double().cpu().numpy(), 300, padding_idx=1)
    for width in (torch.int64, torch.int32):
        grad = kernels.embedding_grad(torch.from_numpy(tok).to(width).cuda(), dy,
                                      torch.empty(300, 8, device="cuda"), padding_idx=1)
        assert (np.abs(grad.double().cpu().numpy() - want) <= HALF32 * ((terms[:, None] + 4) * mag
                                                                        + np.abs(want))).all()
        torch.cuda.synchronize()
        with pytest.raises(IndexError):
            kernels.check_tokens("cuda")
