"""Token table, its gradient and dropout on the GPU against the 64-bit oracle.

Tolerances.  Every operator computes in FP32 and rounds once to the output
type.  A rounding is off by at most half a step of its type, eps/2 relative
(or half the spacing of the subnormals).

- dropout: 1/(1-p) rounded to FP32, the product, the sum with the residual:
  at most 3 FP32 roundings relative to |x s| + |r|.
- lookup: scale rounded to FP32, the product, 1/(1-p) rounded, its product:
  4 FP32 roundings.
- gradient of a row with m terms: m - 1 additions in any order are off by at
  most (m - 1) half steps of the sum of the absolute terms (to first order);
  the scale (rounded to FP32), its product and the addition to an existing
  gradient make 3 more; m + 4 is used, of |g| + the sum of absolute terms.
"""

import numpy as np
import pytest
import torch

from oracle import tokens as T
from t3st_b200 import DFCAdamW, kernels, nn

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF32 = 2.0 ** -24
# half the spacing of subnormals
TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def assert_close(got, want, dtype, fp32_error):
    """|got - want| within half a step of dtype plus the FP32 error given."""
    got = f64(got)
    half = torch.finfo(dtype).eps / 2
    tol = half * (np.abs(want) + fp32_error) + fp32_error + TINY[dtype]
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], tol[bad][:4])


def randn(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


# ---- dropout -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 0.999995, 1.0])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 4095, 4096, 4097, 100003])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(cuda, dtype, p, n, residual):
    x, r = randn(n, dtype, n), randn(n, dtype, n + 1) if residual else None
    seed, off = 0xFEDCBA9876543210, 0x1234567890 + n
    y = nn.dropout(x, p, seed=seed, offset=off, residual=r)
    d = T.drop(f64(x), p, seed, off)
    rr = f64(r) if residual else np.zeros(n)
    assert y.dtype == dtype
    assert_close(y, d + rr, dtype, 3 * HALF32 * (np.abs(d) + np.abs(rr)))
    if not residual:
        dropped = ~T.keep((n,), p, seed, off)
        assert (f64(y)[dropped] == 0).all()


@pytest.mark.parametrize("p", [0.1, 0.3, 2.0 ** -17, 1 - 2.0 ** -17, 0.25, 1 / 65536, 3 / 131072])
def test_masks_are_exact_where_the_high_halves_tie(cuda, p):
    n = 1 << 21  # about 32 ties with the threshold's high half
    x = torch.ones(n, device=cuda)
    got = nn.dropout(x, p, seed=9, offset=5).cpu().numpy() != 0
    assert np.array_equal(got, T.keep((n,), p, 9, 5))


def test_dropped_elements_are_zero_whatever_they_hold(cuda):
    n = 4096 + 5
    x = torch.full((n,), float("nan"), device=cuda)
    x[::2] = float("inf")
    keep = T.keep((n,), 0.5, 3, 4)
    for dtype in (F32, BF16, F16):
        y = f64(nn.dropout(x.to(dtype), 0.5, seed=3, offset=4))
        assert (y[~keep] == 0).all() and not np.isfinite(y[keep]).any()
    assert (f64(nn.dropout(x, 1.0, seed=3)) == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [1, 2, 5])
def test_dropout_alignment_and_in_place(cuda, dtype, shift):
    n = 5000
    base = randn(n + 16, dtype, 1)
    res = randn(n + 16, dtype, 2)
    x, r = base[shift:shift + n], res[3:3 + n]
    want = kernels.dropout(x.clone(), torch.empty(n, dtype=dtype, device=cuda), 0.3, 7, 8,
                           residual=r.clone())
    out = torch.full((n + 16,), 5.0, dtype=dtype, device=cuda)
    kernels.dropout(x, out[shift:shift + n], 0.3, 7, 8, residual=r)
    assert torch.equal(out[shift:shift + n], want)
    assert (out[:shift] == 5).all() and (out[shift + n:] == 5).all()
    xc, rc = x.clone(), r.clone()
    kernels.dropout(xc, xc, 0.3, 7, 8, residual=r)
    assert torch.equal(xc, want)
    kernels.dropout(x, rc, 0.3, 7, 8, residual=rc)
    assert torch.equal(rc, want)


def test_dropout_strides_and_empty(cuda):
    x = randn((64, 48), BF16, 3)
    for v in (x.t(), x[:, :40], x[::3], x[:1].expand(5, 48)):
        want = nn.dropout(v.contiguous(), 0.2, seed=1, offset=2)
        got = nn.dropout(v, 0.2, seed=1, offset=2, residual=None)
        assert got.is_contiguous() and torch.equal(got, want)
    assert nn.dropout(x[:0], 0.5, seed=1).shape == (0, 48)
    with pytest.raises(ValueError):
        kernels.dropout(x.t(), torch.empty_like(x.t()), 0.5)
    with pytest.raises(TypeError):
        nn.dropout(x.double(), 0.5)
    with pytest.raises(TypeError):
        nn.dropout(torch.ones(4, device=cuda, dtype=torch.int32), 0.5)


def test_dropout_gradients(cuda):
    n = 3001
    x, r, dy, v = (randn(n, F32, s) for s in (1, 2, 3, 4))
    x.requires_grad_(), r.requires_grad_()
    y = nn.dropout(x, 0.4, seed=5, offset=6, residual=r)
    dx, dr = torch.autograd.grad(y, [x, r], dy, create_graph=False)
    want = T.drop(f64(dy), 0.4, 5, 6)
    assert_close(dx, want, F32, 3 * HALF32 * np.abs(want))
    assert torch.equal(dr, dy)
    # the operator is linear: f(x + v) - f(x) = J v, and <J v, dy> = <v, dx>.
    # Each of the two passes is off by at most 3 half steps of |x s| + |r|, the sum x + v by one
    jv = f64(nn.dropout((x + v).detach(), 0.4, seed=5, offset=6, residual=r)) - f64(y)
    size = (np.abs(f64(x)) + np.abs(f64(v))) / 0.6 + np.abs(f64(r))
    assert abs((jv * f64(dy)).sum() - (f64(v) * f64(dx)).sum()) <= 10 * HALF32 * (size * np.abs(f64(dy))).sum()
    # a backward pass of the backward pass; an expanded incoming gradient
    g = torch.autograd.grad(nn.dropout(x, 0.4, seed=5, offset=6), x, dy.requires_grad_(),
                            create_graph=True)[0]
    (gg,) = torch.autograd.grad(g, dy, v)
    assert torch.equal(gg, nn.dropout(v, 0.4, seed=5, offset=6))
    (dx,) = torch.autograd.grad(nn.dropout(x, 0.4, seed=5, offset=6).sum(), x)
    assert torch.equal(dx, nn.dropout(torch.ones_like(x), 0.4, seed=5, offset=6))


def test_generator_state_on_the_device(cuda):
    rng = nn.CounterRng(seed=(1 << 64) - 12345, device=cuda)
    drop = nn.Dropout(0.3, rng)
    nn.Dropout(0.3, rng)
    last = nn.Dropout(0.3, rng)
    x = randn(777, F32, 1).requires_grad_()
    for step in range(3):
        for m, site in ((drop, 0), (last, 2)):
            want = nn.dropout(x, 0.3, seed=(1 << 64) - 12345, offset=(step << 32) + site)
            assert torch.equal(m(x), want)
        rng.advance()
    assert torch.equal(nn.dropout(x, 0.3, seed=np.int64(5)), nn.dropout(x, 0.3, seed=5))
    y = drop(x)
    rng.advance()
    with pytest.raises(RuntimeError):  # the mask of the forward is gone
        y.sum().backward()


# ---- lookup ------------------------------------------------------------------

@pytest.mark.parametrize("table_dtype,out_dtype", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16),
                                                   (BF16, F32), (BF16, F16), (F16, F16), (F16, F32),
                                                   (F16, BF16)])
@pytest.mark.parametrize("n,dim", [(1, 1), (5, 3), (100, 8), (17, 64), (33, 65), (3, 1001), (700, 1),
                                   (9, 4096), (2000, 24)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_embedding(cuda, table_dtype, out_dtype, n, dim, p):
    vocab = 97
    table = randn((vocab, dim), table_dtype, dim, 0.02)
    gen = torch.Generator().manual_seed(n)
    tok = torch.randint(0, vocab, (n,), generator=gen)
    scale = dim ** 0.5
    for t in (tok.cuda(), tok.int().cuda()):
        out = nn.embedding(t, table, scale, p=p, seed=21, offset=4, out_dtype=out_dtype)
        want = T.embedding(tok.numpy(), f64(table), scale, p, 21, 4)
        assert out.dtype == out_dtype and out.shape == (n, dim)
        assert_close(out, want, out_dtype, 4 * HALF32 * np.abs(want))


def test_embedding_shapes_strides_and_empty(cuda):
    big = randn((50, 80), BF16, 1)
    tok = torch.randint(0, 50, (6, 7), generator=torch.Generator().manual_seed(2)).cuda()
    for table in (big[:, :64], big[:, 3:60], big[::2], big[:, 8:72], big[:1].expand(50, 80)):
        tk = tok % table.shape[0]
        assert torch.equal(nn.embedding(tk, table), table[tk])
        assert torch.equal(nn.embedding(tk.t(), table), table[tk.t()])
        assert torch.equal(nn.embedding(tk[:, ::2], table), table[tk[:, ::2]])
    assert nn.embedding(tok[:0], big).shape == (0, 7, 80)
    assert nn.embedding(tok[0, 0], big).shape == (80,)
    out = torch.full((42 * 80 + 8,), 3.0, dtype=BF16, device=cuda)
    for shift in (0, 1, 4):
        o = out[shift:shift + 42 * 80].view(42, 80)
        kernels.embedding(tok, big, o)
        assert torch.equal(o, big[tok.view(-1)])
        assert (out[shift + 42 * 80:] == 3).all()
    with pytest.raises(ValueError):
        kernels.embedding(tok, big, torch.empty(42, 40, dtype=BF16, device=cuda))
    with pytest.raises(ValueError):
        kernels.embedding(tok, big.t(), torch.empty(42, 50, dtype=BF16, device=cuda))
    with pytest.raises(TypeError):
        nn.embedding(tok.float(), big)
    with pytest.raises(TypeError):
        nn.embedding(tok, big.double())
    with pytest.raises(RuntimeError):
        nn.embedding(tok.cpu(), big)


@pytest.mark.parametrize("dim", [64, 33])
def test_tokens_outside_the_table(cuda, dim):
    table = randn((10, dim), F32, 1)
    tok = torch.tensor([3, -1, 9, 10, 1 << 40, 0, -(1 << 62)], device=cuda)
    bad = torch.tensor([0, 1, 0, 1, 1, 0, 1], dtype=torch.bool, device=cuda)
    out = nn.embedding(tok, table)
    torch.cuda.synchronize()
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], table[tok[~bad]])
    with pytest.raises(IndexError):
        nn.embedding(tok[:1], table)
    assert torch.equal(nn.embedding(tok[:1], table), table[3:4])  # reported once
    dy = randn((7, dim), F32, 2)
    grad = torch.empty(10, dim, device=cuda)
    kernels.embedding_grad(tok, dy, grad)
    torch.cuda.synchronize()
    with pytest.raises(IndexError):
        kernels.check_tokens("cuda")
    kernels.check_tokens("cuda")
    want, _, _ = T.embedding_grad(tok.cpu().numpy(), f64(dy), 10)
    assert np.array_equal(f64(grad), want)  # one term a row


def test_errors_reach_the_caller(cuda):
    """A token outside the table, met by the forward, raises in the backward;
    a status of the C ABI raises DfcError, in the backward too."""
    from t3st_b200._lib import DFC_ERR_SIZE, DfcError

    w = randn((10, 8), F32, 1).requires_grad_()
    out = nn.embedding(torch.tensor([1, 11], device=cuda), w)
    torch.cuda.synchronize()
    with pytest.raises(IndexError):
        out.sum().backward()
    far = torch.empty((1 << 31) + 64, dtype=BF16, device=cuda).as_strided((2, 8), (1 << 31, 1))
    with pytest.raises(DfcError) as e:
        nn.embedding(torch.tensor([0], device=cuda), far)
    assert e.value.status == DFC_ERR_SIZE
    far.zero_()
    out = nn.embedding(torch.tensor([0, 1], device=cuda), w.detach().to(BF16).requires_grad_())
    with pytest.raises(DfcError):
        out.backward(far)
    assert torch.equal(nn.embedding(torch.tensor([3], device=cuda), w), w[3:4])


# ---- gradient ----------------------------------------------------------------

def draw_tokens(kind, n, vocab, seed):
    g = np.random.default_rng(seed)
    if kind == "equal":
        return np.full(n, vocab - 1)
    if kind == "distinct":
        return g.permutation(vocab)[np.arange(n) % vocab]
    if kind == "uniform":
        return g.integers(0, vocab, n)
    ids = np.floor(vocab * g.random(n) ** 4).astype(np.int64)  # skewed to low ids
    if kind == "padded":
        ids[n // 2:] = min(1, vocab - 1)
    return ids


def check_grad(tok, dy, vocab, *, grad_dtype=F32, accumulate=False, padding_idx=None, scale=1.0, p=0.0,
               seed=17, offset=5, grad=None, wide=True):
    dim = dy.shape[1]
    if grad is None:
        grad = randn((vocab, dim), grad_dtype, 99)
    before = grad.clone()
    t = torch.from_numpy(tok).cuda()
    got = kernels.embedding_grad(t if wide else t.int(), dy, grad, scale=scale, padding_idx=padding_idx,
                                 p=p, seed=seed, offset=offset, accumulate=accumulate)
    assert got is grad
    want, mag, terms = T.embedding_grad(tok, f64(dy), vocab, scale, padding_idx, p, seed, offset)
    base = f64(before) if accumulate else np.zeros_like(want)
    assert_close(grad, want + base, grad.dtype, HALF32 * (terms[:, None] + 4) * (mag + np.abs(base)))
    untouched = torch.from_numpy(terms == 0).cuda()
    assert torch.equal(grad[untouched], before[untouched] if accumulate
                       else torch.zeros_like(before[untouched]))
    return grad


SHAPES = [(1, 5, 8), (2, 1, 3), (31, 7, 16), (32, 3, 129), (33, 40, 1000), (300, 511, 64), (4097, 513, 24),
          (5000, 1000, 72), (700, 70001, 8), (2049, 263000, 16), (20000, 37, 40),
          (500, 60, 1001), (1500, 99, 523), (512, 300, 264), (513, 300, 264), (256, 70, 40), (1024, 300, 264), (1025, 300, 264), (257, 9, 2056)]


@pytest.mark.parametrize("kind", ["equal", "distinct", "uniform", "skewed", "padded"])
@pytest.mark.parametrize("n,vocab,dim", SHAPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_grad(cuda, kind, n, vocab, dim, accumulate):
    tok = draw_tokens(kind, n, vocab, n)
    check_grad(tok, randn((n, dim), F32, dim), vocab, accumulate=accumulate, scale=1.7)


@pytest.mark.parametrize("n", [5, 400, 5000])
@pytest.mark.parametrize("vocab", [(1 << 23) - 1, 1 << 23, 9_000_001])
def test_embedding_grad_of_large_tables(cuda, n, vocab):
    """Around the table size up to which every CTA sorts few tokens itself."""
    tok = draw_tokens("uniform", n, vocab, n)
    tok[: n // 3] = vocab - 1
    dy = randn((n, 8), F32, 1)
    grad = torch.full((vocab, 8), 3.0, device=cuda)
    t = torch.from_numpy(tok).cuda()
    kernels.embedding_grad(t, dy, grad)
    rows = np.unique(tok)
    want, mag, terms = T.embedding_grad(np.searchsorted(rows, tok), f64(dy), len(rows))
    assert_close(grad[torch.from_numpy(rows).cuda()], want, F32, HALF32 * (terms[:, None] + 4) * mag)
    grad[t] = 0
    assert not grad.any()


@pytest.mark.parametrize("shift", [1, 3, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_grad_alignment(cuda, shift, dtype):
    """dy and grad that begin anywhere; what lies around grad stays as it was."""
    n, vocab, dim = 333, 77, 136
    tok = draw_tokens("skewed", n, vocab, 2)
    dy = randn(n * dim + 16, dtype, 3)[shift:shift + n * dim].view(n, dim)
    for accumulate in (False, True):
        flat = torch.full((vocab * dim + 32,), 7.0, dtype=dtype, device=cuda)
        check_grad(tok, dy, vocab, grad=flat[shift:shift + vocab * dim].view(vocab, dim), accumulate=accumulate)
        assert (flat[:shift] == 7).all() and (flat[shift + vocab * dim:] == 7).all()


@pytest.mark.parametrize("dy_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("grad_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [64, 37, 1])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_grad_types(cuda, dy_dtype, grad_dtype, dim, accumulate):
    n, vocab = 1500, 211
    tok = draw_tokens("skewed", n, vocab, 3)
    check_grad(tok, randn((n, dim), dy_dtype, 4, 0.1), vocab, grad_dtype=grad_dtype,
               accumulate=accumulate, scale=0.3, wide=accumulate)


@pytest.mark.parametrize("dim", [64, 37, 8, 3])
@pytest.mark.parametrize("p", [1e-6, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("kind", ["skewed", "equal"])
def test_embedding_grad_with_dropout(cuda, dim, p, kind):
    n, vocab = 900, 50
    check_grad(draw_tokens(kind, n, vocab, 5), randn((n, dim), BF16, 6), vocab, p=p, scale=2.0)


@pytest.mark.parametrize("padding_idx", [0, 1, 49, -1, -50])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_grad_padding(cuda, padding_idx, accumulate):
    tok = draw_tokens("padded", 1000, 50, 7)
    check_grad(tok, randn((1000, 32), F32, 8), 50, padding_idx=padding_idx, accumulate=accumulate)
    only = np.full(70, padding_idx % 50)
    check_grad(only, randn((70, 32), F32, 9), 50, padding_idx=padding_idx, accumulate=accumulate)


@pytest.mark.parametrize("dim,lead,width", [(64, 0, 72), (64, 3, 80), (60, 4, 64), (33, 1, 40)])
def test_embedding_grad_views(cuda, dim, lead, width):
    """Rows inside wider matrices: what lies beside them stays as it was."""
    n, vocab = 400, 90
    tok = draw_tokens("skewed", n, vocab, 11)
    dy = randn((n, width), BF16, 12)[:, lead:lead + dim]
    for accumulate in (False, True):
        whole = torch.full((vocab, width), 7.0, device=cuda)
        check_grad(tok, dy, vocab, grad=whole[:, lead:lead + dim], accumulate=accumulate)
        assert (whole[:, :lead] == 7).all() and (whole[:, lead + dim:] == 7).all()
    check_grad(tok, dy[:1].expand(n, dim), vocab)
    with pytest.raises(ValueError):
        kernels.embedding_grad(torch.from_numpy(tok).cuda(), dy, torch.empty(1, dim, device=cuda).expand(vocab, dim))


def test_gradients_of_masked_places_do_not_count(cuda):
    """NaN and Inf at padding, out-of-range and dropped places stay there."""
    n, vocab, dim = 300, 20, 64
    tok = draw_tokens("uniform", n, vocab, 1)
    tok[::7] = 5                    # the padding row
    tok[3::11] = vocab + 2          # outside
    dy = randn((n, dim), F32, 2)
    keep = torch.from_numpy(T.keep((n, dim), 0.4, 17, 5)).cuda()
    dy[~keep] = float("nan")
    dy[torch.from_numpy((tok == 5) | (tok >= vocab)).cuda()] = float("inf")
    grad = kernels.embedding_grad(torch.from_numpy(tok).cuda(), dy, torch.empty(vocab, dim, device=cuda),
                                  padding_idx=5, p=0.4, seed=17, offset=5)
    assert torch.isfinite(grad).all() and (grad[5] == 0).all()
    with pytest.raises(IndexError):
        kernels.check_tokens(cuda)


def test_embedding_grad_edges(cuda):
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    grad = torch.ones(5, 16, device=cuda)
    kernels.embedding_grad(none, torch.empty(0, 16, device=cuda), grad, accumulate=True)
    assert (grad == 1).all()
    kernels.embedding_grad(none, torch.empty(0, 16, device=cuda), grad)
    assert (grad == 0).all()
    kernels.embedding_grad(none, torch.empty(0, 16, device=cuda), torch.empty(0, 16, device=cuda))
    kernels.embedding_grad(torch.zeros(3, dtype=torch.int64, device=cuda), torch.empty(3, 0, device=cuda),
                           torch.empty(4, 0, device=cuda))
    tok = torch.zeros(3, dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError):
        kernels.embedding_grad(tok, torch.zeros(2, 16, device=cuda), grad)
    with pytest.raises(ValueError):
        kernels.embedding_grad(tok, torch.zeros(3, 8, device=cuda), grad)
    with pytest.raises(ValueError):
        kernels.embedding_grad(tok, torch.zeros(3, 16, device=cuda), grad, padding_idx=5)
    with pytest.raises(TypeError):
        kernels.embedding_grad(tok, torch.zeros(3, 16, device=cuda).double(), grad)


@pytest.mark.parametrize("n,dim", [(9000, 520), (40000, 64), (140000, 32), (300, 2048)])
@pytest.mark.parametrize("kind", ["skewed", "padded"])
def test_embedding_grad_same_bits(cuda, n, dim, kind):
    tok = draw_tokens(kind, n, 30000, 13)
    dy = randn((n, dim), BF16, 14)
    a = check_grad(tok, dy, 30000, p=0.1)
    t = torch.from_numpy(tok).cuda()
    for _ in range(3):
        b = kernels.embedding_grad(t, dy, torch.empty_like(a), p=0.1, seed=17, offset=5)
        assert torch.equal(a, b)


def test_table_behind_32_bit_offsets(cuda):
    """More than 2^32 elements in the table: rows at its end."""
    vocab, dim = 1_100_000, 4096
    assert vocab * dim > 2 ** 32
    table = torch.zeros(vocab, dim, dtype=BF16, device=cuda)
    tok = np.array([vocab - 1, 5, vocab - 1, 1_048_576, 0, vocab - 2])
    rows = randn((6, dim), BF16, 1)
    t = torch.from_numpy(tok).cuda()
    dy = rows.float()
    kernels.embedding_grad(t, rows, table, accumulate=True)
    want = torch.zeros(6, dim, device=cuda)
    for i in range(6):
        want[i] = dy[torch.from_numpy(tok == tok[i]).cuda()].sum(0)
    assert torch.equal(table[t], want.to(BF16))  # two terms at most: one FP32 rounding is exact here
    assert torch.equal(nn.embedding(t, table), table[t])
    kernels.embedding_grad(t[:1], rows[:1], table)
    assert torch.equal(table[vocab - 1], rows[0])
    for i in range(1, 6):
        if tok[i] != vocab - 1:
            assert (table[tok[i]] == 0).all()


# ---- together, as they are used -----------------------------------------------

class Net(torch.nn.Module):
    def __init__(self, rng, vocab=120, dim=48, in_place=False):
        super().__init__()
        self.emb = nn.Embedding(vocab, dim, padding_idx=0, scale=dim ** 0.5, p=0.1, rng=rng,
                                out_dtype=BF16, grad_in_place=in_place)
        self.lin = torch.nn.Linear(dim, dim, dtype=BF16)
        self.drop = nn.Dropout(0.2, rng)

    def forward(self, tok):
        h = self.emb(tok)
        return self.drop(self.lin(h), residual=h)


def make(in_place=False):
    torch.manual_seed(0)
    rng = nn.CounterRng(seed=3, device="cuda")
    return rng, Net(rng, in_place=in_place).cuda()


def test_training_block_against_the_oracle(cuda):
    rng, net = make()
    rng.advance()
    tok = torch.randint(0, 120, (4, 50), generator=torch.Generator().manual_seed(1)).cuda()
    h = net.emb(tok)
    b = randn(h.shape, BF16, 2).requires_grad_()
    y = net.drop(b, residual=h)
    dy = randn(h.shape, BF16, 3)
    y.backward(dy)
    base = 1 << 32
    flat = tok.view(-1).cpu().numpy()
    want_h = T.embedding(flat, f64(net.emb.weight), 48 ** 0.5, 0.1, 3, base)
    assert_close(h.view(-1, 48), want_h, BF16, 4 * HALF32 * np.abs(want_h))
    d = T.drop(f64(b).reshape(-1), 0.2, 3, base + 1)
    assert_close(y.reshape(-1), d + f64(h).reshape(-1), BF16,
                 3 * HALF32 * (np.abs(d) + np.abs(f64(h).reshape(-1))))
    db = T.drop(f64(dy).reshape(-1), 0.2, 3, base + 1)
    assert_close(b.grad.view(-1), db, BF16, 3 * HALF32 * np.abs(db))
    want, mag, terms = T.embedding_grad(flat, f64(dy).reshape(-1, 48), 120, 48 ** 0.5, 0, 0.1, 3, base)
    assert_close(net.emb.weight.grad, want, F32, HALF32 * (terms[:, None] + 4) * mag)
    assert (net.emb.weight.grad[0] == 0).all()


def test_gradient_of_the_lookup_against_differences(cuda):
    """The lookup is linear in the table: <f(W + V) - f(W), dy> = <V, dW>."""
    tok = torch.randint(0, 30, (200,), generator=torch.Generator().manual_seed(5)).cuda()
    w, v, dy = randn((30, 20), F32, 1), randn((30, 20), F32, 2), randn((200, 20), F32, 3)
    kw = dict(p=0.3, seed=8, offset=9)
    w.requires_grad_()
    y = nn.embedding(tok, w, 3.0, **kw)
    (dw,) = torch.autograd.grad(y, w, dy)
    diff = f64(nn.embedding(tok, (w + v).detach(), 3.0, **kw)) - f64(y)
    # 4 half steps a pass of each value and one of w + v; the rows' sums have at most 200 terms
    size = (np.abs(f64(w)) + np.abs(f64(v)))[tok.cpu().numpy()] * 3.0 / 0.7
    bound = HALF32 * (10 + 204) * (size * np.abs(f64(dy))).sum()
    assert abs((diff * f64(dy)).sum() - (f64(v) * f64(dw)).sum()) <= bound


def test_in_place_gradient_feeds_the_optimizer(cuda):
    """grad_in_place gives the parameters that a dense gradient gives."""
    toks = [torch.randint(0, 120, (3, 40), generator=torch.Generator().manual_seed(s)).cuda()
            for s in range(4)]
    finals = []
    for in_place in (False, True):
        rng, net = make(in_place)
        opt = DFCAdamW(net.parameters(), lr=1e-2, weight_decay=0.01)
        for tok in toks:
            opt.zero_grad(set_to_none=False)
            net(tok).float().square().mean().backward()
            opt.step()
            rng.advance()
        finals.append([p.detach().clone() for p in net.parameters()])
    # adding a run's sum to a zeroed row is exact
    for a, b in zip(*finals):
        assert torch.equal(a, b)


def test_second_derivatives_of_the_lookup(cuda):
    """The lookup and the table's gradient are each other's gradient."""
    tok = torch.randint(0, 20, (60,), generator=torch.Generator().manual_seed(5)).cuda()
    w = randn((20, 24), F32, 1).requires_grad_()
    dy = randn((60, 24), F32, 2).requires_grad_()
    v = randn((20, 24), F32, 3)
    kw = dict(padding_idx=3, p=0.3, seed=8, offset=9)
    (dw,) = torch.autograd.grad(nn.embedding(tok, w, 2.0, **kw), w, dy, create_graph=True)
    assert (dw[3] == 0).all()
    (ddy,) = torch.autograd.grad(dw, dy, v)
    v[3] = 0
    assert torch.equal(ddy, nn.embedding(tok, v, 2.0, **kw))
    w.grad = torch.zeros_like(w)
    with pytest.raises(RuntimeError):
        nn.embedding(tok, w, 2.0, grad_in_place=True).sum().backward(create_graph=True)


def test_in_place_gradient_in_the_sharded_optimizer(cuda):
    """ShardedDFCAdamW owns .grad (a view of its flat buffer): the table's rows
    are added there, and the step is the one that a dense gradient gives."""
    import torch.distributed as dist

    from t3st_b200.zero import ShardedDFCAdamW

    made = not dist.is_initialized()
    if made:
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        tok = torch.randint(0, 120, (3, 40), generator=torch.Generator().manual_seed(1)).cuda()
        finals = []
        for in_place in (False, True):
            torch.manual_seed(0)
            net = nn.Embedding(120, 48, padding_idx=0, scale=2.0, grad_in_place=in_place).cuda()
            opt = ShardedDFCAdamW(net.parameters(), lr=1e-2, weight_decay=0.01)
            for _ in range(3):
                opt.zero_grad()
                net(tok).square().mean().backward()
                assert net.weight.grad.data_ptr() == opt.flat_grad.data_ptr()
                opt.step()
            finals.append(net.weight.detach().clone())
        assert torch.equal(*finals)
    finally:
        if made:
            dist.destroy_process_group()


def test_in_place_gradient_accumulates(cuda):
    rng, net = make(True)
    tok = torch.randint(1, 120, (64,), generator=torch.Generator().manual_seed(1)).cuda()
    w = net.emb.weight
    net.emb(tok).float().sum().backward()  # no .grad yet: a dense one
    first = w.grad
    one = first.clone()
    net.emb(tok).float().sum().backward()
    assert w.grad is first and torch.equal(first, 2 * one)


def test_captured_steps_replay_like_eager_ones(cuda):
    rng, net = make()
    tok = torch.randint(0, 120, (4, 32), device=cuda)
    dy = randn((4, 32, 48), BF16, 7)

    def step():
        y = net(tok)
        grads = torch.autograd.grad(y, list(net.parameters()), dy)
        rng.advance()
        return [y.detach(), *grads]

    eager = [[t.clone() for t in step()] for _ in range(5)]
    rng.state[1] = 0
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = step()
    with torch.cuda.graph(g2, pool=g1.pool()):
        out2 = step()
    rng.state[1] = 0
    for i in range(5):
        (g1, g2)[i % 2].replay()
        for got, want in zip((out1, out2)[i % 2], eager[i]):
            assert torch.equal(got, want)


@pytest.mark.parametrize("in_place", [False, True])
def test_captured_backward_into_existing_gradients(cuda, in_place):
    rng, net = make(in_place)
    tok = torch.randint(0, 120, (4, 32), device=cuda)
    dy = randn((4, 32, 48), BF16, 7)
    for p in net.parameters():
        p.grad = torch.zeros_like(p)

    def step():
        for p in net.parameters():
            p.grad.zero_()
        net(tok).backward(dy)
        rng.advance()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    eager = []
    rng.state[1] = 0
    with torch.cuda.stream(s):
        for _ in range(3):
            step()
            eager.append([p.grad.clone() for p in net.parameters()])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    rng.state[1] = 0
    for want in eager:
        graph.replay()
        assert all(torch.equal(p.grad, g) for p, g in zip(net.parameters(), want))


def test_other_streams(cuda):
    tok = torch.randint(0, 1000, (5000,), device=cuda)
    dy = randn((5000, 256), BF16, 1)
    want = kernels.embedding_grad(tok, dy, torch.empty(1000, 256, device=cuda), p=0.2, seed=1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:  # calls at once, each with a workspace of its own
        with torch.cuda.stream(s):
            for _ in range(4):
                outs.append(kernels.embedding_grad(tok, dy, torch.empty(1000, 256, device=cuda), p=0.2,
                                                   seed=1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
