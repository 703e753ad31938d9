"""Workloads of the token-table and dropout operators: what each call is given,
its plain form in elementary torch operations, its exact values, and the bytes
and operations it cannot do without.

Four kinds of case:

``embed``    rows of a table looked up by token id, scaled, with dropout
``grad``     the table's gradient from the gradient of looked-up rows
``dropout``  dropout with a counter-based generator, optionally added to a residual
``block``    lookup with dropout, a residual dropout on top, and the backward of both

Dropout's random words are a function of (seed, offset, element index):
Philox4x32-10 with the seed as its key and the counter (g, offset), g the number
of the group of eight elements; one call gives the high 16 bits of the group's
eight words, a second one (top counter bit of g set) the low 16 bits.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


# ---- cases -----------------------------------------------------------------

def _embed(name, tokens, vocab, dim, table, out, p):
    return {"name": name, "kind": "embed", "tokens": tokens, "vocab": vocab, "dim": dim,
            "table": table, "out": out, "p": p}


def _grad(name, tokens, vocab, dim, dy, grad, p, into, pad, skip):
    return {"name": name, "kind": "grad", "tokens": tokens, "vocab": vocab, "dim": dim, "dy": dy,
            "grad": grad, "p": p, "into": into, "pad": pad, "skip": skip}


def _dropout(name, n, dtype, p, residual):
    return {"name": name, "kind": "dropout", "n": n, "dtype": dtype, "p": p, "residual": residual}


def listed():
    return [
        # the next tokens of eight sequences: latency
        _embed("embed-8-tokens", 8, 32000, 1024, "bf16", "bf16", 0.0),
        # odd width and a ragged number of tokens, 16-bit table
        _embed("embed-odd", 5003, 49999, 1001, "f16", "f16", 0.1),
        # a training micro-batch of 8 x 2048 from an FP32 table into bf16 activations
        _embed("embed-train", 16384, 131072, 4096, "f32", "bf16", 0.1),
        # a short batch of a small model, into an existing FP32 gradient
        _grad("grad-300-tokens", 300, 5000, 384, "f32", "f32", 0.0, True, 0.0, False),
        # a 16-bit table's gradient as a new dense tensor
        _grad("grad-dense-bf16", 8192, 50000, 1024, "bf16", "bf16", 0.0, False, 0.0, False),
        # a training micro-batch into a zeroed flat FP32 buffer, embedding dropout on
        _grad("grad-into-flat", 32768, 32768, 2048, "bf16", "f32", 0.1, True, 0.0, False),
        # half of the batch is padding that takes part in the gradient: one very long run
        _grad("grad-padded", 32768, 32000, 1536, "f16", "f32", 0.0, False, 0.5, False),
        # the largest batch and table; a padding id that gets no gradient
        _grad("grad-largest", 65539, 131072, 4096, "bf16", "f32", 0.0, False, 0.1, True),
        # one activation row: latency
        _dropout("dropout-row", 4096, "bf16", 0.1, False),
        # FP32 activations of odd length
        _dropout("dropout-f32-odd", 12345677, "f32", 0.3, False),
        # residual dropout of a block's output, 8192 tokens of width 8192
        _dropout("dropout-residual", 8192 * 8192, "bf16", 0.1, True),
        # forward and backward of the input block of a model in training
        {"name": "block-train", "kind": "block", "tokens": 8192, "vocab": 50000, "dim": 2048,
         "table": "f32", "out": "bf16", "p": 0.1},
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))


def _width(rng, lo, hi):
    d = _log(rng, lo, hi)
    return d if rng.random() < 0.3 else max(8, d // 64 * 64 if d >= 64 else d // 8 * 8)


def draw(rng):
    kind = rng.choice(["embed", "grad", "grad", "dropout", "block"])
    p = rng.choice([0.0, 0.05, 0.1, 0.1, 0.25, 0.5])
    if kind == "dropout":
        return {"kind": kind, "n": _log(rng, 1, 8192 * 8192), "dtype": rng.choice(list(DTYPES)),
                "p": rng.choice([0.05, 0.1, 0.2, 0.3, 0.5]), "residual": rng.random() < 0.5}
    dim = _width(rng, 16, 4096)
    vocab = _log(rng, 500, 131072)
    if kind == "embed":
        table = rng.choice(["f32", "bf16", "f16"])
        return {"kind": kind, "tokens": _log(rng, 1, 65536 // (4 if p else 1)), "vocab": vocab,
                "dim": dim, "table": table, "out": "bf16" if rng.random() < 0.4 else table, "p": p}
    if kind == "block":
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "vocab": min(vocab, 65536), "dim": dim,
                "table": "f32", "out": rng.choice(["f32", "bf16", "f16"]), "p": max(p, 0.05)}
    dy = rng.choice(["f32", "bf16", "f16"])
    return {"kind": kind, "tokens": _log(rng, 1, 65536 // (4 if p else 1)), "vocab": vocab,
            "dim": dim, "dy": dy, "grad": rng.choice(["f32", dy]), "p": p,
            "into": rng.random() < 0.5, "pad": rng.choice([0.0, 0.0, 0.3, 0.9]),
            "skip": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------

PAD = 1  # the id of padding tokens


def _probs(vocab):
    # word frequencies fall about as one over the rank
    w = 1.0 / (np.arange(vocab, dtype=np.float64) + 3.0)
    return w / w.sum()


def _tokens(case, gen):
    cdf = torch.from_numpy(np.cumsum(_probs(case["vocab"]))).cuda()
    n = case["tokens"]
    u = torch.rand(n, dtype=torch.float64, device="cuda", generator=gen)
    ids = torch.searchsorted(cdf, u).clamp_(max=case["vocab"] - 1)
    if case.get("pad"):
        # whole tails of sequences are padding
        ids[n - int(n * case["pad"]):] = PAD
    return ids


def _normal(shape, dtype, gen, std=1.0):
    x = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen)
    return x.to(DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case, "seed": 0x9E3779B97F4A7C15 * (seed + 1) % (1 << 63), "offset": seed % 1000 + 1}
    if case["kind"] == "dropout":
        st["x"] = _normal(case["n"], case["dtype"], gen)
        st["residual"] = _normal(case["n"], case["dtype"], gen) if case["residual"] else None
        return st
    n, vocab, dim = case["tokens"], case["vocab"], case["dim"]
    st["tokens"] = _tokens(case, gen)
    st["scale"] = math.sqrt(dim)
    if case["kind"] in ("embed", "block"):
        st["table"] = _normal((vocab, dim), case["table"], gen, 0.02)
    if case["kind"] == "block":
        st["branch"] = _normal((n, dim), case["out"], gen)
        st["dy"] = _normal((n, dim), case["out"], gen, 1e-2)
        if own:
            st["table"].requires_grad_(True)
            st["branch"].requires_grad_(True)
    if case["kind"] == "grad":
        st["dy"] = _normal((n, dim), case["dy"], gen, 1e-2)
        st["pad"] = PAD if case["skip"] else None
        # the optimizer's gradient buffer, which exists before the backward pass
        st["grad"] = torch.zeros((vocab, dim), dtype=DTYPES[case["grad"]], device="cuda")
    return st


# ---- the operators ------------------------------------------------------------

def run(st):
    case = st["case"]
    return (_run_own if own else _run_plain)[case["kind"]](case, st)


def _own_embed(case, st):
    from t3st_b200 import nn
    return nn.embedding(st["tokens"], st["table"], st["scale"], p=case["p"], seed=st["seed"],
                        offset=st["offset"], out_dtype=DTYPES[case["out"]])


def _own_grad(case, st):
    from t3st_b200 import kernels
    if case["into"]:
        grad = st["grad"]
        grad.zero_()  # the optimizer's zero_grad()
    else:
        grad = torch.empty_like(st["grad"])
    return kernels.embedding_grad(st["tokens"], st["dy"], grad, scale=st["scale"],
                                  padding_idx=st["pad"], p=case["p"], seed=st["seed"],
                                  offset=st["offset"], accumulate=case["into"])


def _own_dropout(case, st):
    from t3st_b200 import nn
    return nn.dropout(st["x"], case["p"], seed=st["seed"], offset=st["offset"],
                      residual=st["residual"])


def _own_block(case, st):
    from t3st_b200 import nn
    h = nn.embedding(st["tokens"], st["table"], st["scale"], p=case["p"], seed=st["seed"],
                     offset=st["offset"], out_dtype=DTYPES[case["out"]])
    y = nn.dropout(st["branch"], case["p"], seed=st["seed"], offset=st["offset"] + 1, residual=h)
    d_table, d_branch = torch.autograd.grad(y, [st["table"], st["branch"]], st["dy"])
    return h.detach(), y.detach(), d_table, d_branch


_run_own = {"embed": _own_embed, "grad": _own_grad, "dropout": _own_dropout, "block": _own_block}


def _mulhilo(a, b):
    # 32 x 32 -> 64 bits; the 64-bit product wraps, its bits are right
    prod = a * b
    return (prod >> 32) & 0xFFFFFFFF, prod & 0xFFFFFFFF


def _philox(groups, half, seed, offset):
    """Four 32-bit words (int64 tensors) for each group number."""
    c0, c1 = groups & 0xFFFFFFFF, (groups >> 32) | (half << 31)
    c2 = torch.full_like(groups, offset & 0xFFFFFFFF)
    c3 = torch.full_like(groups, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c0, c1, c2, c3


def _halves(groups, half, seed, offset):
    words = torch.stack(_philox(groups, half, seed, offset), dim=1)
    return torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)


def _keep(n, p, seed, offset, device):
    groups = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    u = (_halves(groups, 0, seed, offset) << 16) | _halves(groups, 1, seed, offset)
    return u[:n] >= math.floor(p * 2.0 ** 32 + 0.5)


def _drop(x, p, seed, offset):
    """x in FP32, any shape."""
    if p == 0.0:
        return x
    keep = _keep(x.numel(), p, seed, offset, x.device).view(x.shape)
    return torch.where(keep, x * (1.0 / (1.0 - p)), torch.zeros_like(x))


def _table_grad(tokens, dx, vocab, scale, pad, out):
    """out[v] += scale * (sum of dx over the tokens that are v), FP32."""
    if pad is not None:
        dx = torch.where((tokens == pad)[:, None], torch.zeros_like(dx), dx)
    return out.index_add_(0, tokens, dx * scale)


def _plain_embed(case, st):
    rows = st["table"][st["tokens"]].float() * st["scale"]
    return _drop(rows, case["p"], st["seed"], st["offset"]).to(DTYPES[case["out"]])


def _plain_grad(case, st):
    dx = _drop(st["dy"].float(), case["p"], st["seed"], st["offset"])
    acc = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float32, device=dx.device)
    _table_grad(st["tokens"], dx, case["vocab"], st["scale"], st["pad"], acc)
    if not case["into"]:
        return acc.to(st["grad"].dtype)
    grad = st["grad"]
    grad.zero_()
    grad.copy_(grad.float() + acc)
    return grad


def _plain_dropout(case, st):
    y = _drop(st["x"].float(), case["p"], st["seed"], st["offset"])
    if st["residual"] is not None:
        y = st["residual"].float() + y
    return y.to(st["x"].dtype)


def _plain_block(case, st):
    out = DTYPES[case["out"]]
    h = _plain_embed(case, st)
    y = h.float() + _drop(st["branch"].float(), case["p"], st["seed"], st["offset"] + 1)
    dy = st["dy"].float()
    d_branch = _drop(dy, case["p"], st["seed"], st["offset"] + 1)
    d_table = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float32, device=dy.device)
    _table_grad(st["tokens"], _drop(dy, case["p"], st["seed"], st["offset"]), case["vocab"],
                st["scale"], None, d_table)
    return h, y.to(out), d_table.to(st["table"].dtype), d_branch.to(out)


_run_plain = {"embed": _plain_embed, "grad": _plain_grad, "dropout": _plain_dropout,
              "block": _plain_block}


# ---- what a pass cannot do without ----------------------------------------------

def _distinct(case):
    n, vocab = case["tokens"], case["vocab"]
    pads = int(n * case.get("pad", 0.0))
    return max(1.0, float(-np.expm1((n - pads) * np.log1p(-_probs(vocab))).sum()))


def work(case):
    if case["kind"] == "dropout":
        size, n = SIZES[case["dtype"]], case["n"]
        return {"bytes": n * size * (3 if case["residual"] else 2),
                "flops": n * (3 if case["residual"] else 2)}
    n, vocab, dim = case["tokens"], case["vocab"], case["dim"]
    rows, e = _distinct(case), n * dim
    if case["kind"] == "embed":
        return {"bytes": 8 * n + rows * dim * SIZES[case["table"]] + e * SIZES[case["out"]],
                "flops": e * 2}
    if case["kind"] == "block":
        ts, os = SIZES[case["table"]], SIZES[case["out"]]
        # tokens, rows, branch and dy are read; h, y, d_branch and the dense d_table written
        return {"bytes": 8 * n + rows * dim * ts + 5 * e * os + vocab * dim * ts, "flops": 8 * e}
    read = n - (int(n * case["pad"]) if case["skip"] else 0)
    gs = SIZES[case["grad"]]
    grad = vocab * dim * gs + (2 * rows * dim * gs if case["into"] else 0)
    return {"bytes": 8 * n + read * dim * SIZES[case["dy"]] + grad, "flops": 2 * read * dim}


# ---- exact values ------------------------------------------------------------------

def _exact_keep(n, p, seed, offset):
    """The same truth values from 32-bit unsigned words on the host."""
    keep = np.empty((n + 7) // 8 * 8, dtype=bool)
    limit = np.uint64(int(math.floor(p * 4294967296.0 + 0.5)))
    step = 1 << 17
    u32, u64 = np.uint32, np.uint64
    for lo in range(0, (n + 7) // 8, step):
        g = np.arange(lo, min(lo + step, (n + 7) // 8), dtype=u64)
        parts = []
        for half in (0, 1):
            x = [(g & u64(0xFFFFFFFF)).astype(u32), ((g >> u64(32)) | u64(half << 31)).astype(u32),
                 np.full(g.size, offset & 0xFFFFFFFF, u32), np.full(g.size, offset >> 32, u32)]
            key = [seed & 0xFFFFFFFF, seed >> 32]
            for _ in range(10):
                a = x[0].astype(u64) * u64(0xD2511F53)
                b = x[2].astype(u64) * u64(0xCD9E8D57)
                x = [(b >> u64(32)).astype(u32) ^ x[1] ^ u32(key[0]), b.astype(u32),
                     (a >> u64(32)).astype(u32) ^ x[3] ^ u32(key[1]), a.astype(u32)]
                key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
            # little-endian words seen as pairs of 16-bit numbers
            parts.append(np.stack(x, axis=1).view(np.uint16).reshape(-1).astype(u64))
        keep[8 * lo: 8 * (lo + g.size)] = parts[0] * u64(65536) + parts[1] >= limit
    return torch.from_numpy(keep[:n]).cuda()


def _exact_drop(x, p, seed, offset):
    """x in FP64; kept values over 1 - p, the others zero."""
    if p == 0.0:
        return x
    keep = _exact_keep(x.numel(), p, seed, offset).view(x.shape)
    return x.div(1.0 - p).masked_fill_(~keep, 0.0)


def _exact_table_grad(tokens, dx, vocab, scale, pad):
    # tokens in sorted order, one sum per run of equal ones
    order = torch.argsort(tokens, stable=True)
    ids, counts = torch.unique_consecutive(tokens[order], return_counts=True)
    sums = torch.segment_reduce(dx[order], "sum", lengths=counts, axis=0)
    out = torch.zeros((vocab, dx.shape[1]), dtype=torch.float64, device=dx.device)
    out[ids] = sums * scale
    if pad is not None:
        out[pad] = 0.0
    return out


def exact(case, seed):
    elements = case["n"] if case["kind"] == "dropout" else case["tokens"] * case["dim"]
    if case["p"] and elements > 3 << 25:
        return None
    st = prepare(case, seed)
    with torch.no_grad():
        p, key, off = case["p"], st["seed"], st["offset"]
        if case["kind"] == "dropout":
            y = _exact_drop(st["x"].double(), p, key, off)
            return y if st["residual"] is None else y + st["residual"].double()
        if case["kind"] == "grad":
            dx = _exact_drop(st["dy"].double(), p, key, off)
            return _exact_table_grad(st["tokens"], dx, case["vocab"], st["scale"], st["pad"])
        h = st["table"].double().index_select(0, st["tokens"])
        h = _exact_drop(h * st["scale"], p, key, off)
        if case["kind"] == "embed":
            return h
        dy = st["dy"].double()
        y = h + _exact_drop(st["branch"].double(), p, key, off + 1)
        d_table = _exact_table_grad(st["tokens"], _exact_drop(dy, p, key, off), case["vocab"],
                                    st["scale"], None)
        return h, y, d_table, _exact_drop(dy, p, key, off + 1)
