"""CPU oracle of the token-table and dropout operators, in 64-bit floats.

Masks: Philox4x32-10 (Salmon et al., SC 2011) on NumPy words, written from
the published round function; element i of a tensor is kept when its 32-bit
word is at least floor(p * 2^32 + 1/2).
"""

from __future__ import annotations

import math

import numpy as np

M0, M1 = 0xD2511F53, 0xCD9E8D57
W0, W1 = 0x9E3779B9, 0xBB67AE85


def philox(counter, key, rounds: int = 10) -> np.ndarray:
    """[n, 4] uint32 words of counters [n, 4] under key (k0, k1)."""
    c = [np.asarray(x, dtype=np.uint64) for x in np.asarray(counter, dtype=np.uint64).T]
    k0, k1 = (int(k) for k in key)
    low = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(M0), c[2] * np.uint64(M1)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & low,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + W0) & 0xFFFFFFFF, (k1 + W1) & 0xFFFFFFFF
    return np.stack(c, axis=1).astype(np.uint32)


def words(n: int, seed: int, offset: int, first: int = 0) -> np.ndarray:
    """The 32-bit words of elements first .. first + n - 1 (first a multiple of 8)."""
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    g = first // 8 + np.arange((n + 7) // 8, dtype=np.uint64)
    parts = []
    for half in (0, 1):
        c = np.stack([g & np.uint64(0xFFFFFFFF), (g >> np.uint64(32)) | np.uint64(half << 31),
                      np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)], axis=1)
        w = philox(c, (seed & 0xFFFFFFFF, seed >> 32))
        parts.append(np.stack([w & 0xFFFF, w >> 16], axis=2).reshape(-1))
    return ((parts[0] << 16) | parts[1])[:n]


def threshold(p: float) -> int:
    return math.floor(p * 2.0 ** 32 + 0.5)


def keep(shape, p: float, seed: int, offset: int) -> np.ndarray:
    n = int(np.prod(shape))
    return (words(n, seed, offset).astype(np.uint64) >= np.uint64(threshold(p))).reshape(shape)


def drop(x, p: float, seed: int, offset: int) -> np.ndarray:
    x = np.asarray(x, dtype=np.float64)
    if p == 0.0:
        return x
    factor = 1.0 / (1.0 - p) if p < 1.0 else 0.0
    with np.errstate(invalid="ignore"):
        return np.where(keep(x.shape, p, seed, offset), x * factor, 0.0)


def embedding(tokens, table, scale=1.0, p=0.0, seed=0, offset=0) -> np.ndarray:
    table = np.asarray(table, dtype=np.float64)
    ok = (tokens >= 0) & (tokens < table.shape[0])
    rows = np.where(ok[:, None], table[np.where(ok, tokens, 0)] * float(scale), np.nan)
    return drop(rows, p, seed, offset)


def embedding_grad(tokens, dy, vocab, scale=1.0, padding_idx=None, p=0.0, seed=0, offset=0):
    """(sum, sum of absolute terms, terms per row) of the table's gradient."""
    dx = drop(dy, p, seed, offset)
    ok = (tokens >= 0) & (tokens < vocab)
    if padding_idx is not None:
        ok &= tokens != padding_idx % vocab
    out = np.zeros((vocab, dx.shape[1]))
    mag = np.zeros_like(out)
    np.add.at(out, tokens[ok], dx[ok])
    np.add.at(mag, tokens[ok], np.abs(dx[ok]))
    return out * float(scale), mag * abs(float(scale)), np.bincount(tokens[ok], minlength=vocab)
