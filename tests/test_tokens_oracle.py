"""Token-table and dropout operators without a GPU: the oracle's generator
against published vectors, the C ABI's and the Python layer's refusals."""

import ctypes
import struct

import numpy as np
import pytest
import torch

from oracle import tokens as T
from t3st_b200 import _lib, kernels, nn

no_device = pytest.mark.skipif(
    torch.cuda.is_available(),
    reason="passes made-up device addresses; runs only where no GPU is visible")


@pytest.mark.parametrize("counter,key,want", [
    # known-answer vectors of Philox4x32-10
    ([0, 0, 0, 0], [0, 0], [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]),
])
def test_philox_known_answers(counter, key, want):
    assert T.philox([counter], key)[0].tolist() == want


def test_words_are_a_function_of_the_element_index():
    w = T.words(1003, 5, 7)
    assert np.array_equal(T.words(99, 5, 7), w[:99])
    assert np.array_equal(T.words(11, 5, 7, first=992), w[992:])
    assert not np.array_equal(T.words(1003, 5, 8), w)
    assert not np.array_equal(T.words(1003, 6, 7), w)
    # a billion groups on, the second counter word changes
    assert not np.array_equal(T.words(8, 5, 7, first=8 << 32), w[:8])


def test_keep_rate():
    n = 1 << 20
    for p in (0.05, 0.1, 0.5, 0.9):
        dropped = n - T.keep((n,), p, 11, 3).sum()
        assert abs(dropped - n * p) < 6 * (n * p * (1 - p)) ** 0.5
    assert T.keep((64,), 0.0, 1, 1).all() and not T.keep((64,), 1.0, 1, 1).any()


def drop_arg(p, state=0):
    return struct.pack("<QQQd", 1, 2, state, p)


@no_device
def test_dropout_refusals():
    f = _lib.lib().dfc_dropout
    X, R, Y = 0x10000, 0x20000, 0x30000
    assert f(X, R, Y, -1, 0, None, None) == _lib.DFC_ERR_SIZE
    assert f(X, R, Y, (1 << 39) + 1, 0, None, None) == _lib.DFC_ERR_SIZE
    assert f(X, R, Y, 8, 3, None, None) == _lib.DFC_ERR_DTYPE
    for p in (-0.1, 1.0000001, float("nan"), float("inf")):
        assert f(X, R, Y, 8, 0, drop_arg(p), None) == _lib.DFC_ERR_VALUE
    assert f(X, R, Y, 8, 0, drop_arg(0.5, state=0x1004), None) == _lib.DFC_ERR_ALIGN
    assert f(None, R, Y, 8, 0, None, None) == _lib.DFC_ERR_NULL
    assert f(X, R, None, 8, 0, None, None) == _lib.DFC_ERR_NULL
    assert f(X + 2, R, Y, 8, 0, None, None) == _lib.DFC_ERR_ALIGN
    assert f(X, R + 1, Y, 8, 1, None, None) == _lib.DFC_ERR_ALIGN
    assert f(None, None, None, 0, 0, drop_arg(0.5), None) == _lib.DFC_OK


@no_device
def test_embedding_refusals():
    lib = _lib.lib()

    def f(tokens=0x1000, tb=8, n=4, table=0x20000, tdt=0, pitch=16, vocab=10, dim=16, out=0x30000,
          odt=0, drop=None, flag=0x40000):
        return lib.dfc_embedding(tokens, tb, n, table, tdt, pitch, vocab, dim, 1.0, out, odt, drop,
                                 flag, None)

    for bad in (dict(n=-1), dict(n=(1 << 28) + 1), dict(vocab=-1), dict(vocab=(1 << 30) + 1),
                dict(dim=-1), dict(dim=(1 << 20) + 1), dict(pitch=-1), dict(pitch=1 << 31), dict(n=1 << 28, dim=1 << 12)):
        assert f(**bad) == _lib.DFC_ERR_SIZE, bad
    for bad in (dict(tb=2), dict(tdt=4), dict(odt=-1)):
        assert f(**bad) == _lib.DFC_ERR_DTYPE, bad
    assert f(drop=drop_arg(2.0)) == _lib.DFC_ERR_VALUE
    for bad in (dict(tokens=None), dict(table=None), dict(out=None)):
        assert f(**bad) == _lib.DFC_ERR_NULL, bad
    for bad in (dict(tokens=0x1004), dict(table=0x20002), dict(out=0x30001, odt=1), dict(flag=0x40002)):
        assert f(**bad) == _lib.DFC_ERR_ALIGN, bad
    assert f(n=0, tokens=None, out=None) == _lib.DFC_OK
    assert f(dim=0, out=None) == _lib.DFC_OK


@no_device
def test_embedding_grad_refusals():
    lib = _lib.lib()
    need = lib.dfc_embedding_grad_scratch_bytes(4, 10, 16)
    assert need > 0
    assert lib.dfc_embedding_grad_scratch_bytes(-1, 10, 16) == 0
    assert lib.dfc_embedding_grad_scratch_bytes(4, 10, (1 << 20) + 1) == 0

    def f(tokens=0x1000, tb=8, n=4, dy=0x20000, ddt=0, dpitch=16, grad=0x30000, gdt=0, gpitch=16,
          vocab=10, dim=16, drop=None, flag=0x40000, scratch=0x50000, nbytes=need):
        return lib.dfc_embedding_grad(tokens, tb, n, dy, ddt, dpitch, grad, gdt, gpitch, vocab, dim,
                                      1.0, -1, 0, drop, flag, scratch, nbytes, None)

    for bad in (dict(n=-1), dict(n=(1 << 28) + 1), dict(vocab=-1), dict(dim=-1), dict(dpitch=-1),
                dict(dpitch=1 << 31), dict(gpitch=1 << 31), dict(gpitch=15), dict(n=1 << 28, dim=1 << 12, gpitch=1 << 12)):
        assert f(**bad) == _lib.DFC_ERR_SIZE, bad
    for bad in (dict(tb=1), dict(ddt=3), dict(gdt=9)):
        assert f(**bad) == _lib.DFC_ERR_DTYPE, bad
    assert f(drop=drop_arg(-1.0)) == _lib.DFC_ERR_VALUE
    for bad in (dict(tokens=None), dict(dy=None), dict(grad=None), dict(scratch=None)):
        assert f(**bad) == _lib.DFC_ERR_NULL, bad
    for bad in (dict(tokens=0x1004), dict(dy=0x20002), dict(grad=0x30001, gdt=1),
                dict(flag=0x40001), dict(scratch=0x50008)):
        assert f(**bad) == _lib.DFC_ERR_ALIGN, bad
    assert f(nbytes=need - 1) == _lib.DFC_ERR_SCRATCH
    assert f(n=0, vocab=0, tokens=None, dy=None, grad=None, scratch=None, nbytes=0) == _lib.DFC_OK
    assert f(dim=0) == _lib.DFC_OK


def test_struct_matches_header():
    assert struct.calcsize("<QQQd") == _lib.DROPOUT_DTYPE.itemsize == 32
    assert _lib.strerror(_lib.DFC_ERR_VALUE) not in ("", "unknown status")
    assert isinstance(drop_arg(0.5), bytes) and ctypes.sizeof(ctypes.c_void_p) == 8


def test_python_refusals_without_a_gpu():
    x = torch.zeros(8)
    w, tok = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        nn.dropout(x, 0.5)
    with pytest.raises(ValueError):
        nn.dropout(x, 0.5, residual=torch.zeros(4))
    with pytest.raises(ValueError):
        nn.dropout(x, 0.5, residual=x.half())
    with pytest.raises(RuntimeError):
        nn.embedding(tok, w)
    with pytest.raises(ValueError):
        nn.embedding(tok, x)
    for bad in (4, -5):
        with pytest.raises(ValueError):
            nn.embedding(tok, w, padding_idx=bad)
        with pytest.raises(ValueError):
            nn.Embedding(4, 8, padding_idx=bad)
    with pytest.raises(ValueError):
        nn.embedding(tok, (w.requires_grad_() * 2), grad_in_place=True)
    with pytest.raises(ValueError):
        nn.Embedding(4, 8, p=0.1)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            nn.Dropout(p, nn.CounterRng())
        with pytest.raises(ValueError):
            nn.Embedding(4, 8, p=p, rng=nn.CounterRng())
        with pytest.raises(ValueError):
            nn.dropout(x, p)
    with pytest.raises(TypeError):
        nn.dropout(x, 0.5, seed=torch.zeros(2))
    with pytest.raises(TypeError):
        nn.dropout(x, 0.5, seed=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        kernels.embedding_grad(tok, torch.zeros(3, 8), w)
    with pytest.raises(ValueError):
        kernels.embedding_grad(tok, torch.zeros(3, 8), w, padding_idx=4)
    for bad in (dict(seed="1"), dict(offset=1.5), dict(residual=3)):
        with pytest.raises(TypeError):
            nn.dropout(x, 0.5, **bad)
    with pytest.raises(TypeError):
        nn.embedding(tok, w, out_dtype="bf16")


def test_modules_on_the_host():
    rng = nn.CounterRng(seed=(1 << 64) - 3)
    assert rng.state.tolist() == [-3, 0]
    a, b = nn.Dropout(0.5, rng), nn.Dropout(0.5, rng)
    emb = nn.Embedding(6, 4, padding_idx=-1, p=0.1, rng=rng)
    assert (a.site, b.site, emb.site) == (0, 1, 2)
    assert emb.padding_idx == 5 and emb.weight[5].abs().max() == 0
    rng.advance()
    assert rng.state.tolist() == [-3, 1 << 32]
    other = nn.CounterRng()
    other.load_state_dict(rng.state_dict())
    assert torch.equal(other.state, rng.state)
    x = torch.randn(5)
    assert a.eval()(x) is x
    assert torch.equal(a(x, residual=x), x + x)
