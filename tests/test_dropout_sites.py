"""Every module with a generator has a site of its own, also one whose p is
raised from zero later."""

from types import SimpleNamespace

import pytest
import torch

from t3st_b200 import _lib, nn


@pytest.fixture
def offsets(monkeypatch):
    """Offsets that the modules hand to the native calls."""
    seen = []
    monkeypatch.setattr(_lib, "host", lambda: SimpleNamespace(
        nn_dropout=lambda x, p, seed, offset, state, residual: seen.append((p, offset)),
        nn_embedding=lambda tok, w, scale, pad, p, seed, offset, state, out, in_place:
            seen.append((p, offset))))
    return seen


def test_a_table_whose_p_is_raised_later(offsets):
    rng = nn.CounterRng()
    a = nn.Dropout(0.1, rng)
    early = nn.Embedding(4, 8, p=0.0, rng=rng)
    late = nn.Embedding(4, 8, rng=rng)
    b = nn.Embedding(4, 8, p=0.1, rng=rng)
    tok, x = torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    early(tok), late(tok)
    early.p = late.p = 0.2
    for m, arg in ((a, x), (early, tok), (late, tok), (b, tok)):
        m(arg)
    assert [p for p, _ in offsets] == [0.0, 0.0, 0.1, 0.2, 0.2, 0.1]
    used = [offset for _, offset in offsets[2:]]
    assert len(set(used)) == 4
    assert (used[0], used[3]) == (0, 1)  # numbered as before
    assert all(0 <= offset < 1 << 32 for offset in used)  # within one step's block


def test_a_table_without_a_generator_refuses_p(offsets):
    m = nn.Embedding(4, 8)
    m(torch.zeros(3, dtype=torch.int64))
    m.p = 0.1
    with pytest.raises(ValueError, match="CounterRng"):
        m(torch.zeros(3, dtype=torch.int64))
    assert len(offsets) == 1
