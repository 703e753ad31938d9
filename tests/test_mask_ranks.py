"""Data-parallel ranks draw masks of their own, also after buffers were
broadcast or one rank's checkpoint was loaded everywhere."""

import copy
import io
import pickle
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import tokens as T
from t3st_b200 import _lib, nn

P = 0.5


@pytest.fixture
def masks(monkeypatch):
    """Modules' masks on the host: the native calls give the mask of their arguments."""
    def keep(x, p, seed, offset, state):
        if state is not None:
            seed, offset = state[0].item(), state[1].item() + offset
        return torch.from_numpy(T.keep(tuple(x.shape), p, seed, offset))

    fake = SimpleNamespace(
        nn_dropout=lambda x, p, seed, offset, state, residual: keep(x, p, seed, offset, state),
        nn_embedding=lambda tok, w, scale, pad, p, seed, offset, state, out, in_place:
            keep(w[tok], p, seed, offset, state))
    monkeypatch.setattr(_lib, "host", lambda: fake)


class Net(torch.nn.Module):
    def __init__(self, rank):
        super().__init__()
        self.rng = nn.CounterRng(seed=5, rank=rank)
        self.emb = nn.Embedding(9, 16, p=P, rng=self.rng)
        self.drop = nn.Dropout(P, self.rng)

    def forward(self):
        x = torch.zeros(20, 16)
        return torch.stack([self.emb(torch.zeros(20, dtype=torch.int64)), self.drop(x),
                            nn.dropout(x, P, seed=self.rng, offset=7)])


def test_ranks_differ_and_rank_0_is_the_default(masks):
    nets = [Net(r) for r in range(4)]
    for step in range(3):
        out = [n() for n in nets]
        rows = torch.cat([o.flatten(1) for o in out])
        assert len({r.numpy().tobytes() for r in rows}) == len(rows)  # 4 ranks x 3 places
        for i, offset in enumerate((0, 1, 7)):
            assert np.array_equal(out[0][i].numpy(), T.keep((20, 16), P, 5, (step << 32) + offset))
        for n in nets:
            n.rng.advance()
    x = torch.zeros(20, 16)
    one = nn.CounterRng(seed=5, rank=1)
    assert torch.equal(nn.dropout(x, P, seed=one, offset=np.int64(3)), nn.dropout(x, P, seed=one, offset=3))
    with pytest.raises(TypeError):
        nn.dropout(x, P, seed=one, offset=1.5)
    a, b = nn.CounterRng(seed=5), nn.CounterRng(seed=5, rank=0)
    assert torch.equal(nn.dropout(x, P, seed=a), nn.dropout(x, P, seed=b))


def test_broadcast_buffers_and_checkpoints_keep_the_ranks_apart(masks):
    nets = [Net(r) for r in range(3)]
    nets[0].rng.advance()
    want = [n() for n in nets]
    file = io.BytesIO()
    torch.save(nets[0].state_dict(), file)
    for n in nets[1:]:  # as broadcast from rank 0, and as loaded from its checkpoint
        for mine, first in zip(n.buffers(), nets[0].buffers()):
            mine.copy_(first)
    after = [n() for n in nets]
    file.seek(0)
    state = torch.load(file)
    for r in (1, 2):
        n = Net(r)
        n.load_state_dict(state)
        assert torch.equal(n(), after[r]) and not torch.equal(n(), after[0])
        assert not torch.equal(after[r], want[r])  # rank 0 had advanced
    assert not torch.equal(after[1], after[2]) and torch.equal(after[0], want[0])
    for twin in (copy.deepcopy(nets[2]), pickle.loads(pickle.dumps(nets[2]))):
        assert torch.equal(twin(), after[2])


@pytest.mark.parametrize("ranks", [1, 2, 8, 1000])
def test_ranks_stay_apart_for_many_steps(ranks):
    """The offsets of R ranks (a power of two) are 2^64 / R apart: their steps
    do not meet before 2^32 / R steps."""
    base = sorted(nn.CounterRng(rank=r).base for r in range(ranks))
    gaps = [b - a for a, b in zip(base, base[1:] + [base[0] + (1 << 64)])]
    assert min(gaps) >= (1 << 64) >> (ranks - 1).bit_length()
    assert all(0 <= b < 1 << 64 for b in base)


def test_refusals():
    for bad in (-1, 1 << 32):
        with pytest.raises(ValueError):
            nn.CounterRng(rank=bad)
    with pytest.raises(TypeError):
        nn.CounterRng(rank=1.5)


def test_counters_saved_before_ranks_existed(masks):
    old = nn.CounterRng(seed=5)
    for name in ("rank", "base"):
        old.__dict__.pop(name, None)
    assert torch.equal(nn.dropout(torch.zeros(64), P, seed=old),
                       nn.dropout(torch.zeros(64), P, seed=nn.CounterRng(seed=5)))
