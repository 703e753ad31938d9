"""The ends of a training step that surround the optimizer for a language
model: a token table whose gradient is summed by sorted tokens, in a fixed
order, straight into the optimizer's gradient buffer; and dropout whose mask
is computed from a counter and never stored.  (No reference counterpart: the
reference, YellowJune/T3st, trains convolutional models.)

    rng = CounterRng(seed=1, device="cuda")
    emb = Embedding(50000, 1024, scale=32.0, p=0.1, rng=rng, out_dtype=torch.bfloat16)
    drop = Dropout(0.1, rng)
    h = emb(tokens)                 # lookup, scale and dropout in one pass
    h = drop(block(h), residual=h)  # h + dropout(block(h)) in one pass
    loss(h).backward()              # both masks are computed again
    optimizer.step(); rng.advance()

Both run through the C ABI of libdfc_b200.so on CUDA tensors only, and give
the same bits for the same inputs.
"""

from __future__ import annotations

import operator

import torch

from . import _lib

__all__ = ["CounterRng", "Dropout", "Embedding", "dropout", "embedding"]

# sites of one CounterRng before advance() moves on to a new block of offsets
_SITES = 1 << 32


class CounterRng(torch.nn.Module):
    """(seed, offset) of dropout masks, on the device.

    Each dropout place takes a ``site()`` number of its own; ``advance()``
    (once per step, after backward) moves every site to fresh masks.  The
    kernels read the state when they run, so a captured graph that contains
    ``advance()`` draws new masks at each replay.  The state is a buffer:
    checkpoints carry it.  ``advance()`` between a forward and its backward
    makes that backward raise, as any in-place change of a saved tensor does.

    ``rank``: ranks with data of their own (data parallel) each give their
    number, or all drop the same elements; ranks that hold the same activations
    (tensor parallel) give the same one.  It is not part of the state, so that
    broadcast buffers and a checkpoint loaded on every rank leave the ranks
    apart.  R ranks (rounded up to a power of two) share no mask for
    2^32 / R steps.  ``state`` alone, given as a seed, is rank 0's.
    """

    rank = base = _spares = 0  # counters pickled without them

    def __init__(self, seed: int = 0, device=None, *, rank: int = 0):
        super().__init__()
        seed = int(seed) & 0xFFFFFFFFFFFFFFFF
        rank = operator.index(rank)
        if not 0 <= rank < 1 << 32:
            raise ValueError("rank must be in [0, 2^32)")
        self.register_buffer("state", torch.tensor(
            [seed - (1 << 64) if seed >> 63 else seed, 0], dtype=torch.int64, device=device))
        # added to every offset: the bits of the rank, reversed, so that few
        # ranks lie far apart in the 64 bits
        self.rank, self.base = rank, int(f"{rank:064b}"[::-1], 2)
        self._sites = 0

    def site(self) -> int:
        """A new site number."""
        if self._sites + self._spares >= _SITES:
            raise RuntimeError("too many dropout sites")
        self._sites += 1
        return self._sites - 1

    def spare_site(self) -> int:
        """A new site number from the other end, for a place that does not drop
        yet: the numbers that site() gives do not depend on it."""
        if self._sites + self._spares >= _SITES:
            raise RuntimeError("too many dropout sites")
        self._spares += 1
        return _SITES - self._spares

    @torch.no_grad()
    def advance(self) -> None:
        self.state[1:].add_(_SITES)


def _generator(seed, offset):
    """(seed, offset, state) of a seed argument: an integer, a CounterRng or its tensor."""
    if isinstance(seed, CounterRng):
        return 0, operator.index(offset) + seed.base, seed.state
    if isinstance(seed, torch.Tensor):
        return 0, offset, seed
    return seed, offset, None


def dropout(x: torch.Tensor, p: float, *, seed=0, offset: int = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """residual + (kept ? x / (1 - p) : 0), one rounding; a dropped element is
    zero whatever x holds.  Element i (row-major) is kept as a function of
    (seed, offset, i) alone.  ``seed``: an int, a :class:`CounterRng` or a CUDA
    int64 tensor (seed, offset).  x: FP32, bf16 or fp16, any strides (the
    result is contiguous); residual: x's shape and dtype."""
    seed, offset, state = _generator(seed, offset)
    return _lib.host().nn_dropout(x, p, seed, offset, state, residual)


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, *,
              padding_idx: int | None = None, p: float = 0.0, seed=0, offset: int = 0,
              out_dtype: torch.dtype | None = None, grad_in_place: bool = False) -> torch.Tensor:
    """drop(scale * weight[tokens]) in one pass, rounded once to ``out_dtype``
    (default: weight's).  Dropout as in :func:`dropout` over the result's
    elements.  The gradient of ``weight`` is dense, summed by sorted tokens in
    FP32 in a fixed order; ``padding_idx`` gets none.

    A token outside the table makes its row NaN and a later call raise
    IndexError (``kernels.check_tokens``); its gradient is left out.

    ``grad_in_place``: when ``weight`` already has a ``.grad`` (as under
    ``ShardedDFCAdamW``, which owns it), backward adds the touched rows to it
    directly instead of returning a dense gradient to be added.  For leaf
    weights; ``torch.autograd.grad`` and hooks on the weight's gradient get a
    dense gradient all the same (hooks that run after its accumulation find the
    rows in ``.grad``).  The rows are added on the stream that ran this forward.
    They are ordered with gradients that reach the weight in other ways, and
    what the caller of ``backward()`` launches next on its stream sees them.
    The buffer must have been zeroed on the stream that ran this forward, or be
    ordered before it.
    """
    seed, offset, state = _generator(seed, offset)
    return _lib.host().nn_embedding(tokens, weight, scale, padding_idx, p, seed, offset, state,
                                    out_dtype, grad_in_place)


class Dropout(torch.nn.Module):
    """Dropout at one site of a :class:`CounterRng`; identity (plus the
    residual) in eval mode.  Called twice between two ``advance()``, it draws
    the same mask twice: give each place of a step a module of its own."""

    def __init__(self, p: float, rng: CounterRng):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("dropout probability must be in [0, 1]")
        self.p, self.rng, self.site = float(p), rng, rng.site()

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        return dropout(x, self.p, seed=self.rng, offset=self.site, residual=residual)

    def extra_repr(self) -> str:
        return f"p={self.p}, site={self.site}"


class Embedding(torch.nn.Module):
    """Token table with scaling and, in training, dropout in the same pass
    (arguments as for :func:`embedding`)."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None, *,
                 scale: float = 1.0, p: float = 0.0, rng: CounterRng | None = None,
                 out_dtype: torch.dtype | None = None, grad_in_place: bool = False, device=None,
                 dtype=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("dropout probability must be in [0, 1]")
        if p and rng is None:
            raise ValueError("dropout needs a CounterRng")
        if padding_idx is not None:
            if not -num_embeddings <= padding_idx < num_embeddings:
                raise ValueError("padding_idx must be within the table")
            padding_idx %= num_embeddings
        self.padding_idx, self.scale, self.p, self.rng = padding_idx, float(scale), float(p), rng
        self.site = 0 if rng is None else rng.site() if p else rng.spare_site()
        self.out_dtype, self.grad_in_place = out_dtype, grad_in_place
        self.weight = torch.nn.Parameter(torch.empty(num_embeddings, embedding_dim, device=device,
                                                     dtype=dtype))
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        torch.nn.init.normal_(self.weight)
        if self.padding_idx is not None:
            self.weight[self.padding_idx].zero_()

    def forward(self, tokens):
        p = self.p if self.training else 0.0
        if p and self.rng is None:
            raise ValueError("dropout needs a CounterRng")
        return embedding(tokens, self.weight, self.scale, padding_idx=self.padding_idx, p=p,
                         seed=self.rng if p else 0, offset=self.site, out_dtype=self.out_dtype,
                         grad_in_place=self.grad_in_place)

    def extra_repr(self) -> str:
        n, d = self.weight.shape
        return f"{n}, {d}, padding_idx={self.padding_idx}, scale={self.scale}, p={self.p}"
