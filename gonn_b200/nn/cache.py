"""Rotary positions and a paged cache of keys and values, for generating token by token."""
from __future__ import annotations

from typing import Optional

import torch

from ..ops import cache as _cache
from ..ops.rotary import frequencies, rotary, turns_of
from .module import Module


class RotaryEmbedding(Module):
    """Turns the pairs of a head's first ``dim`` columns by the token's position: (a, b) at position p becomes
    (a cos - b sin, a sin + b cos) * ``amplitude`` with the angle p w_i, w_i = base^(-2 i / dim).  Pair i is columns (i, i + dim / 2), or
    (2 i, 2 i + 1) if ``interleaved``; columns from ``dim`` on stay as they are.  No parameters.

    ``scaling``, for longer contexts than a model was trained on:
      "linear"  w_i / factor
      "base"    base * factor^(dim / (dim - 2)) in the base's place
      "bands"   w_i (g + (1 - g) / factor), g = (original w_i / 2 pi - low) / (high - low) kept within 0 and 1: pairs that turn at least
                ``high`` times over ``original`` positions keep their frequency, those below ``low`` times have it divided"""

    def __init__(self, dim: int, base: float = 10000.0, *, interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
                 original: int = 0, low: float = 1.0, high: float = 32.0, amplitude: float = 1.0, device=None):
        super().__init__()
        if dim < 2 or dim % 2 or dim > 2048:
            raise ValueError(f"RotaryEmbedding: dim must be an even number from 2 to 2048, got {dim}")
        if scaling not in ("none", "linear", "base", "bands"):
            raise ValueError(f"RotaryEmbedding: scaling is 'none', 'linear', 'base' or 'bands', not {scaling!r}")
        if not (base > 0 and factor > 0 and amplitude > 0):
            raise ValueError("RotaryEmbedding: base, factor and amplitude must be positive")
        if scaling == "base" and dim == 2:
            raise ValueError("RotaryEmbedding: scaling by the base needs more than one pair")
        if scaling == "bands" and (original < 1 or not high > low):
            raise ValueError("RotaryEmbedding: bands need the original number of positions and high > low")
        self.dim, self.base, self.interleaved, self.amplitude = dim, float(base), bool(interleaved), float(amplitude)
        self.scaling, self.factor, self.original, self.low, self.high = scaling, float(factor), original, float(low), float(high)
        self._w = frequencies(dim, self.base, scaling, self.factor, original, self.low, self.high)
        self.turns = turns_of(self._w).to(device)              # (no buffer: it follows from the options, whatever a checkpoint holds)

    def _apply(self, fn, *a, **kw):
        r = super()._apply(fn, *a, **kw)
        self.turns = fn(self.turns)
        return r

    def forward(self, x, positions: Optional[torch.Tensor] = None):
        """x (batch, tokens, heads, width) with any strides, bf16, fp16 or fp32 on CUDA; positions int32 or int64, (tokens,) or
        (batch, tokens), None for 0, 1, ...  Differentiable in x."""
        return rotary(x, positions, self._w, self.turns, self.interleaved, self.amplitude)

    def _plan(self):
        return self._w, self.turns, self.interleaved, self.amplitude


class KVCache:
    """Keys and values of many sequences in pages of ``page_size`` positions: two tensors (pages, heads, page size, head size), ``Keys``
    and ``Values``.  Which page holds what is the caller's: position p of sequence b lies in row p % page_size of page
    ``table[b, p // page_size]``.  ``lengths[b]`` positions are there before a call, token t of a call takes position lengths[b] + t.
    In a padded batch the first ``counts[b]`` tokens count.  table, lengths and counts are int32 tensors on the cache's device and are read there:
    calls neither synchronise nor depend on their values in any other way, so they may be captured and replayed.

    bf16, fp16 and fp32 on CUDA, heads of up to 128 columns and whole 16 bytes there; nothing has a gradient.  On CUDA a position behind
    its table's end or a page that is none of the cache's is reported by ``lib.assert_status_ok``: nothing is written there, and attention
    takes zeros (pages) or nothing (positions) in its place.  On the CPU it raises ValueError."""

    def __init__(self, pages: int, page_size: int, num_heads: int, head_dim: int, *, dtype=torch.float32, device=None):
        if min(pages, page_size, num_heads, head_dim) < 1:
            raise ValueError("KVCache: pages, page_size, num_heads and head_dim must be >= 1")
        shape = (pages, num_heads, page_size, head_dim)
        self._of = _cache.Layout(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    @classmethod
    def Over(cls, keys: torch.Tensor, values: torch.Tensor) -> "KVCache":
        """A cache in tensors that are there already."""
        c = cls.__new__(cls)
        c._of = _cache.Layout(keys, values)
        return c

    Keys = property(lambda self: self._of.keys)
    Values = property(lambda self: self._of.values)

    def Append(self, k, v, table, lengths, counts=None, rotary: Optional[RotaryEmbedding] = None, q=None):
        """Writes k and v (batch, tokens, heads, head size), any strides, to the pages of their sequences: k turned by ``rotary`` at its
        positions, if one is given.  ``q`` (batch, tokens, its heads, head size) is turned on the way and returned (zeros where a token does
        not count).  No two sequences may write the same row."""
        return _cache.append(self._of, k, v, table, lengths, counts, None if rotary is None else rotary._plan(), q)

    def Attend(self, q, table, lengths, counts=None, scale: Optional[float] = None, shared_pages: int = 0):
        """softmax(scale q K^T) V of q (batch, tokens, heads, head size) over its sequence's positions up to its own, keys and values of
        this call's tokens included: they have been appended.  heads may be a multiple of the cache's: query heads h n .. h n + n - 1 share key
        head h.  Zeros where a token does not count.  scale: 1 / sqrt(head size).  A value of a later token of the same call that is infinite or NaN
        may reach the earlier ones (0 times it), as in a plain product.

        ``shared_pages``: all sequences have the same first pages (a common prompt), which are taken from the table's first row and read
        once for many sequences: all those that have them whole; one that ends inside them is read by itself.  (bf16 and fp16 with more than 64
        rows, tokens times heads to a key head: once for each sequence.)"""
        return _cache.attend(self._of, q, table, lengths, counts, scale, shared_pages)
