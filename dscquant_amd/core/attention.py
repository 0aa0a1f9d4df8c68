"""Attention block on the W4A4 path with a 4-bit paged key/value cache.

The reference quantizes the q, k, v and o projections of a Llama layer, each through its
own QuantLinear with the v / o rotation folded in (core/linear.py:22-52), and leaves what
lies between them to the model (core/model_ops.py:18-29 runs it).  ``QuantAttention``
keeps the four modules and runs

    q, k, v = q(x), k(x), v(x)                            (W4A4 linears)
    q = kv4.append(cache, q, k, v, ...)                   position, rotation, 4 bits, pages
    y = kv4.attention(cache, q, ...)                      causal, over the 4-bit pages
    o(y)                                                  (W4A4 linear)

for the new tokens of any number of sequences: whole prompts, chunks of them, single
tokens, mixed.  What the layers of one pass share -- where its tokens go, which pages they
see -- is a ``Step``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import nn

from .. import kv4
from .linear import QuantLinear


class Step(NamedTuple):
    """One pass over new tokens of B sequences; the same for every layer.

    ``slots`` int64 [T] and ``positions`` int64 [T]: each token's place in the cache and
    its row of ``cos`` / ``sin`` (fp32 [rows, R / 2]; None: no position rotation).
    ``tables`` int32 [B, width], ``lengths`` int32 [B], ``starts`` int32 [B + 1] or None,
    ``max_q``, ``max_length``: as ``kv4.attention``.  For a captured graph the tensors are
    updated in place and ``max_length`` is a bound for all replays."""
    slots: torch.Tensor
    positions: Optional[torch.Tensor]
    tables: torch.Tensor
    lengths: torch.Tensor
    starts: Optional[torch.Tensor]
    max_q: int
    max_length: int
    cos: Optional[torch.Tensor] = None
    sin: Optional[torch.Tensor] = None


def step(tables: torch.Tensor, cached, new, page_size: int, cos=None, sin=None) -> Step:
    """The step that adds ``new[b]`` tokens to each sequence b of ``cached[b]`` tokens (lists
    of ints); ``tables`` int32 [B, width] already holds the pages of both.  A token's position
    is its place in its sequence."""
    cached, new = [int(n) for n in cached], [int(n) for n in new]
    B, width = tables.shape
    if len(cached) != B or len(new) != B:
        raise RuntimeError(f"step: {B} sequences have tables, {len(cached)} and {len(new)} counts")
    if min([0, *cached, *new]) < 0:
        raise RuntimeError("step: a sequence has no negative number of tokens")
    lengths = [a + n for a, n in zip(cached, new)]
    if max([0, *lengths]) > width * page_size:
        raise RuntimeError(f"step: {max(lengths)} tokens do not fit {width} pages of {page_size}")
    count = torch.tensor(new, dtype=torch.int64)
    starts = torch.cat((torch.zeros(1, dtype=torch.int64), count.cumsum(0)))
    sequences = torch.repeat_interleave(torch.arange(B), count)
    places = torch.arange(sequences.numel()) + (torch.tensor(cached, dtype=torch.int64)
                                                - starts[:-1])[sequences]
    dev = tables.device
    sequences, places = sequences.to(dev), places.to(dev)
    one = all(n == 1 for n in new)
    return Step(kv4.slots(tables, sequences, places, page_size), None if cos is None else places,
                tables, torch.tensor(lengths, dtype=torch.int32, device=dev),
                None if one else starts.to(torch.int32).to(dev), max([1, *new]),
                max([0, *lengths]), cos, sin)


class QuantAttention(nn.Module):
    """q, k, v and o projections (QuantLinear) with 4-bit causal attention between them.

    ``heads`` query heads share ``kv_heads`` key/value heads of ``head_dim`` (64 or 128).
    ``rotate`` (default) stores the keys rotated by the Sylvester Hadamard matrix, which
    spreads the few large channels of keys over their row before it is quantized; values
    can carry the learned v / o rotation of the layer's interface.  ``interleaved`` and
    ``window`` as in ``kv4``.  fp16 and bf16."""

    def __init__(self, q: QuantLinear, k: QuantLinear, v: QuantLinear, o: QuantLinear, heads: int,
                 kv_heads: int, head_dim: int, rotate: bool = True, interleaved: bool = False,
                 window: int = 0, scale=None):
        super().__init__()
        rows = [m.base.weight.shape[0] for m in (q, k, v)]
        if rows != [heads * head_dim, kv_heads * head_dim, kv_heads * head_dim]:
            raise RuntimeError(f"QuantAttention: {heads} and {kv_heads} heads of {head_dim} need "
                               f"projections of other sizes (got {rows})")
        if o.base.weight.shape[1] != heads * head_dim:
            raise RuntimeError("QuantAttention: the o projection takes "
                               f"{o.base.weight.shape[1]} of {heads * head_dim} elements")
        self.q, self.k, self.v, self.o = q, k, v, o
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.rotate, self.interleaved, self.window, self.scale = rotate, interleaved, window, scale

    def new_cache(self, pages: int, page_size: int) -> torch.Tensor:
        """An empty cache for this layer, on its device."""
        return kv4.new_cache(pages, page_size, self.kv_heads, self.head_dim,
                             self.k.base.weight.device)

    def forward(self, x: torch.Tensor, cache: torch.Tensor, step: Step) -> torch.Tensor:
        """``x`` [T, hidden], the new tokens of all sequences one after another; the cache is
        updated in place."""
        T, D = x.shape[0], self.head_dim
        q = self.q(x).reshape(T, self.heads, D)
        k = self.k(x).reshape(T, self.kv_heads, D)
        v = self.v(x).reshape(T, self.kv_heads, D)
        q = kv4.append(cache, q, k, v, step.slots, step.positions, step.cos, step.sin,
                       self.interleaved, self.rotate)
        y = kv4.attention(cache, q, step.tables, step.lengths, step.starts, step.max_q,
                          step.max_length, self.scale, self.window)
        return self.o(y.reshape(T, self.heads * D))
