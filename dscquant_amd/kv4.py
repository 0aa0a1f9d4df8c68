"""The 4-bit paged key/value cache of an attention layer.

    new_cache(pages, page_size, heads, head_dim, device)
                          -> u8 [pages, heads, page_size, head_dim + 8]
    append(cache, q, k, v, slots, ...)    a step's rows into their slots, q turned and rotated
    attention(cache, q, tables, ...)      a ragged batch's queries over their pages
    read(cache, slots, dtype)             cached tokens as 16-bit rows
    slots(tables, sequences, places, page_size)   the slots of tokens, once a step for all layers

Between the q/k/v projections and o of a layer (core/linear.py:22-46 folds the transforms
of v and o) the reference runs attention in torch on 16-bit keys and values; here they are
kept at 4 bits by the rule of its activations (core/quantization.py:13-21), a scale and a
zero-point for each row of a head: (head_dim + 8) / (4 head_dim) of their 16-bit size.
Layout, rule and limits: include/dscq.h.  Keys and values enter the products as the whole
numbers their codes stand for, so attention reads the cache as it is and rounds nothing of
it; the softmax's weights enter theirs as fp16.  Kernels run on torch's current stream; outputs and scratch come from torch's
allocator, so the calls can be captured in a HIP graph.  There is no gradient: the cache
serves inference, as the integer linear path does.
"""
from __future__ import annotations

import math

import torch

from . import _lib

__all__ = ["new_cache", "append", "read", "attention", "slots"]

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_NO_GRAD = "the 4-bit cache is inference-only (codes carry no gradient)"


def _check_layout(page_size: int, heads: int, head_dim: int) -> None:
    if head_dim not in (64, 128):
        raise RuntimeError(f"kv4: head_dim must be 64 or 128 (got {head_dim})")
    if page_size < 16 or page_size % 16 or page_size > 4096:
        raise RuntimeError(f"kv4: page size must be a multiple of 16 up to 4096 (got {page_size})")
    if not 0 < heads <= 1024:
        raise RuntimeError(f"kv4: 1 to 1024 key/value heads (got {heads})")


def new_cache(pages: int, page_size: int, heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """An empty cache of ``pages`` pages of ``page_size`` tokens for one layer."""
    _check_layout(page_size, heads, head_dim)
    if pages <= 0:
        raise RuntimeError(f"kv4: a cache has at least one page (got {pages})")
    return torch.zeros((pages, heads, page_size, head_dim + 8), dtype=torch.uint8, device=device)


def _check_cache(cache: torch.Tensor):
    """(pages, heads, page size, head_dim) of a cache tensor."""
    if not (cache.is_cuda and cache.is_contiguous()):
        raise RuntimeError("Expected contiguous CUDA tensor")
    if cache.dtype != torch.uint8 or cache.dim() != 4 or cache.size(0) == 0:
        raise RuntimeError("kv4: the cache is u8 [pages, heads, page_size, head_dim + 8]")
    pages, heads, page_size, row = cache.shape
    _check_layout(page_size, heads, row - 8)
    return pages, heads, page_size, row - 8


# The checks read each property of a tensor once (a call's host time is its checks, its
# allocations and the call through ctypes) and look for what is wrong only if something is.

def _rows(name: str, x: torch.Tensor, index: int, shape) -> tuple:
    """The strides of rows [tokens, heads, head_dim] on device ``index``."""
    if x.shape == shape and x.dtype in _DTYPES and x.get_device() == index:
        strides = x.stride()
        if strides[2] == 1 or not x.numel():
            if x.requires_grad and torch.is_grad_enabled():
                raise RuntimeError(_NO_GRAD)
            return strides
    if x.get_device() != index:
        raise RuntimeError("All buffers must be on the same device")
    if x.dtype not in _DTYPES:
        raise RuntimeError("Only FP16 and BF16 inputs are supported")
    if x.shape != shape:
        raise RuntimeError(f"kv4: {name} must be {list(shape)} (got {list(x.shape)})")
    raise RuntimeError(f"kv4: the elements of a head of {name} must be contiguous")


def _heads(name: str, x: torch.Tensor, dim: int) -> int:
    if x.dim() != 3:
        raise RuntimeError(f"kv4: {name} must be [tokens, heads, {dim}] (got {list(x.shape)})")
    return x.size(1)


def _check_index(name: str, t: torch.Tensor, index: int, dtype, shape) -> None:
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return
    if t.get_device() != index:
        raise RuntimeError("All buffers must be on the same device")
    raise RuntimeError(f"kv4: {name} must be contiguous {str(dtype)[6:]} {list(shape)} "
                       f"(got {str(t.dtype)[6:]} {list(t.shape)})")


def slots(tables: torch.Tensor, sequences: torch.Tensor, places: torch.Tensor,
          page_size: int) -> torch.Tensor:
    """The slots (int64) of the tokens at ``places`` of ``sequences`` (int64, one entry a
    token) in the pages of ``tables`` [B, width]: what ``append`` and ``read`` take.  The
    same for every layer of a step."""
    return tables[sequences, places // page_size].long() * page_size + places % page_size


def append(cache: torch.Tensor, q, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
           positions=None, cos=None, sin=None, interleaved: bool = False, rotate: bool = False):
    """A step's keys and values into the cache; returns the queries for ``attention``.

    ``q`` [T, Hq, D] (or None: None is returned), ``k``, ``v`` [T, H, D]: fp16 or bf16, each
    head's elements contiguous, any strides above (parts of one q|k|v product).  ``slots``
    int64 [T], distinct; a slot outside the cache leaves its token out (a place of a new cache
    that nothing was stored in is a key and a value of zeros to who sees it).  With ``cos``,
    ``sin`` (fp32 [rows, R / 2], R a multiple of 16 up to D) the first R elements of each
    head of q and k are turned by the row ``positions`` (int64 [T]) names: pairs
    (i, i + R / 2), or (2 i, 2 i + 1) if ``interleaved``.  A position outside the table:
    NaN queries, nothing stored.  ``rotate`` stores H_D k and returns H_D q / D (the same
    scores; the activations' Hadamard for keys with a few large channels)."""
    pages, H, P, D = _check_cache(cache)
    dev = cache.get_device()
    T = k.size(0)
    k_strides = _rows("k", k, dev, (T, H, D))
    v_strides = _rows("v", v, dev, (T, H, D))
    if v.dtype is not k.dtype or (q is not None and q.dtype is not k.dtype):
        raise RuntimeError("kv4: q, k and v must have the same dtype")
    Hq, q_args, out = 0, (None, 0, 0), None
    if q is not None:
        Hq = _heads("q", q, D)
        q_strides = _rows("q", q, dev, (T, Hq, D))
        if Hq == 0 or Hq > 4096:
            raise RuntimeError(f"kv4: 1 to 4096 query heads (got {Hq})")
        q_args = (q.data_ptr(), q_strides[0], q_strides[1])
    _check_index("slots", slots, dev, torch.int64, (T,))
    turn = (None, None, None, 0, 0)
    if cos is not None or sin is not None or positions is not None:
        if cos is None or sin is None or positions is None:
            raise RuntimeError("kv4: cos, sin and positions go together")
        rows, half = cos.shape if cos.dim() == 2 else (0, 0)
        if rows == 0 or half % 8 or not 8 <= half <= D // 2:
            raise RuntimeError("kv4: cos and sin must be [rows, R / 2] with R a multiple of 16 "
                               f"up to {D} (got {list(cos.shape)})")
        _check_index("cos", cos, dev, torch.float32, (rows, half))
        _check_index("sin", sin, dev, torch.float32, (rows, half))
        _check_index("positions", positions, dev, torch.int64, (T,))
        turn = (positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), rows, 2 * half)
    device = cache.device
    _lib.require_gfx950(device)
    if q is not None:
        out = q.new_empty((T, Hq, D))
    if T == 0:
        return out
    with _lib.on(device):
        _lib.call("dscq_kv_append", *q_args, k.data_ptr(), k_strides[0], k_strides[1], v.data_ptr(),
                  v_strides[0], v_strides[1], _DTYPES[k.dtype], T, Hq, H, D, *turn,
                  1 if interleaved else 0, 1 if rotate else 0, slots.data_ptr(), cache.data_ptr(),
                  pages, P, None if out is None else out.data_ptr(), _lib.stream(device))
    return out


def read(cache: torch.Tensor, slots: torch.Tensor, dtype=torch.float16, rotate: bool = False):
    """Cached tokens as rows: (k, v) [T, H, D] of ``dtype`` (fp16 or bf16) at ``slots`` int64
    [T]; zeros for a slot outside the cache.  ``rotate`` as they were appended: keys come
    back in the model's own basis."""
    pages, H, P, D = _check_cache(cache)
    if dtype not in _DTYPES:
        raise RuntimeError("Only FP16 and BF16 inputs are supported")
    T, dev = slots.numel(), cache.device
    _check_index("slots", slots, cache.get_device(), torch.int64, (T,))
    _lib.require_gfx950(dev)
    k = torch.empty((T, H, D), dtype=dtype, device=dev)
    v = k.new_empty((T, H, D))
    if T:
        with _lib.on(dev):
            _lib.call("dscq_kv_read", cache.data_ptr(), pages, P, H, D, slots.data_ptr(), T,
                      1 if rotate else 0, _DTYPES[dtype], k.data_ptr(), v.data_ptr(),
                      _lib.stream(dev))
    return k, v


def attention(cache: torch.Tensor, q: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
              starts=None, max_q: int = 1, max_length=None, scale=None, window: int = 0,
              return_lse: bool = False):
    """Causal attention of a ragged batch over the cache: [T, Hq, D] of q's dtype.

    ``q`` [T, Hq, D] fp16 or bf16 (what ``append`` returned); query head h reads cache head
    h / (Hq / H).  ``tables`` int32 [B, width]: each sequence's pages; ``lengths`` int32 [B]:
    its cached tokens, the new ones among them.  ``starts`` int32 [B + 1]: its queries are
    rows starts[b] .. starts[b + 1] - 1, the last ones of its tokens; None: one query a
    sequence.  ``max_q`` and ``max_length`` (default: what the tables hold) bound a
    sequence's queries and length on the host, which plans the launch by them.  ``scale``
    defaults to D ** -0.5; ``window`` > 0: a query sees that many tokens, its own the last.
    A query that sees none gives zeros, and so do rows of no sequence and queries past
    ``max_q``.  ``return_lse``: also the logarithm of each query's softmax sum, fp32 [T, Hq]
    (-inf for one that sees none), with which results over parts of a context are joined."""
    pages, H, P, D = _check_cache(cache)
    index = cache.get_device()
    T, Hq = q.size(0), _heads("q", q, D)
    strides = _rows("q", q, index, (T, Hq, D))
    if Hq == 0 or Hq % H or Hq > 4096:
        raise RuntimeError("kv4: query heads must be a multiple of the cache's heads, up to 4096")
    if tables.dim() != 2 or tables.size(0) > 65535:
        raise RuntimeError("kv4: tables must be [B, width] with B up to 65535")
    B, width = tables.shape
    _check_index("tables", tables, index, torch.int32, (B, width))
    _check_index("lengths", lengths, index, torch.int32, (B,))
    max_q, window = int(max_q), int(window)
    if starts is not None:
        _check_index("starts", starts, index, torch.int32, (B + 1,))
    elif max_q != 1 or T != B:
        raise RuntimeError("kv4: without starts every sequence has one query")
    max_length = width * P if max_length is None else int(max_length)
    if max_q < 0 or max_length < 0 or window < 0:
        raise RuntimeError("kv4: max_q, max_length and window must not be negative")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < 3.0e38:
        raise RuntimeError(f"kv4: scale must be positive (got {scale})")
    dev = cache.device
    _lib.require_gfx950(dev)
    out = q.new_empty((T, Hq, D))
    lse = q.new_empty((T, Hq), dtype=torch.float32) if return_lse else None
    if T:
        with _lib.on(dev):
            # The plan, and with it the scratch, depends on the device's compute units.
            need = int(_lib.lib().dscq_kv_attention_workspace_bytes(B, Hq, H, D, max_q, max_length,
                                                                    window))
            ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need > 0 else None
            _lib.call("dscq_kv_attention", q.data_ptr(), strides[0], strides[1], _DTYPES[q.dtype],
                      T, Hq, cache.data_ptr(), pages, P, H, D, _lib.ptr(tables), width,
                      lengths.data_ptr(), None if starts is None else starts.data_ptr(), B, max_q,
                      max_length, scale, window, out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws),
                      max(need, 0),
                      _lib.stream(dev))
    return (out, lse) if return_lse else out
