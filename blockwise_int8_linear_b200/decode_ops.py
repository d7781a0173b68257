"""Model-side helpers for a decode step that sit between two of the library's kernels (the reference has no model code).

``rope_cache_append`` takes what a fused q/k/v ``BlockInt8Linear`` leaves for one new token per sequence, rotates q and k by
the position's angle and appends k and v to the caches in one launch (``bi8_rope_cache_append``); written with tensor
operations the same step is five launches per layer.

The same step for a cache held in 4 bits: ``int4_kv_cache`` allocates one, ``rope_cache_append_int4`` rotates and appends any number of
new tokens, ``attention_int4_cache`` attends to it.  The cache's blocks have 64 values, in the format of ``int4_functions``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

__all__ = ["rope_cache_append", "Int4KVCache", "int4_kv_cache", "rope_cache_append_int4", "attention_int4_cache"]


def rope_cache_append(qkv: torch.Tensor, cis: torch.Tensor, pos: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor) -> torch.Tensor:
    """``qkv [B, 3, H, D]`` (bf16 / fp16, contiguous): q, k, v of one new token per sequence.  ``cis [D/2]`` complex64 (or
    ``[D/2, 2]`` float32: cos, sin) of the step's position, ``pos`` an int64 device tensor with one element (the cache row),
    ``kcache`` / ``vcache [B, H, max_len, D]`` contiguous.  Returns the rotated q as ``[B, H, 1, D]``; row ``pos`` of the caches
    receives the rotated k and v.  Feature pairs are (even, odd) neighbours: ``(x0 + i x1) * cis``."""
    return _lib.native().rope_cache_append(qkv, cis, pos, kcache, vcache)


class Int4KVCache(NamedTuple):
    """Keys and values in 4-bit blocks of 64: codes uint8 ``[B, Hkv, max_len, D/2]`` and scales ``[B, Hkv, max_len, D/64]`` in the
    activations' type.  Rows of a head are dense, so views of some sequences, heads or first rows are caches too."""
    k: torch.Tensor
    k_state: torch.Tensor
    v: torch.Tensor
    v_state: torch.Tensor


def int4_kv_cache(batch: int, heads: int, max_len: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda") -> Int4KVCache:
    """An empty cache for ``heads`` key/value heads of ``head_dim`` (64, 128 or 256) features."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head size must be 64, 128 or 256, got {head_dim}")
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"the cache's scales must be bfloat16 or float16, got {dtype}")
    codes = lambda: torch.full((batch, heads, max_len, head_dim // 2), 0x88, device=device, dtype=torch.uint8)
    state = lambda: torch.zeros((batch, heads, max_len, head_dim // 64), device=device, dtype=dtype)
    return Int4KVCache(codes(), state(), codes(), state())


def rope_cache_append_int4(qkv: torch.Tensor, cis: torch.Tensor, pos: torch.Tensor, cache: Int4KVCache) -> torch.Tensor:
    """``qkv [B, T, Hq + 2 Hkv, D]`` (bf16 / fp16): q, k, v of T new tokens per sequence, as a fused projection leaves them.  ``cis
    [rows, D/2]`` complex64 (or ``[rows, D/2, 2]`` float32: cos, sin) is the table of all positions, ``pos`` an int64 device tensor
    with the first token's position, one for all sequences or ``[B]``.  Token t of a sequence has position and cache row ``pos + t``:
    q and k are rotated (feature pairs are (even, odd) neighbours, the result rounded to the activations' type), k and v
    quantized into the cache.  Returns the rotated q ``[B, Hq, T, D]``.  A position outside the cache or the table writes nothing and
    its query is zero.  Other rows stay what they are."""
    return _lib.native().rope_cache_append_int4(qkv, cis, pos, cache.k, cache.k_state, cache.v, cache.v_state)


def attention_int4_cache(q: torch.Tensor, cache: Int4KVCache, lengths: torch.Tensor, *, starts: torch.Tensor = None, scale: float = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` of ``q [B, Hq, T, D]`` over the cache; query head h reads cache head ``h // (Hq / Hkv)``.

    ``lengths`` (int64 on the device, one element or ``[B]``): how many rows a sequence has, the last T of which are the queries' own:
    query t sees the rows up to ``lengths - T + t`` (T = 1: all of them).  ``starts`` (the same form): the first row that is seen, for
    batches padded on the left or a window.  A query that sees no row gives zeros; rows that it does not see may hold anything.  Keys of
    2^100 and more may overflow in the scores, which are fp32.  ``scale``
    is a number of at most 2e38, by default ``1 / sqrt(D)``.  Lengths and starts are read by the kernel, so the call can be replayed from a
    CUDA graph while they change."""
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    return _lib.native().attention_int4(q, cache.k, cache.k_state, cache.v, cache.v_state, lengths, starts, scale)
