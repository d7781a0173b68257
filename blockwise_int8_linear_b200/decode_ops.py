"""Model-side helpers for a decode step that sit between two of the library's kernels (the reference has no model code).

``rope_cache_append`` takes what a fused q/k/v ``BlockInt8Linear`` leaves for one new token per sequence, rotates q and k by
the position's angle and appends k and v to the caches in one launch (``bi8_rope_cache_append``); written with tensor
operations the same step is five launches per layer.

The same step for a cache held in 4 bits: ``int4_kv_cache`` allocates one, ``rope_cache_append_int4`` rotates and appends any number of
new tokens, ``attention_int4_cache`` attends to it.  The cache's blocks have 64 values, in the format of ``int4_functions``.

A 16-bit cache in pages, for batches whose sequences come, grow and go: ``paged_kv_cache`` allocates one, ``rope_cache_append_paged`` rotates and
appends the new tokens of any number of sequences, packed one behind the other, ``attention_paged_cache`` attends to their pages, single tokens
and parts of prompts in one call.

The rotation by itself, for training and for models without these caches: ``rope``, with its gradient, in both layouts of feature pairs and for
a part of the head; ``rope_table`` makes the angles of all positions, stretched for long contexts where wanted.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib

__all__ = ["rope_cache_append", "Int4KVCache", "int4_kv_cache", "rope_cache_append_int4", "attention_int4_cache", "rope_table", "rope", "PagedKVCache",
           "paged_kv_cache", "rope_cache_append_paged", "attention_paged_cache"]


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


_LAYOUTS = {"interleaved": _lib.ROPE_INTERLEAVED, "half": _lib.ROPE_HALF}


def _layout(name: str) -> int:
    if name not in _LAYOUTS:
        raise ValueError(f"layout must be 'interleaved' or 'half', got {name!r}")
    return _LAYOUTS[name]


def rope_table(rows: int, features: int, *, base: float = 10000.0, factor: float = 1.0, parts=None, magnitude: float = 1.0, device="cuda") -> torch.Tensor:
    """The rotation of positions 0 to ``rows - 1`` for ``features`` rotated features, complex64 ``[rows, features/2]``: pair j of position p has the
    angle ``p * base**(-2j/features) / factor``, computed in 64 bits, and the length ``magnitude``.

    ``factor`` stretches all positions for contexts that long times the trained one.  With ``parts = (trained, low, high)`` only slow pairs
    are stretched: a pair that makes ``high`` turns or more over the ``trained`` positions keeps its angles, one that makes ``low`` or fewer is
    stretched fully, between them the inverse wavelength goes linearly from one to the other."""
    if rows < 0 or features < 2 or features % 2:
        raise ValueError(f"expected rows and an even number of features, got {rows} and {features}")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor) and math.isfinite(magnitude)):
        raise ValueError(f"base and factor must be positive numbers and magnitude a number, got {base}, {factor} and {magnitude}")
    step = base ** (-torch.arange(0, features, 2, device=device, dtype=torch.float64) / features)
    if parts is None:
        step = step / factor
    else:
        trained, low, high = parts
        if not (trained > 0 and 0 <= low < high):
            raise ValueError(f"parts must be (trained positions, low, high) with low below high, got {parts}")
        keep = ((trained * step / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        step = keep * step + (1.0 - keep) * step / factor
    angle = torch.arange(rows, device=device, dtype=torch.float64)[:, None] * step
    return torch.complex((angle.cos() * magnitude).float(), (angle.sin() * magnitude).float())


def rope(x: torch.Tensor, cis: torch.Tensor, positions: torch.Tensor = None, *, layout: str = "interleaved") -> torch.Tensor:
    """``x [B, T, H, D]`` or ``[T, H, D]`` (bf16, fp16 or fp32) with the first R features of every head turned by the angles of the token's position,
    the others as they are; the result is dense and of x's type.

    ``cis [rows, R/2]`` complex64 (or ``[rows, R/2, 2]`` float32: cos, sin) is the table of all positions, R even and at most D.  ``positions``:
    int64 on the device, ``[T]`` for all sequences or ``[B, T]``; by default 0 to T - 1.  ``layout``: pairs are neighbours ("interleaved") or R/2
    features apart ("half").  fp32 products and sums are each rounded on their own, the result once.  A token whose position the table does not
    have is zero, and so is its gradient.

    x's gradient is the rotation the other way, and can be differentiated again; the table has none and is refused if it wants one.  Any strides
    are read as they are where features are dense; rows that begin on 16-byte boundaries, with R and D multiples of 16, are read fastest."""
    return _lib.native().rope(x, cis, positions, _layout(layout))


class PagedKVCache(NamedTuple):
    """Keys and values in pages: ``[pages, Hkv, page_size, D]`` each, bf16 or fp16, features dense.  Other steps are free as long as no two values
    share memory, so one tensor may hold both, or have its dimensions in another order."""
    k: torch.Tensor
    v: torch.Tensor


def paged_kv_cache(pages: int, heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda") -> PagedKVCache:
    """``pages`` pages of ``page_size`` rows (a multiple of 16) for ``heads`` key/value heads of ``head_dim`` (64, 128 or 256) features.  A page's
    rows hold nothing until they are appended: the memory is not cleared."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head size must be 64, 128 or 256, got {head_dim}")
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"the cache must be bfloat16 or float16, got {dtype}")
    if page_size < 16 or page_size % 16:
        raise ValueError(f"pages must have a multiple of 16 rows, got {page_size}")
    return PagedKVCache(*(torch.empty((pages, heads, page_size, head_dim), device=device, dtype=dtype) for _ in range(2)))


def rope_cache_append_paged(qkv: torch.Tensor, cis: torch.Tensor, cache: PagedKVCache, pages: torch.Tensor, lengths: torch.Tensor,
                            cu_tokens: torch.Tensor = None, *, layout: str = "interleaved") -> torch.Tensor:
    """``qkv [N, Hq + 2 Hkv, D]`` (bf16 / fp16): q, k, v of the new tokens of B sequences, one sequence behind the other, as a fused projection leaves
    them.  Rotates q and k as ``rope`` does (R a multiple of 16), puts k and v into their sequences' pages and returns the rotated q ``[N, Hq, D]``.

    ``pages`` int32 ``[B, width]``: row r of a sequence is row ``r % page_size`` of page ``pages[b, r // page_size]``.  ``lengths`` (int64, one element
    or ``[B]``): rows that a sequence has with its new tokens, which are the last; the first of its n has position and row ``lengths - n``.
    ``cu_tokens`` (int64 ``[B + 1]``, from 0): the tokens of sequence b are ``cu_tokens[b]`` to ``cu_tokens[b + 1] - 1``, those behind the last
    sequence's belong to nobody; without it every sequence has N / B.  All are read by the kernel, so the call can be replayed from a CUDA
    graph while they change.

    A token whose position is outside the table of angles or its row of ``pages``, or whose page is none of the cache's, writes nothing, and its
    query is zero; so are the queries of tokens that belong to nobody.  Other rows of the cache stay what they are.  Sequences that append to the same row
    of a page leave either's values there."""
    return _lib.native().rope_cache_append_paged(qkv, cis, cache.k, cache.v, pages, lengths, cu_tokens, _layout(layout))


def attention_paged_cache(q: torch.Tensor, cache: PagedKVCache, pages: torch.Tensor, lengths: torch.Tensor, cu_tokens: torch.Tensor = None, *,
                          starts: torch.Tensor = None, scale: float = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` of ``q [N, Hq, D]``, the new tokens' queries, over their sequences' pages; query head h reads cache head
    ``h // (Hq / Hkv)``.  ``pages``, ``lengths`` and ``cu_tokens`` as in ``rope_cache_append_paged``, so that one sequence may bring a part of
    its prompt and another a single token.

    The query of a sequence's token i of n sees the rows up to ``lengths - n + i``, its own.  ``starts`` (as ``lengths``): the first row that is seen.  A
    query that sees no row gives zeros, as do tokens that belong to nobody; rows that it does not see may hold anything.  Infinite values that it sees
    give nothing finite in their feature.  A page number that is none of the cache's reads as a page of zeros.  Scores are fp32 and overflow where
    ``q k^T`` does, before the scale.  ``scale`` is a number of at most 2e38, by default ``1 / sqrt(D)``.

    Statistics and sums are fp32.  In a sequence with up to 16 queries on a cache head (new tokens times ``Hq / Hkv``) each weight enters the product with v as two
    numbers of the cache's type, and the result is off by its own rounding; with more queries as one, which adds up to half a step of the type
    times ``sum p |v|`` and on average 0.7 to 1 times that rounding again.

    A call is planned from its tensors' sizes, since lengths are on the device.  For single tokens, tables much wider than the sequences and tokens that belong to
    nobody cost time: 32 sequences of 600 rows on 8 heads take 20 us, with tables of 32768 rows 43, with 7 unused tokens 28; one of 131072 rows 90 us, with
    unused tokens three times that."""
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    return _lib.native().attention_paged(q, cache.k, cache.v, pages, lengths, cu_tokens, starts, scale)
