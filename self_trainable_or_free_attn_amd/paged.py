"""Paged caches of keys and values in 16 or 4 bits: new tokens into one, their attention over it, rows back out of it
(include/paged_hip.h; the reference has no counterpart).

  PagedCache, paged_cache   the tensors of a cache, and an empty one
  append_paged              new tokens' keys and values into a cache, normed and rotated on the way, with their queries
  paged_attention           new tokens over all that the cache holds of their sequences, causal or not, grouped heads
  paged_rows                what a cache holds of its sequences' last tokens, as packed tokens

Sequences grow in pages of 16 to 4096 rows that stand anywhere in the cache: `pages` [B, max_pages] names those of each
sequence, `lens` [B] how many tokens it has, the new ones included. Both stay on the GPU (int32): no call synchronises, so all of
them can be captured into a graph and replayed with other lengths and pages. Tokens are bf16 or fp16 with D = 64 or 128.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .packed import _check_gpu, _check_heads, _check_ints, _check_tokens, _ops, _scale
from .rotary import _check_turn


class PagedCache(NamedTuple):
    """Keys and values in pages. 16 bits: k and v [num_pages, Hk, page_size, D] in the tokens' type, with any strides that both
    have, that leave the channels 1 apart and give each row memory of its own (a cache of [num_pages, page_size, Hk, D] is
    passed with its middle dimensions transposed), k_scales and v_scales None.

    4 bits: k and v are codes, uint8 [num_pages, Hk, page_size, D / 2], channel 2 i in the low half of byte i, and k_scales and
    v_scales uint8 [num_pages, Hk, page_size, D / 32], all contiguous. A code is a sign (bit 3) and the number of one of the
    magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6; 32 channels share the power of two 2 ** (scale - 127), scale 1 to 254 (the values must
    be within the type that the cache is read as)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scales: Optional[torch.Tensor] = None
    v_scales: Optional[torch.Tensor] = None


def paged_cache(num_pages: int, heads: int, dim: int, *, page_size: int = 64, bits: int = 16, dtype: torch.dtype = torch.bfloat16,
                device="cuda") -> PagedCache:
    """An empty cache of num_pages pages of page_size rows for `heads` key heads of `dim` channels: bits 16 in `dtype`, or 4 (a row
    of 128 channels then takes 68 bytes instead of 256)."""
    if dim not in (64, 128):
        raise ValueError(f"head dim must be 64 or 128, got {dim}")
    if num_pages < 0 or heads < 1:
        raise ValueError(f"num_pages must not be negative and heads positive, got {num_pages} and {heads}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be a power of two from 16 to 4096, got {page_size}")
    shape = (num_pages, heads, page_size)
    if bits == 4:
        zeros = lambda n, fill=0: torch.full((*shape, n), fill, dtype=torch.uint8, device=device)
        return PagedCache(zeros(dim // 2), zeros(dim // 2), zeros(dim // 32, 127), zeros(dim // 32, 127))
    if bits != 16:
        raise ValueError(f"bits must be 16 or 4, got {bits}")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    return PagedCache(*(torch.zeros(*shape, dim, dtype=dtype, device=device) for _ in "kv"))


PAGE_SIZES = frozenset(1 << i for i in range(4, 13))
MAX_TOKENS = 1 << 30      # that a row of `pages` can name


def _rows_apart(shape, strides, dim):
    """Whether rows of `dim` channels stand apart: each dimension steps over all that those of smaller strides hold."""
    dims = [(s, n) for n, s in zip(shape, strides) if n > 1]
    return all(s >= dim + sum((m - 1) * r for j, (r, m) in enumerate(dims) if j != i and r <= s) for i, (s, _) in enumerate(dims))


def _check_cache(cache, dtype, device, like):
    """(heads, page_size, dim) of a cache that holds tokens of `dtype`."""
    k, v, ks, vs = cache
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"cache.k and cache.v must have one shape [num_pages, heads, page_size, dim], got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    if k.device != device or v.device != device:
        raise ValueError(f"the cache is on {k.device} and {v.device}, {like} on {device}")
    pages, heads, size, dim = k.shape
    if size not in PAGE_SIZES:
        raise ValueError(f"the page size must be a power of two from 16 to 4096, got {size}")
    if (ks is None) != (vs is None):
        raise ValueError("k_scales and v_scales go together")
    if ks is not None:
        dim *= 2
        for name, x, n in (("k", k, dim // 2), ("v", v, dim // 2), ("k_scales", ks, dim // 32), ("v_scales", vs, dim // 32)):
            if x.dtype is not torch.uint8:
                raise TypeError(f"cache.{name} must be uint8 in a cache of 4 bits, got {x.dtype}")
            if x.shape != (pages, heads, size, n) or not x.is_contiguous():
                raise ValueError(f"cache.{name} must be a contiguous {(pages, heads, size, n)} tensor, got {tuple(x.shape)}")
            if x.device != device:
                raise ValueError(f"cache.{name} is on {x.device}, {like} on {device}")
    else:
        if k.dtype is not dtype or v.dtype is not dtype:
            raise TypeError(f"a cache of 16 bits must be {dtype} like the tokens, got {k.dtype} and {v.dtype}")
        if k.stride() != v.stride() or k.stride(3) != 1 or any(n > 1 and s % 8 for n, s in zip(k.shape[:3], k.stride())):
            raise ValueError(f"cache.k and cache.v must have the same strides, channels 1 apart and the others multiples of 8, got "
                             f"{k.stride()} and {v.stride()}")
        if not _rows_apart(k.shape[:3], k.stride(), dim):
            raise ValueError(f"rows of the cache must not overlap, got strides {k.stride()}")
    if dim not in (64, 128):
        raise ValueError(f"head dim must be 64 or 128, got {dim}")
    return heads, size, dim


def _check_places(pages, lens, cu, page_size, rows, device):
    """Number of sequences."""
    if pages.dtype is not torch.int32:
        raise TypeError(f"pages must be int32, got {pages.dtype}")
    if pages.dim() != 2 or not pages.is_contiguous():
        raise ValueError("pages must be a contiguous [sequences, pages] tensor")
    if pages.device != device:
        raise ValueError(f"pages is on {pages.device}, the tokens on {device}")
    B = pages.shape[0]
    if B < 1:
        raise ValueError("pages must name at least one sequence")
    if pages.shape[1] * page_size >= MAX_TOKENS:
        raise ValueError(f"a row of pages must name fewer than {MAX_TOKENS} tokens")
    _check_ints("lens", lens, device)
    if lens.shape[0] != B:
        raise ValueError(f"lens must hold {B} values like pages, got {lens.shape[0]}")
    if cu is not None:
        _check_ints("cu", cu, device)
        if cu.shape[0] != B + 1:
            raise ValueError(f"cu must hold {B + 1} values, got {cu.shape[0]}")
    elif rows % B:
        raise ValueError(f"without cu the {rows} tokens must divide into {B} equal counts")
    return B


def _check_append(cache, k, v, pages, lens, cu, q, q_weight, k_weight, table, eps):
    """The arguments of append_paged; eps."""
    dims = k.dim()
    if dims not in (3, 4) or k.shape != v.shape:
        raise ValueError(f"k and v must be [T, Hk, D], or both [B, n, Hk, D], got {tuple(k.shape)} and {tuple(v.shape)}")
    _check_tokens(k, (("v", v),) if q is None else (("v", v), ("q", q)))
    device = k.device
    heads, size, D = _check_cache(cache, k.dtype, device, "k")
    kshape = k.shape
    if kshape[-2] != heads or kshape[-1] != D:
        raise ValueError(f"the cache holds {heads} heads of {D}, k has {kshape[-2]} of {kshape[-1]}")
    if heads > 4096:
        raise ValueError(f"at most 4096 heads, got {heads}")
    rows = kshape[0] if dims == 3 else kshape[0] * kshape[1]
    B = _check_places(pages, lens, cu, size, rows, device)
    if dims == 4 and (cu is not None or kshape[0] != B):
        raise ValueError(f"[B, n, heads, D] tensors go without cu and with {B} sequences")
    if q is not None:
        shape = q.shape
        if q.dim() != dims or shape[:-2] != kshape[:-2] or shape[-1] != D:
            raise ValueError(f"q {tuple(shape)} and k {tuple(kshape)} do not go together")
        if not 0 < shape[-2] <= 4096:
            raise ValueError(f"q must have 1 to 4096 heads, got {shape[-2]}")
        if (q_weight is None) != (k_weight is None):
            raise ValueError("q_weight and k_weight go together")
    elif q_weight is not None:
        raise ValueError("q_weight goes with q")
    return _check_turn(k, D, q_weight, k_weight, table, eps)


def append_paged(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, lens: torch.Tensor,
                 cu: Optional[torch.Tensor] = None, *, q: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 halves: bool = False) -> Optional[torch.Tensor]:
    """Keys and values of new tokens into the cache, in place, and with q their queries normed and rotated, returned: one launch.

    k, v [T, Hk, D] and q [T, H, D]: packed tokens (column ranges of a projection's rows are read where they are), those of
    sequence b from cu[b] to cu[b + 1] - 1 (int32 [B + 1], running counts from 0); without cu T / B each, also as [B, n, heads, D].
    pages int32 [B, max_pages], lens int32 [B]: the sequence's tokens with the new ones, so token i of n has position
    lens[b] - n + i, which is held in row position % page_size of page pages[b, position // page_size]. Weights, table, eps and
    halves as in `norm_rotate`, for k (and q) at that position (past the table's last: as the last); without them k and q stay
    as they are.

    4 bits: keys are normed and rotated in 64 bits and rounded to float32, then every 32 channels of keys and values take the
    smallest power of two s with max |x| <= 7 s (2^-120 .. 2^120, for fp16 2^-13 .. 2^13) and the nearest of their values, ties
    to the even code. Values must be finite.

    Nothing is written for tokens behind the last sequence, of negative positions, past the named pages, or whose page number is
    outside the cache; q's rows of the first two are zeros. What a row holds that two tokens of a call share is not defined: pages
    may be shared for reading only. Returns the new q, contiguous and shaped like q, or None without q. There is no derivative: tensors
    that require a gradient are refused unless gradients are off."""
    if k.is_cuda and k.dim() == 3:      # the operator checks everything itself; what it refuses is named by the checks below
        try:
            out = _ops().append_paged(q, k, v, q_weight, k_weight, table, pages, lens, cu, *cache, bool(halves), eps)
        except (RuntimeError, TypeError):
            _check_append(cache, k, v, pages, lens, cu, q, q_weight, k_weight, table, eps)
            raise
        return None if q is None else out
    eps = _check_append(cache, k, v, pages, lens, cu, q, q_weight, k_weight, table, eps)
    _check_gpu(k)
    flat = (lambda x: x) if k.dim() == 3 else lambda x: x.flatten(0, 1)
    out = _ops().append_paged(None if q is None else flat(q), flat(k), flat(v), q_weight, k_weight, table, pages, lens, cu, *cache,
                              bool(halves), eps)
    return None if q is None else out.view(q.shape)


def paged_rows(cache: PagedCache, pages: torch.Tensor, lens: torch.Tensor, cu: Optional[torch.Tensor] = None, *, rows: int,
               dtype: Optional[torch.dtype] = None):
    """(k, v) [rows, Hk, D]: what the cache holds of each sequence's last tokens, packed: cu[b + 1] - cu[b] of sequence b (int32
    [B + 1]), without cu rows / B. pages and lens as in `append_paged`; with running counts of lens it returns every sequence
    whole. Zeros for rows behind the last sequence, tokens of negative positions or past the named pages, and pages outside the
    cache. dtype: of the result, bf16 or fp16, the cache's own by default and at 16 bits."""
    if dtype is None:
        dtype = cache.k.dtype if cache.k_scales is None else torch.bfloat16
    if cache.k.is_cuda:      # the operator checks everything itself; what it refuses is named by the checks below
        try:
            return _ops().paged_rows(*cache, pages, lens, cu, rows, dtype)
        except (RuntimeError, TypeError):
            _check_rows(cache, pages, lens, cu, rows, dtype)
            raise
    _check_rows(cache, pages, lens, cu, rows, dtype)
    _check_gpu(cache.k)
    return _ops().paged_rows(*cache, pages, lens, cu, rows, dtype)


def _check_rows(cache, pages, lens, cu, rows, dtype):
    """The arguments of paged_rows."""
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    device = cache.k.device
    _, size, _ = _check_cache(cache, dtype, device, "cache.k")
    if not 0 <= rows < MAX_TOKENS:
        raise ValueError(f"rows must be 0 to {MAX_TOKENS - 1}, got {rows}")
    _check_places(pages, lens, cu, size, rows, device)


def _check_attention(q, cache, pages, lens, cu, scale):
    """The arguments of paged_attention; the scale."""
    dims = q.dim()
    if dims not in (3, 4):
        raise ValueError(f"q must be [T, H, D] or [B, n, H, D], got {tuple(q.shape)}")
    _check_tokens(q, ())
    device, shape = q.device, q.shape
    heads, size, D = _check_cache(cache, q.dtype, device, "q")
    if shape[-1] != D:
        raise ValueError(f"the cache holds heads of {D} channels, q has {shape[-1]}")
    _check_heads(shape[-2], heads)
    rows = shape[0] if dims == 3 else shape[0] * shape[1]
    B = _check_places(pages, lens, cu, size, rows, device)
    if dims == 4 and (cu is not None or shape[0] != B):
        raise ValueError(f"[B, n, H, D] tensors go without cu and with {B} sequences")
    return _scale(scale, D)


def paged_attention(q: torch.Tensor, cache: PagedCache, pages: torch.Tensor, lens: torch.Tensor, cu: Optional[torch.Tensor] = None,
                    *, causal: bool = True, scale: Optional[float] = None, return_lse: bool = False):
    """Attention of new tokens over a cache that holds their own keys already (`append_paged`).

    q [T, H, D], H a multiple of the cache's heads, packed: sequence b has rows cu[b] to cu[b + 1] - 1 (int32 [B + 1]), without cu
    T / B each, also as [B, n, H, D]. pages and lens as in `append_paged`: lens[b] keys, the n new tokens' own the last of them.
    Token i sees them all, with causal those up to its position lens[b] - n + i. Single tokens, pieces of prompts and whole ones
    may share a call. scale: 1 / sqrt(D) if None.

    Keys past the named pages and of pages outside the cache are left out. Cache rows from lens[b] on are never used; the values in use must be finite
    (those of a 4-bit cache within q's type), scores below 2^22 in magnitude. Values of 4 bits are used exactly as they are held.

    Returns out like q, with return_lse also the natural-log LSE [T, H] ([B, n, H]) in float32; a token that sees no key, and rows
    behind the last sequence, give zeros and -inf. The same inputs give the same bits. There is no derivative: tensors that require
    a gradient are refused unless gradients are off."""
    if q.is_cuda and q.dim() == 3:      # the operator checks everything itself; what it refuses is named by the checks below
        try:
            out = _ops().paged_attention(q.contiguous(), *cache, pages, lens, cu, bool(causal),
                                         max(q.shape[2], 1) ** -0.5 if scale is None else scale)
        except (RuntimeError, TypeError):
            _check_attention(q, cache, pages, lens, cu, scale)
            raise
        return out if return_lse else out[0]
    scale = _check_attention(q, cache, pages, lens, cu, scale)
    _check_gpu(q)
    shape = q.shape
    q = q.contiguous()
    out, lse = _ops().paged_attention(q if len(shape) == 3 else q.flatten(0, 1), *cache, pages, lens, cu, bool(causal), scale)
    out, lse = out.view(shape), lse.view(shape[:-1])
    return (out, lse) if return_lse else out
