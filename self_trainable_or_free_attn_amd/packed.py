"""Attention over packed sequences of different lengths, its learned position bias by buckets, and attention of a batch
over a prefix that its sequences share (include/packed_hip.h; the reference has no counterpart).

  packed_attention          [T, H, D] rows of several sequences end to end (or a [B, L, H, D] batch), every token over its
                            own sequence, causal or not, grouped heads, with a gradient: clips or prompts of different
                            sizes in one call, pieces of prompts and single tokens against longer histories
  relative_buckets          the distance -> bucket table of its position bias
  shared_prefix_attention   new tokens of B sequences over one prefix, read once for all, and each sequence's own cache

Token tensors are bf16 or fp16 with D = 64 or 128. Lengths stay on the GPU (int32 tensors): no call synchronises, so all of
them can be captured into a graph and replayed with other lengths. The HIP library is loaded at the first call.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

MAX_BIAS_ROWS = 784      # ES_PACKED_BIAS_ROWS of include/packed_hip.h


_op_table = None


def _ops():
    """torch.ops.echosparse_gfx950 (loaded at the first call)."""
    global _op_table
    if _op_table is None:
        from . import _lib
        _op_table = _lib.ops()
    return _op_table


# ------------------------------------------------------------------ checks
# (written so that a call that passes formats no message: the checks are a good part of a short call's host time)
def _check_tokens(q, named):
    """q's dtype and head dim; dtype and device of every (name, tensor) like q's."""
    dtype, device = q.dtype, q.device
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"q must be bfloat16 or float16, got {dtype}")
    if q.shape[-1] not in (64, 128):
        raise ValueError(f"head dim must be 64 or 128, got {q.shape[-1]}")
    for name, x in named:
        if x.dtype is not dtype:
            raise TypeError(f"{name} must be {dtype} like q, got {x.dtype}")
        if x.device != device:
            raise ValueError(f"{name} is on {x.device}, q on {device}")


def _check_heads(H, Hk):
    if Hk <= 0 or H <= 0 or H % Hk:
        raise ValueError(f"q's {H} heads must be a multiple of k's {Hk}")
    if H > 4096:
        raise ValueError(f"at most 4096 heads, got {H}")


def _check_ints(name, x, device):
    if x.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, got {x.dtype}")
    if x.dim() != 1 or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-dimensional tensor")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, q on {device}")


def _check_gpu(q):
    if not (q.is_cuda or q.is_meta):
        raise ValueError(f"tensors must be on the GPU, got {q.device}")


def _scale(scale, D):
    if scale is None:
        return D ** -0.5
    scale = float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


# ------------------------------------------------------------------ position bias
@functools.lru_cache(maxsize=32)
def _bucket_list(num_buckets, max_distance, bidirectional):
    n = num_buckets // 2 if bidirectional else num_buckets
    exact = n // 2
    steps = n - exact
    # first[s]: the smallest distance of logarithmic step s, (a / exact)^steps >= (max_distance / exact)^s, in whole numbers
    first = []
    for s in range(steps):
        lo, hi, want = exact, max_distance, max_distance ** s * exact ** (steps - s)
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if mid ** steps >= want else (mid + 1, hi)
        first.append(lo)
    reach = max(first[-1], 1)

    def bucket(d):
        base = n if bidirectional and d > 0 else 0
        a = abs(d) if bidirectional else max(-d, 0)
        return base + (a if a < exact else exact + sum(a >= f for f in first) - 1)

    return tuple(bucket(d) for d in range(-reach, reach + 1))


def relative_buckets(num_buckets: int, max_distance: int, bidirectional: bool = True, device=None) -> torch.Tensor:
    """Table of the bucket of every key position minus query position d, int32 [2 R + 1] for d = -R .. R; `packed_attention`
    clamps d to that range. Half of a direction's buckets hold one distance each, the others are spaced evenly in the
    logarithm up to max_distance, and the last one holds every distance from its first on (R is where that is reached, so R
    is less than max_distance). bidirectional: half of the buckets for keys behind the query, half for keys ahead; otherwise
    all of them for keys behind, and keys ahead share bucket 0 with the query's own position. Borders are exact integers
    (floating-point formulas may put a distance that stands on one into the bucket before). `packed_attention` takes tables
    of up to 784 // (H // Hk) entries: 32 buckets to 128 have 183 both ways and serve four heads a group."""
    n = num_buckets // 2 if bidirectional else num_buckets
    if n < 2 or (bidirectional and num_buckets % 2):
        raise ValueError(f"num_buckets must be at least {4 if bidirectional else 2}"
                         f"{' and even' if bidirectional else ''}, got {num_buckets}")
    if max_distance <= n // 2:
        raise ValueError(f"max_distance must exceed the {n // 2} distances with buckets of their own")
    return torch.tensor(_bucket_list(int(num_buckets), int(max_distance), bool(bidirectional)), dtype=torch.int32,
                        device=device)


# ------------------------------------------------------------------ packed attention
def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
                     cu_k: Optional[torch.Tensor] = None, *, causal: bool = False, scale: Optional[float] = None,
                     bias: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None,
                     return_lse: bool = False):
    """Attention of every query over the keys of its own sequence, with gradients for q, k, v and bias.

    q [Tq, H, D], k and v [Tk, Hk, D], bf16 or fp16, D 64 or 128, H a multiple of Hk (query head h reads kv head
    h // (H // Hk)). cu_q, cu_k: int32 [B + 1] GPU tensors of running lengths from 0; sequence b holds rows cu[b] to
    cu[b + 1] - 1 (cu_k None: the queries' own). Without both, q / k / v are one sequence, or a batch [B, Lq, H, D] /
    [B, Lk, Hk, D]. Lengths may be zero. Rows behind the last sequence give zeros, and key rows there are never used; within
    a sequence values must be finite, also where the causal mask hides them, and scores below 2^22 in magnitude.

    With nq queries and nk keys query i stands at position i + nk - nq (the last query at the last key): with causal it sees
    the keys up to that position. A row that sees no key gives zeros and an LSE of -inf, and no gradient. scale: 1 / sqrt(D)
    if None. bias [num_buckets, H] with buckets (`relative_buckets`, int32 [2 R + 1]) adds bias[buckets[d + R], h] to the
    score of a key at distance d from the query, d clamped to -R .. R; (H // Hk) * (2 R + 1) is at most 784. Its values are finite
    or -inf, which masks; finite ones are held to +-131072 (and get no gradient beyond that).

    Returns out like q, with return_lse also the natural-log LSE [Tq, H] ([B, Lq, H]) in float32 (no gradient). Gradients
    are deterministic, and those of a bias are summed in float32; the backward itself is not differentiable. With fp16 tensors
    the output's gradient may be of any size (a scaled loss): a gradient overflows or vanishes only where fp16 cannot hold it."""
    dims = q.dim()
    if dims not in (3, 4) or k.dim() != dims or v.dim() != dims:
        raise ValueError("q, k and v must be [T, H, D], or all [B, L, H, D]")
    _check_tokens(q, (("k", k), ("v", v)))
    shape, kshape = q.shape, k.shape
    if kshape != v.shape:
        raise ValueError(f"k and v must have one shape, got {tuple(kshape)} and {tuple(v.shape)}")
    H, D, Hk = shape[-2], shape[-1], kshape[-2]
    if kshape[-1] != D:
        raise ValueError(f"q has head dim {D}, k {kshape[-1]}")
    _check_heads(H, Hk)
    if dims == 4:
        if cu_q is not None or cu_k is not None:
            raise ValueError("cu_q / cu_k go with packed [T, H, D] tensors")
        if kshape[0] != shape[0]:
            raise ValueError(f"q has {shape[0]} sequences, k {kshape[0]}")
        B = shape[0]
    elif cu_q is None:
        if cu_k is not None:
            raise ValueError("cu_k needs cu_q")
        B = 1
    else:
        _check_ints("cu_q", cu_q, q.device)
        B = cu_q.shape[0] - 1
        if B < 1:
            raise ValueError("cu_q must hold at least two values")
        if cu_k is None:
            if kshape[0] != shape[0]:
                raise ValueError(f"without cu_k k must have q's {shape[0]} rows, got {kshape[0]}")
            cu_k = cu_q
        else:
            _check_ints("cu_k", cu_k, q.device)
            if cu_k.shape[0] != B + 1:
                raise ValueError(f"cu_k must hold {B + 1} values like cu_q, got {cu_k.shape[0]}")
    scale = _scale(scale, D)
    if (bias is None) != (buckets is None):
        raise ValueError("bias and buckets go together")
    if bias is not None:
        if bias.dim() != 2 or bias.shape[1] != H or bias.shape[0] == 0 or not bias.is_floating_point():
            raise ValueError(f"bias must be a floating-point [num_buckets, {H}] tensor, got {tuple(bias.shape)} {bias.dtype}")
        if bias.device != q.device:
            raise ValueError(f"bias is on {bias.device}, q on {q.device}")
        _check_ints("buckets", buckets, q.device)
        width = buckets.shape[0]
        if width % 2 == 0:
            raise ValueError(f"buckets must hold 2 R + 1 values, got {width}")
        if H // Hk * width > MAX_BIAS_ROWS:
            raise ValueError(f"(H // Hk) * (2 R + 1) must be at most {MAX_BIAS_ROWS}, got {H // Hk} * {width}")
    _check_gpu(q)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if dims == 4:
        if B == 0:
            return (q.clone(), q.new_empty(shape[:-1], dtype=torch.float32)) if return_lse else q.clone()
        q, k, v = (x.flatten(0, 1) for x in (q, k, v))
    out, lse = _ops().packed_attention(q, k, v, bias, cu_q, cu_k, buckets, B, bool(causal), scale)
    if dims == 4:
        out, lse = out.view(shape), lse.view(shape[:-1])
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------ shared prefix
def shared_prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k: torch.Tensor,
                            v: torch.Tensor, lens: torch.Tensor, *, scale: Optional[float] = None,
                            return_lse: bool = False):
    """Attention of n new tokens of each of B sequences over one prefix and the sequence's own cache, in one softmax; the
    prefix is read once for the whole batch.

    q [B, n, H, D]; k_prefix, v_prefix [P, Hk, D], seen whole by every token; k, v [B, S, Hk, D], the caches as they were
    allocated, and lens int32 [B] how many rows of each are in use (clamped to 0 .. S), the n tokens' own keys, which the
    caller has written, the last of them. Token i of sequence b sees its cache rows 0 to lens[b] - n + i. Cache rows from
    lens[b] on are never used. bf16 or fp16, D 64 or 128, H a multiple of Hk, every tensor contiguous and
    aligned to 16 bytes. scale: 1 / sqrt(D) if None.

    Returns out like q, with return_lse also the natural-log LSE [B, n, H] in float32; a token without keys gives zeros and
    -inf. There is no derivative: tensors that require a gradient are refused unless gradients are off, tensors that
    carry a forward-mode tangent always."""
    if q.dim() != 4 or k.dim() != 4 or k_prefix.dim() != 3:
        raise ValueError("q must be [B, n, H, D], k and v [B, S, Hk, D], k_prefix and v_prefix [P, Hk, D]")
    named = (("k_prefix", k_prefix), ("v_prefix", v_prefix), ("k", k), ("v", v))
    _check_tokens(q, named)
    shape, kshape, pshape = q.shape, k.shape, k_prefix.shape
    if kshape != v.shape:
        raise ValueError(f"k and v must have one shape, got {tuple(kshape)} and {tuple(v.shape)}")
    if pshape != v_prefix.shape:
        raise ValueError(f"k_prefix and v_prefix must have one shape, got {tuple(pshape)} and {tuple(v_prefix.shape)}")
    if kshape[0] != shape[0] or kshape[3] != shape[3] or pshape[1:] != kshape[2:]:
        raise ValueError(f"q {tuple(shape)}, k {tuple(kshape)} and k_prefix {tuple(pshape)} do not go together")
    _check_heads(shape[2], kshape[2])
    _check_ints("lens", lens, q.device)
    if lens.shape[0] != shape[0]:
        raise ValueError(f"lens must hold {shape[0]} values, got {lens.shape[0]}")
    scale = _scale(scale, shape[3])
    grad = torch.is_grad_enabled()
    for name, x in (("q", q), *named):
        if not x.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if grad and x.requires_grad:
            raise ValueError(f"shared_prefix_attention has no backward, and {name} requires a gradient")
    _check_gpu(q)
    if shape[0] == 0 or shape[1] == 0:
        out, lse = torch.empty_like(q), q.new_empty(shape[:3], dtype=torch.float32)
    else:
        out, lse = _ops().shared_prefix_attention(q, k_prefix, v_prefix, k, v, lens, scale)
    return (out, lse) if return_lse else out
