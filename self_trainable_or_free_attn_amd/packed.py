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
import math
from typing import Optional

import torch

DTYPES = {torch.bfloat16: "", torch.float16: "_f16"}     # token dtype -> suffix of the entry points
MAX_BIAS_ROWS = 784                                      # ES_PACKED_BIAS_ROWS of include/packed_hip.h


# ------------------------------------------------------------------ workspace sizes
# The C ABI's size functions in Python arithmetic, which Dynamo can trace and a ctypes call cannot be; the reasons for the
# rules stand in csrc/packed_fwd.hip and csrc/packed_bwd.hip. An entry point refuses a workspace smaller than its own rule's.
def _tile_numbers(m, B, T, G):
    return T * G // m + B + 1


def _range_bytes(tiles, Hk, D):
    resident = 1024 if D == 64 else 512
    return (tiles + resident // Hk + 1) * Hk * (128 * D + 256) * 4


def forward_workspace_bytes(B, Tq, Tk, H, Hk, D):
    if Tq <= 0:
        return 0
    tiles = _tile_numbers(128, B, Tq, H // Hk)
    if tiles * Hk >= (2048 if D == 64 else 1024) or Tk < (1024 if Tq * (H // Hk) <= 32 * B else 4096):
        return 0
    return _range_bytes(tiles, Hk, D)


def backward_workspace_bytes(B, Tq, Tk, H, Hk, D, R=0, with_bias=False):
    floats = 2 * Tq * H
    if with_bias:
        floats += _tile_numbers(64, B, Tq, H // Hk) * H * (2 * R + 1)
    return 4 * floats


def shared_workspace_bytes(B, n, P, S, H, Hk, D):
    rows = n * (H // Hk)
    return _range_bytes(-(-B * rows // 128) + B * -(-rows // 128), Hk, D)


# ------------------------------------------------------------------ checks
def _require(ok, message, kind=ValueError):
    if not ok:
        raise kind(message)


def _check_tokens(q, named):
    """q's dtype, head dim and device; every (name, tensor) alike."""
    _require(q.dtype in DTYPES, f"q must be bfloat16 or float16, got {q.dtype}", TypeError)
    _require(q.shape[-1] in (64, 128), f"head dim must be 64 or 128, got {q.shape[-1]}")
    for name, x in named:
        _require(x.dtype == q.dtype, f"{name} must be {q.dtype} like q, got {x.dtype}", TypeError)
        _require(x.device == q.device, f"{name} is on {x.device}, q on {q.device}")


def _check_gpu(q):
    _require(q.is_cuda or q.is_meta, f"tensors must be on the GPU, got {q.device}")


def _check_heads(H, Hk):
    _require(Hk > 0 and H % Hk == 0, f"q's {H} heads must be a multiple of k's {Hk}")
    _require(H <= 4096, f"at most 4096 heads, got {H}")


def _check_ints(name, x, device, dim=1):
    _require(x.dtype == torch.int32, f"{name} must be int32, got {x.dtype}", TypeError)
    _require(x.dim() == dim and x.is_contiguous(), f"{name} must be a contiguous {dim}-dimensional tensor")
    _require(x.device == device, f"{name} is on {x.device}, q on {device}")


def _scale(scale, D):
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    _require(0.0 < scale < 1e30, f"scale must be positive and finite, got {scale}")
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
    (floating-point formulas may put a distance that stands on one into the bucket before)."""
    n = num_buckets // 2 if bidirectional else num_buckets
    _require(n >= 2 and (not bidirectional or num_buckets % 2 == 0),
             f"num_buckets must be at least {4 if bidirectional else 2}{' and even' if bidirectional else ''}, "
             f"got {num_buckets}")
    _require(max_distance > n // 2, f"max_distance must exceed the {n // 2} distances with buckets of their own")
    return torch.tensor(_bucket_list(int(num_buckets), int(max_distance), bool(bidirectional)), dtype=torch.int32,
                        device=device)


# ------------------------------------------------------------------ packed attention
def _forward(q, k, v, cu_q, cu_k, bias, buckets, B, causal, scale):
    from . import _lib
    (Tq, H, D), (Tk, Hk) = q.shape, k.shape[:2]
    out = torch.empty_like(q)
    lse = torch.empty(Tq, H, device=q.device, dtype=torch.float32)
    if Tq > 0:
        n = forward_workspace_bytes(B, Tq, Tk, H, Hk, D)
        ws = torch.empty(n, device=q.device, dtype=torch.uint8) if n else None
        _lib.call("es_packed_fwd" + DTYPES[q.dtype], q, k, v, cu_q, cu_k, bias, buckets,
                  0 if bias is None else bias.shape[0], 0 if bias is None else buckets.shape[0] // 2, out, lse, ws, n, B,
                  Tq, Tk, H, Hk, D, int(causal), scale)
    return out, lse


class _PackedFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, cu_q, cu_k, buckets, B, causal, scale):
        weight = None if bias is None else bias.detach().float().contiguous()
        out, lse = _forward(q, k, v, cu_q, cu_k, weight, buckets, B, causal, scale)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k, weight, buckets)
        ctx.call = (B, causal, scale, None if bias is None else bias.dtype)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _dlse):
        from . import _lib
        q, k, v, out, lse, cu_q, cu_k, weight, buckets = ctx.saved_tensors
        B, causal, scale, bias_dtype = ctx.call
        if dout is None:
            return (None,) * 10
        (Tq, H, D), (Tk, Hk) = q.shape, k.shape[:2]
        dout = dout.contiguous()
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        R = 0 if weight is None else buckets.shape[0] // 2
        dbias = None if weight is None else torch.empty_like(weight)
        n = backward_workspace_bytes(B, Tq, Tk, H, Hk, D, R, weight is not None)
        ws = torch.empty(n, device=q.device, dtype=torch.uint8)
        _lib.call("es_packed_bwd" + DTYPES[q.dtype], q, k, v, dout, out, lse, cu_q, cu_k, weight, buckets,
                  0 if weight is None else weight.shape[0], R, dq, dk, dv, dbias, ws, n, B, Tq, Tk, H, Hk, D, int(causal),
                  scale)
        return (dq, dk, dv, None if dbias is None else dbias.to(bias_dtype)) + (None,) * 6


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
                     cu_k: Optional[torch.Tensor] = None, *, causal: bool = False, scale: Optional[float] = None,
                     bias: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None,
                     return_lse: bool = False):
    """Attention of every query over the keys of its own sequence, with gradients for q, k, v and bias.

    q [Tq, H, D], k and v [Tk, Hk, D], bf16 or fp16, D 64 or 128, H a multiple of Hk (query head h reads kv head
    h // (H // Hk)). cu_q, cu_k: int32 [B + 1] GPU tensors of running lengths from 0; sequence b holds rows cu[b] to
    cu[b + 1] - 1 (cu_k None: the queries' own). Without both, q / k / v are one sequence, or a batch [B, Lq, H, D] /
    [B, Lk, Hk, D]. Lengths may be zero. Rows behind the last sequence give zeros, and key rows there are never used; within
    a sequence values must be finite, also where the causal mask hides them.

    With nq queries and nk keys query i stands at position i + nk - nq (the last query at the last key): with causal it sees
    the keys up to that position. A row that sees no key gives zeros and an LSE of -inf, and no gradient. scale: 1 / sqrt(D)
    if None. bias [num_buckets, H] with buckets (`relative_buckets`, int32 [2 R + 1]) adds bias[buckets[d + R], h] to the
    score of a key at distance d from the query, d clamped to -R .. R; (H // Hk) * (2 R + 1) is at most 784.

    Returns out like q, with return_lse also the natural-log LSE [Tq, H] ([B, Lq, H]) in float32 (no gradient). Gradients
    are deterministic, and those of a bias are summed in float32; the backward itself is not differentiable."""
    batched = q.dim() == 4
    _require(q.dim() in (3, 4) and k.dim() == q.dim() and v.dim() == q.dim(),
             "q, k and v must be [T, H, D], or all [B, L, H, D]")
    _check_tokens(q, (("k", k), ("v", v)))
    _require(k.shape == v.shape, f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    _require(k.shape[-1] == q.shape[-1], f"q has head dim {q.shape[-1]}, k {k.shape[-1]}")
    H, Hk, D = q.shape[-2], k.shape[-2], q.shape[-1]
    _check_heads(H, Hk)
    if batched:
        _require(cu_q is None and cu_k is None, "cu_q / cu_k go with packed [T, H, D] tensors")
        _require(k.shape[0] == q.shape[0], f"q has {q.shape[0]} sequences, k {k.shape[0]}")
        B = q.shape[0]
    elif cu_q is None:
        _require(cu_k is None, "cu_k needs cu_q")
        B = 1
    else:
        _check_ints("cu_q", cu_q, q.device)
        B = cu_q.shape[0] - 1
        _require(B >= 1, "cu_q must hold at least two values")
        if cu_k is None:
            _require(k.shape[0] == q.shape[0], f"without cu_k k must have q's {q.shape[0]} rows, got {k.shape[0]}")
            cu_k = cu_q
        else:
            _check_ints("cu_k", cu_k, q.device)
            _require(cu_k.shape[0] == B + 1, f"cu_k must hold {B + 1} values like cu_q, got {cu_k.shape[0]}")
    scale = _scale(scale, D)
    _require((bias is None) == (buckets is None), "bias and buckets go together")
    if bias is not None:
        _require(bias.dim() == 2 and bias.shape[1] == H and bias.shape[0] > 0 and bias.is_floating_point(),
                 f"bias must be a floating-point [num_buckets, {H}] tensor, got {tuple(bias.shape)} {bias.dtype}")
        _require(bias.device == q.device, f"bias is on {bias.device}, q on {q.device}")
        _check_ints("buckets", buckets, q.device)
        width = buckets.shape[0]
        _require(width % 2 == 1, f"buckets must hold 2 R + 1 values, got {width}")
        _require(H // Hk * width <= MAX_BIAS_ROWS,
                 f"(H // Hk) * (2 R + 1) must be at most {MAX_BIAS_ROWS}, got {H // Hk} * {width}")
    _check_gpu(q)
    shape = q.shape
    q, k, v = (x.contiguous() for x in (q, k, v))
    if batched:
        if B == 0:
            return (q.clone(), q.new_empty(shape[:-1], dtype=torch.float32)) if return_lse else q.clone()
        q, k, v = (x.flatten(0, 1) for x in (q, k, v))
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, bias)):
        out, lse = _PackedFunction.apply(q, k, v, bias, cu_q, cu_k, buckets, B, bool(causal), scale)
    else:
        weight = None if bias is None else bias.float().contiguous()
        out, lse = _forward(q, k, v, cu_q, cu_k, weight, buckets, B, bool(causal), scale)
    if batched:
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
    lens[b] on are never used. bf16 or fp16, D 64 or 128, H a multiple of Hk, every tensor contiguous. scale: 1 / sqrt(D) if
    None.

    Returns out like q, with return_lse also the natural-log LSE [B, n, H] in float32; a token without keys gives zeros and
    -inf. There is no backward: tensors that require a gradient are refused unless gradients are off."""
    from . import _lib
    _require(q.dim() == 4 and k.dim() == 4 and k_prefix.dim() == 3,
             "q must be [B, n, H, D], k and v [B, S, Hk, D], k_prefix and v_prefix [P, Hk, D]")
    named = (("k_prefix", k_prefix), ("v_prefix", v_prefix), ("k", k), ("v", v))
    _check_tokens(q, named)
    _require(k.shape == v.shape, f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    _require(k_prefix.shape == v_prefix.shape,
             f"k_prefix and v_prefix must have one shape, got {tuple(k_prefix.shape)} and {tuple(v_prefix.shape)}")
    (B, n, H, D), (_, S, Hk, _) = q.shape, k.shape
    _require(k.shape[0] == B and k.shape[3] == D and k_prefix.shape[1:] == k.shape[2:],
             f"q {tuple(q.shape)}, k {tuple(k.shape)} and k_prefix {tuple(k_prefix.shape)} do not go together")
    _check_heads(H, Hk)
    _check_ints("lens", lens, q.device)
    _require(lens.shape[0] == B, f"lens must hold {B} values, got {lens.shape[0]}")
    scale = _scale(scale, D)
    for name, x in (("q", q), *named):
        _require(x.is_contiguous(), f"{name} must be contiguous")
        _require(not (x.requires_grad and torch.is_grad_enabled()),
                 f"shared_prefix_attention has no backward, and {name} requires a gradient")
    _check_gpu(q)
    out = torch.empty_like(q)
    lse = torch.empty(B, n, H, device=q.device, dtype=torch.float32)
    if q.numel() > 0:
        size = shared_workspace_bytes(B, n, k_prefix.shape[0], S, H, Hk, D)
        ws = torch.empty(size, device=q.device, dtype=torch.uint8)
        _lib.call("es_shared_prefix_fwd" + DTYPES[q.dtype], q, k_prefix, v_prefix, k, v, lens, out, lse, ws, size, B, n,
                  k_prefix.shape[0], S, H, Hk, D, scale)
    return (out, lse) if return_lse else out
