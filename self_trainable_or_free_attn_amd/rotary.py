"""Norms of queries and keys for each head with the position rotation in the same pass (include/paged_hip.h; the reference has no
counterpart).

  rotary_table   cosines and sines of positions on one axis (text) or several (a video's frames, rows and columns)
  norm_rotate    root-mean-square norm of every head's row, times a weight, rotated by position, with gradients

Token tensors are bf16 or fp16 with D = 64 or 128. No call synchronises. The HIP library is loaded at the first call.
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from .packed import _check_gpu, _check_ints, _check_tokens, _ops


def rotary_table(sizes: Union[int, Sequence[int]], dims: Union[int, Sequence[int]], theta: float = 10000.0,
                 device=None) -> torch.Tensor:
    """Angles for `norm_rotate` and `append_paged`: float32 [P, R / 2, 2], the cosine and sine of every position and pair of
    channels, computed in 64 bits. sizes and dims whole numbers: positions 0 .. sizes - 1, pair i of R = dims channels turns by
    position * theta ** (-2 i / R). Sequences: the points of a grid in order (the last axis the fastest), axis a with dims[a]
    channels of its own, one axis' pairs behind the other's. R, the sum, is a multiple of 16."""
    sizes = (sizes,) if isinstance(sizes, int) else tuple(sizes)
    dims = (dims,) if isinstance(dims, int) else tuple(dims)
    if len(sizes) != len(dims) or not sizes:
        raise ValueError(f"sizes and dims must have one entry an axis, got {sizes} and {dims}")
    if min(sizes) < 1 or min(dims) < 0 or any(d % 2 for d in dims):
        raise ValueError(f"sizes must be positive and dims even, got {sizes} and {dims}")
    if sum(dims) % 16 or not sum(dims):
        raise ValueError(f"the rotated channels must be a multiple of 16, got {sum(dims)}")
    parts = []
    for axis, (n, d) in enumerate(zip(sizes, dims)):
        freq = theta ** (-torch.arange(0, d, 2, dtype=torch.float64, device=device) / max(d, 1))
        angle = torch.arange(n, dtype=torch.float64, device=device)[:, None] * freq
        shape = [1] * len(sizes) + [d // 2, 2]
        shape[axis] = n
        part = torch.stack([angle.cos(), angle.sin()], -1).float().view(shape)
        parts.append(part.expand(*sizes, d // 2, 2))
    return torch.cat(parts, -2).reshape(-1, sum(dims) // 2, 2).contiguous()


def _check_turn(x, D, q_weight, k_weight, table, eps):
    """The arguments of the norm and the rotation; x: a token tensor. Returns eps."""
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if w.dim() != 1 or w.shape[0] != D:
            raise ValueError(f"{name} must be [{D}], got {tuple(w.shape)}")
        if w.dtype is not x.dtype and w.dtype is not torch.float32:
            raise TypeError(f"{name} must be float32 or {x.dtype} like the tokens, got {w.dtype}")
        if w.device != x.device:
            raise ValueError(f"{name} is on {w.device}, the tokens on {x.device}")
    if q_weight is not None and k_weight is not None and q_weight.dtype is not k_weight.dtype:
        raise TypeError(f"q_weight and k_weight must have one dtype, got {q_weight.dtype} and {k_weight.dtype}")
    if table is not None:
        if table.dtype is not torch.float32:
            raise TypeError(f"table must be float32, got {table.dtype}")
        if table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous() or table.shape[0] == 0:
            raise ValueError(f"table must be a contiguous [positions, R / 2, 2] tensor, got {tuple(table.shape)}")
        R = 2 * table.shape[1]
        if R == 0 or R % 16 or R > D:
            raise ValueError(f"the rotated channels must be a multiple of 16 up to {D}, got {R}")
        if table.device != x.device:
            raise ValueError(f"table is on {table.device}, the tokens on {x.device}")
    eps = float(eps)
    if not 0.0 <= eps < 1e30:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    return eps


def _check_rotate(q, k, q_weight, k_weight, table, positions, eps):
    """The arguments of norm_rotate; eps and the positions of all rows."""
    dims = q.dim()
    if dims not in (3, 4) or k.dim() != dims:
        raise ValueError("q and k must be [T, H, D], or both [B, L, H, D]")
    _check_tokens(q, (("k", k),))
    shape, kshape = q.shape, k.shape
    if shape[:-2] != kshape[:-2] or shape[-1] != kshape[-1]:
        raise ValueError(f"q {tuple(shape)} and k {tuple(kshape)} do not go together")
    for n in (shape[-2], kshape[-2]):
        if not 0 < n <= 4096:
            raise ValueError(f"q and k must have 1 to 4096 heads, got {shape[-2]} and {kshape[-2]}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight go together")
    if q_weight is None and table is None:
        raise ValueError("norm_rotate needs weights, a table or both")
    eps = _check_turn(q, shape[-1], q_weight, k_weight, table, eps)
    L = shape[-3]
    if positions is not None:
        if table is None:
            raise ValueError("positions go with a table")
        if positions.shape != shape[:-2]:
            raise ValueError(f"positions must be {tuple(shape[:-2])}, got {tuple(positions.shape)}")
        if dims == 4:
            positions = positions.flatten()
        _check_ints("positions", positions, q.device)
    elif table is not None and table.shape[0] < L:
        raise ValueError(f"the table has {table.shape[0]} positions for {L} rows")
    return eps, positions


def norm_rotate(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                k_weight: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6, halves: bool = False):
    """Queries and keys normed and rotated in one pass, with gradients for q, k and the weights.

    q [T, H, D] and k [T, Hk, D] (or [B, L, H, D] and [B, L, Hk, D]), bf16 or fp16, D 64 or 128; column ranges of a projection's
    rows are read where they are. With weights ([D], the tokens' type or float32, both or neither) a head's row x becomes
    x / sqrt(mean x^2 + eps) * weight. With a table (`rotary_table`) its first R channels are then turned in pairs by the angles
    of the row's position, channels 2 i and 2 i + 1, with halves i and i + R / 2. positions: int32 [T] ([B, L]) rows of the
    table, clamped to it; None: a row's place in q (in its sequence of the batch).

    Returns the new q and k, contiguous. All arithmetic is float32, rounded once at the end (so the squares of a row have to stay
    within float32: bf16 values to about 1e18, with eps = 0 from 1e-19 on). Gradients are deterministic and those
    of the weights are summed in float32; the backward itself is not differentiable, and a table gets no gradient. A capture with
    gradients takes leaves made inside it; those that an eager graph of another stream holds are refused."""
    if q.is_cuda and q.dim() == 3:      # the operator checks everything itself; what it refuses is named by the checks below
        try:
            return _ops().norm_rotate(q, k, q_weight, k_weight, table, positions, max(q.shape[0], 1), bool(halves), eps)
        except (RuntimeError, TypeError):
            _check_rotate(q, k, q_weight, k_weight, table, positions, eps)
            raise
    eps, positions = _check_rotate(q, k, q_weight, k_weight, table, positions, eps)
    _check_gpu(q)
    if q.dim() == 3:
        return _ops().norm_rotate(q, k, q_weight, k_weight, table, positions, max(q.shape[0], 1), bool(halves), eps)
    shape, kshape = q.shape, k.shape
    q, k = _ops().norm_rotate(q.flatten(0, 1), k.flatten(0, 1), q_weight, k_weight, table, positions, max(shape[1], 1),
                              bool(halves), eps)
    return q.view(shape), k.view(kshape)
