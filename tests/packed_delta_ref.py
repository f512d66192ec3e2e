"""64-bit dq, dk and dS of attention with bounds for a backward that takes delta = sum p (do v) itself and not from the rounded
output: no term for the rounding of o. u = eps / 2 of the token type, F as in packed_ref.py (float32), m the largest |dS| of the
row (dq) or key (dk):
  dS      float32: F |dS| + F p (|do| |v| + |do| sum p |v|) (b32); its rounding u |dS|; fp16: 2^-32 m + 2^-65 for its subnormal
          steps (dS is stored times a power of two that takes m to 2^7 or more)
  dq, dk  scale sum bound(dS) |k| (|q|), float32 F scale sum |dS| |k|, own rounding u (fp16: and 2^-25)
  dbias   1.01 sum of b32: its sums are float32
"""
import math

import torch

import packed_ref as ref

F = ref.F


def attention(q, k, v, do, seen, scale, extra, dtype, delta=None):
    """One kv head: q, do [G, n, D], k, v [m, D] float64, seen [n, m], extra [G, n, m] or None. delta: this one instead (to see what
    a mistake in it does)."""
    u = torch.finfo(dtype).eps / 2
    step, own = (2.0 ** -32, 2.0 ** -25) if dtype is torch.float16 else (0.0, 0.0)
    s = scale * (q @ k.t()) + (0 if extra is None else extra)
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - torch.where(lse > -math.inf, lse, 0.0))
    dp, pd = do @ v.t(), do.abs() @ v.abs().t()
    ds = p * (dp - ((p * dp).sum(-1, keepdim=True) if delta is None else delta))
    b32 = F * ds.abs() + p * F * (pd + (do.abs() * (p @ v.abs())).sum(-1, keepdim=True))
    top = ds.abs() + b32
    each = u * ds.abs() + b32 * (1 + u)
    row = each + (step * top.amax(-1, keepdim=True) + step ** 2) * (p > 0)
    col = each + (step * top.amax((0, 1)) + step ** 2) * (p > 0)
    dq, dk = scale * (ds @ k), scale * (ds.transpose(-1, -2) @ q).sum(0)
    adq, adk = scale * (ds.abs() @ k.abs()), scale * (ds.abs().transpose(-1, -2) @ q.abs()).sum(0)
    return dict(ds=(ds, b32), dq=(dq, scale * (row @ k.abs()) + F * adq + u * dq.abs() + own),
                dk=(dk, scale * (col.transpose(-1, -2) @ q.abs()).sum(0) + F * adk + u * dk.abs() + own))


def by_bucket(ds, at, buckets):
    """(value, bound) of dbias [buckets, G]; at [n, m]: the bucket of each pair."""
    value, b32 = (torch.stack([(x.flatten(1) * (at.flatten() == b)).sum(1) for b in range(buckets)]) for x in ds)
    return value, 1.01 * b32


def telling_inputs(n, m, H, Hk, D, dtype):
    """Inputs whose output rounds the same way in every channel of every row: q = 0 (equal weights), values of 1 and, for three keys
    in five, the next number of the type. The output stands 2 / 5 of a step from the number it is stored as, so delta = sum do o is
    off by D times that; the bounds allow D 2^-15."""
    up = 1 + torch.finfo(dtype).eps
    a = torch.tensor([up if j % 5 in (0, 2, 3) else 1.0 for j in range(m)])
    return (torch.zeros(n, H, D, dtype=dtype), torch.ones(m, Hk, D, dtype=dtype), a[:, None, None].expand(m, Hk, D).to(dtype),
            torch.ones(n, H, D, dtype=dtype))
