"""fp16 gradients of packed_attention for output gradients and values of any size (scaled losses): against 64 bits, where the
results are representable.

dS = p (do v - delta) follows the sizes of do and v, and the kernels round it to fp16 times a power of two of its row (for dq) or
key (for dk). Bounds, with u = 2^-11, F as in packed_ref.py, and m the largest |dS| of the row or key:
  dS      u |dS| for its rounding; 2^-32 m for fp16's subnormal steps (half a step is 2^-25, m is stored as 2^7 or more unless it
          is below 2^-25 itself: then 2^-65); float32: F |dS| + F p (|do| |v| + |do| sum p |v|); and, where delta comes from the stored
          out (rows of more than 512 keys without a bias), p |do| bound(out)
  dq, dk  scale sum bound(dS) |k| (|q|), float32 F scale sum |dS| |k|, own rounding u and 2^-25
  dbias   sum of bound(dS) without its rounding
Everything else as in packed_ref.py."""
import math

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

FP, U, F = torch.float16, 2.0 ** -11, ref.F


def _head(q, k, v, do, seen, scale, extra, exact):
    """Values and bounds of one kv head: q, do [G, n, D], k, v [m, D], float64."""
    r = ref.attention(q, k, v, seen, scale, extra, do, FP)
    s = scale * (q @ k.t()) + (0 if extra is None else extra)
    s = s.masked_fill(~seen, -math.inf)
    lse = r["lse"][0]
    p = torch.exp(s - torch.where(lse > -math.inf, lse, 0.0)[..., None])
    mag = do.abs() * (p @ v.abs())
    b32 = F * r["ds"][0].abs() + p * (F * (do.abs() @ v.abs().t()) + F * mag.sum(-1, keepdim=True))
    if not exact:
        b32 = b32 + p * (do.abs() * r["out"][1]).sum(-1, keepdim=True)
    ds = r["ds"][0]
    each, top = U * ds.abs() + b32 * (1 + U), ds.abs() + b32
    row = each + (2.0 ** -32 * top.amax(-1, keepdim=True) + 2.0 ** -65) * (p > 0)
    col = each + (2.0 ** -32 * top.amax((0, 1)) + 2.0 ** -65) * (p > 0)
    dq, dk = r["dq"][0], r["dk"][0]
    adq, adk = scale * (ds.abs() @ k.abs()), scale * (ds.abs().transpose(-1, -2) @ q.abs()).sum(0)
    return dict(dv=r["dv"], ds=(ds, b32),
                dq=(dq, scale * (row @ k.abs()) + F * adq + U * dq.abs() + 2.0 ** -25),
                dk=(dk, scale * (col.transpose(-1, -2) @ q.abs()).sum(0) + F * adk + U * dk.abs() + 2.0 ** -25))


def _rows(n, D, heads, g, std=1.0):
    return std * torch.randn(n, heads, D, generator=g)


def _case(dev, t, causal=False, scale=None, table=None, exact=True):
    """One sequence: t of q, k, v, dout (and bias) on the CPU, float32, rounded here."""
    import self_trainable_or_free_attn_amd as api
    x = {n: y.to(FP if n != "bias" else torch.float32).to(dev) for n, y in t.items()}
    (n, H, D), (m, Hk) = x["q"].shape, x["k"].shape[:2]
    G, scale = H // Hk, scale or D ** -0.5
    i, j = torch.arange(n, device=dev)[:, None] + m - n, torch.arange(m, device=dev)[None]
    seen = j <= i if causal else torch.ones(n, m, dtype=torch.bool, device=dev)
    names = [a for a in ("q", "k", "v", "bias") if a in x]
    leaves = [x[a].clone().requires_grad_() for a in names]
    out = api.packed_attention(*leaves[:3], causal=causal, scale=scale, bias=leaves[3] if table is not None else None,
                               buckets=table)
    grads = dict(zip(names, torch.autograd.grad(out, leaves, x["dout"])))
    head = lambda y, h: y[:, h * G:h * G + G].double().transpose(0, 1)
    if table is not None:
        at = table.long()[(j - i).clamp(-(table.numel() // 2), table.numel() // 2) + table.numel() // 2]
    for h in range(Hk):
        hs = slice(h * G, h * G + G)
        extra = x["bias"][:, hs].double().t()[:, at] if table is not None else None
        w = _head(head(x["q"], h), x["k"][:, h].double(), x["v"][:, h].double(), head(x["dout"], h), seen, scale, extra, exact)
        for a in ("dq", "dk", "dv"):
            assert float((w[a][0].abs() + w[a][1]).max()) < 65504, (a, "not representable")
        ref.check(f"dq of kv head {h}", grads["q"][:, hs].transpose(0, 1), *w["dq"])
        ref.check(f"dk of kv head {h}", grads["k"][:, h], *w["dk"])
        ref.check(f"dv of kv head {h}", grads["v"][:, h], *w["dv"])
        if table is not None:
            for b in range(x["bias"].shape[0]):
                value, bound = ((y.flatten(1) * (at.flatten() == b)).sum(1) for y in w["ds"])
                ref.check(f"dbias {b}", grads["bias"][b, hs], value, 1.01 * bound)
    return grads


def _inputs(n, m, H, Hk, D, seed, dout=1.0, v=1.0, buckets=0):
    g = torch.Generator().manual_seed(seed)
    t = dict(q=_rows(n, D, H, g, 1.5), k=_rows(m, D, Hk, g), v=_rows(m, D, Hk, g, v), dout=_rows(n, D, H, g, dout))
    if buckets:
        t["bias"] = torch.randn(buckets, H, generator=g)
    return t


SIZES = [(2, 2, 2, 2), (70, 70, 2, 2), (130, 130, 6, 2), (40, 333, 4, 1)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dout, v", [(1e-6, 1.0), (1e-4, 1.0), (1e-3, 1e-2), (300.0, 1.0), (3000.0, 3.0), (0.25, 3000.0)])
@pytest.mark.parametrize("n, m, H, Hk", SIZES)
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_any_size(dev, D, dout, v, n, m, H, Hk, causal):
    _case(dev, _inputs(n, m, H, Hk, D, 1, dout, v), causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dout", [1e-4, 1000.0])
def test_long_rows(dev, D, dout):
    """Rows of 4096 keys (probabilities of 2^-12 and less; delta from the stored out), and a causal sequence."""
    _case(dev, _inputs(130, 4096, 2, 1, D, 2, dout), exact=False)
    _case(dev, _inputs(1100, 1100, 2, 2, D, 3, dout), causal=True, exact=False)


@pytest.mark.parametrize("D", [64, 128])
def test_row_ranges(dev, D):
    """One key tile's rows cut into ranges, each with its own powers of two."""
    _case(dev, _inputs(1500, 200, 8, 1, D, 4, 500.0))
    t = _inputs(1500, 200, 8, 1, D, 5)
    t["dout"] *= 2.0 ** (torch.arange(1500)[:, None, None] * 20 // 1500 - 12)
    _case(dev, t)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("causal", [False, True])
def test_sizes_that_change_along_the_way(dev, D, order, causal):
    """Rows whose output gradients, and keys whose values, grow or shrink over 20 powers of two: the factors change in the middle."""
    n = 300
    grow = 2.0 ** (torch.arange(n) * 20 // n - 12.0)[:, None, None]
    grow = grow if order == 1 else grow.flip(0)
    t = _inputs(n, n, 4, 2, D, 6)
    _case(dev, dict(t, dout=t["dout"] * grow), causal, scale=0.02)
    _case(dev, dict(t, v=t["v"] * grow), causal, scale=0.02)
    _case(dev, dict(t, v=t["v"] * grow, dout=t["dout"] * grow.flip(0)), causal, scale=0.02)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_and_keys_of_different_sizes(dev, D):
    g = torch.Generator().manual_seed(7)
    size = lambda n, lo, hi: 2.0 ** torch.randint(lo, hi, (n, 1, 1), generator=g)
    for n, m, H, Hk in SIZES[1:]:
        t = _inputs(n, m, H, Hk, D, 8)
        t["dout"] = t["dout"] * size(n, -14, 8)
        t["v"] = t["v"] * size(m, -8, 3)
        _case(dev, t)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H, Hk", [(2, 2), (4, 2)])
@pytest.mark.parametrize("dout", [1e-5, 2000.0])
def test_bias_gradients(dev, D, H, Hk, dout):
    import self_trainable_or_free_attn_amd as api
    table = api.relative_buckets(16, 60, device=dev)
    _case(dev, _inputs(200, 200, H, Hk, D, 9, dout, buckets=16), table=table)
    t = _inputs(200, 200, H, Hk, D, 10, buckets=16)
    t["dout"] *= 2.0 ** (torch.arange(200)[:, None, None] * 20 // 200 - 12)
    _case(dev, t, causal=True, table=table)


@pytest.mark.parametrize("D", [64, 128])
def test_infinite_and_zero_gradients(dev, D):
    """An infinite row of dout reaches its own dq and every key it sees, no other row and no other tile of keys; zeros give
    zeros."""
    import self_trainable_or_free_attn_amd as api
    t = {n: y.to(FP).to(dev) for n, y in _inputs(200, 200, 2, 1, D, 11).items()}
    leaves = [t[n].requires_grad_() for n in "qkv"]
    out = api.packed_attention(*leaves, causal=True)
    clean = torch.autograd.grad(out, leaves, t["dout"], retain_graph=True)
    t["dout"][77, 1] = math.inf
    dq, dk, dv = torch.autograd.grad(out, leaves, t["dout"], retain_graph=True)
    assert torch.equal(dq[:77], clean[0][:77]) and torch.equal(dq[78:], clean[0][78:]) and torch.equal(dq[77, 0], clean[0][77, 0])
    assert not dq[77, 1].isfinite().any()
    assert not dk[:78].isfinite().any() and not dv[:78].isfinite().any()
    assert torch.equal(dk[128:], clean[1][128:]) and torch.equal(dv[128:], clean[2][128:])
    for x in torch.autograd.grad(out, leaves, torch.zeros_like(out)):
        assert not x.any()
