"""Plain 64-bit attention over packed sequences for the tests of packed.py, with bounds of what the kernels may be off.

Each result comes with an elementwise bound. Per rounding to the token type u = eps / 2 relative; every float32 product, sum
and exponential together F = 2^-16 of the terms' magnitudes (a sum of 128 products is off by at most 128 * 2^-24 = 2^-17 of
them; the exponent's argument is below 64, so its last bit is 2^-18 of the probability). With A = sum p |v|:
  out     the probabilities' rounding u A, float32 F A, its own rounding u |o|
  lse     F, and of its magnitude 2^-22
  dv      (u + F) sum p |do|, its own u |dv|
  ds      rounding u |ds|, float32 F |ds| + F p sum |do| |v|, and what delta = sum do o inherits from out: p sum |do| bound(o)
  dq, dk  scale sum bound(ds) |k| (|q|), float32 F scale sum |ds| |k|, their own rounding
  dbias   sum of bound(ds) without the rounding of ds (its sums are float32)
Type ranges: probabilities below the token type's subnormal range may vanish: TINY a key. A value below fp16's smallest
normal 2^-14 is stored in steps of 2^-24, so its rounding is off by up to HALF = 2^-25 whatever its size (bf16 has float32's
range: nothing to add).
"""
import torch

F = 2.0 ** -16
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -30}
HALF = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def attention(q, k, v, seen, scale, extra=None, dout=None, dtype=None):
    """One kv head: q [G, n, D], k, v [m, D] float64, seen [n, m] bool, extra [G, n, m]. Dict of name -> (value, bound)."""
    u = torch.finfo(dtype).eps / 2
    tiny, half = TINY[dtype], HALF[dtype]
    s = scale * (q @ k.t())
    if extra is not None:
        s = s + extra
    s = s.masked_fill(~seen, float("-inf"))
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full(q.shape[:2], float("-inf"), device=q.device).double()
    live = lse > float("-inf")
    p = torch.exp(s - torch.where(live, lse, 0.0)[..., None])
    o = p @ v
    mag = p @ v.abs()
    bo = (u + F) * mag + u * o.abs() * (1 + F) + tiny * v.abs().sum(0) + half
    res = dict(out=(o, bo), lse=(lse, torch.where(live, F + 2.0 ** -22 * lse.abs(), 0.0)))
    if dout is None:
        return res
    dp, pd = dout @ v.t(), dout.abs() @ v.abs().t()
    delta = (dout * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    b32 = F * ds.abs() + p * (F * pd + F * (dout.abs() * mag).sum(-1, keepdim=True)
                              + (dout.abs() * bo).sum(-1, keepdim=True))
    bds = u * ds.abs() + b32 * (1 + u)
    bds = bds + half * (p > 0)
    dv = (p.transpose(-1, -2) @ dout).sum(0)
    pdo = (p.transpose(-1, -2) @ dout.abs()).sum(0)
    res["dv"] = (dv, (u + F) * pdo + u * dv.abs() * (1 + F) + tiny * dout.abs().sum((0, 1)) + half)
    dq, dk = scale * (ds @ k), scale * (ds.transpose(-1, -2) @ q).sum(0)
    adq, adk = scale * (ds.abs() @ k.abs()), scale * (ds.abs().transpose(-1, -2) @ q.abs()).sum(0)
    res["dq"] = (dq, scale * (bds @ k.abs()) + F * adq + u * dq.abs() + half)
    res["dk"] = (dk, scale * (bds.transpose(-1, -2) @ q.abs()).sum(0) + F * adk + u * dk.abs() + half)
    res["ds"] = (ds, b32)
    return res


def packed(q, k, v, lens, keys, causal, scale, bias=None, buckets=None, dout=None):
    """The results of packed_attention and its gradients for sequences of `lens` queries and `keys` keys, rows in order:
    name -> (value, bound), float64."""
    dt, dev = q.dtype, q.device
    (Tq, H, D), (Tk, Hk) = q.shape, k.shape[:2]
    G = H // Hk
    z = lambda *shape: torch.zeros(*shape, device=dev, dtype=torch.float64)
    res = dict(out=(z(Tq, H, D), z(Tq, H, D)), lse=(z(Tq, H) - float("inf"), z(Tq, H)))
    if dout is not None:
        res.update(dq=(z(Tq, H, D), z(Tq, H, D)), dk=(z(Tk, Hk, D), z(Tk, Hk, D)), dv=(z(Tk, Hk, D), z(Tk, Hk, D)))
        if bias is not None:
            res["dbias"] = (z(*bias.shape), z(*bias.shape))
    a = c = 0
    for n, m in zip(lens, keys):
        i = torch.arange(n, device=dev)[:, None] + m - n
        j = torch.arange(m, device=dev)[None]
        seen = j <= i if causal else torch.ones(n, m, dtype=torch.bool, device=dev)
        if bias is not None:
            R = buckets.numel() // 2
            at = buckets.long()[(j - i).clamp(-R, R) + R]
        for h in range(Hk):
            hs = slice(h * G, h * G + G)
            extra = bias[:, hs].double().t()[:, at] if bias is not None else None
            r = attention(q[a:a + n, hs].double().transpose(0, 1), k[c:c + m, h].double(), v[c:c + m, h].double(), seen,
                          scale, extra, None if dout is None else dout[a:a + n, hs].double().transpose(0, 1), dt)
            for x in (0, 1):
                res["out"][x][a:a + n, hs] = r["out"][x].transpose(0, 1)
                res["lse"][x][a:a + n, hs] = r["lse"][x].transpose(0, 1)
                if dout is None:
                    continue
                res["dq"][x][a:a + n, hs] = r["dq"][x].transpose(0, 1)
                res["dk"][x][c:c + m, h] = r["dk"][x]
                res["dv"][x][c:c + m, h] = r["dv"][x]
                if bias is not None:
                    flat = r["ds"][x].flatten(1)
                    for b in range(bias.shape[0]):
                        res["dbias"][x][b, hs] += (flat * (at.flatten() == b)).sum(1)
        a, c = a + n, c + m
    if "dbias" in res:      # (float32 sums over distances and tiles)
        value, bound = res["dbias"]
        res["dbias"] = (value, bound * 1.01)
    return res


def check(name, got, want, bound):
    """got within bound of want, elementwise; infinities equal, no NaN."""
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), f"{name}: infinities differ"
    over = (got - want).abs()[fine] - bound[fine]
    assert not over.numel() or not bool((over > 0).any() | over.isnan().any()), \
        f"{name}: off by {float((got - want).abs()[fine].max()):.3g}, {int((over > 0).sum())} values over their bounds by " \
        f"up to {float(over.max()):.3g}, NaN {int(over.isnan().sum())}"
