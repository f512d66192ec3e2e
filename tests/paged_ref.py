"""Plain 64-bit norms with rotation, 4-bit values and paged caches for the tests of rotary.py and paged.py, with bounds of what the
kernels may be off.

Each result comes with an elementwise bound. Roundings to the token type: u = eps / 2 relative, below fp16's smallest normal value
HALF = 2^-25 absolute. Float32 operations, in units of 2^-24 relative to the terms' magnitudes:
  r        sum of D squares by 16 a lane and 3 steps across: 20; mean and eps: 2; both halved by the root; its reciprocal: 4: 15
  y        x r w: 2, products with cosine and sine and their sum: 3, and what r has: 20, below 2^-19 of |a c| + |b s|
  g        the incoming gradient turned back: 3
  h xh     g, w, x, r: 3 + 1 + 16 + 1, its mean: 21; dx = r (h - xh mean): below 2^-17 of r (|h| + |xh| mean |h xh|)
  dw       g xh: 20, and one a term that is added to a partial sum: n of them
"""
import math

import torch

F = 2.0 ** -19
FB = 2.0 ** -17
HALF = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def turn(x, cs, halves, back=False):
    """x [T, H, D] float64 turned by cs [T, R / 2, 2]."""
    R = 2 * cs.shape[1]
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    s = -s if back else s
    if halves:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = x[..., :R:2], x[..., 1:R:2]
        y = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([y, x[..., R:]], -1)


def _turn_abs(x, cs, halves):
    """|a c| + |b s| of every channel."""
    cs = cs.abs().clone()
    R = 2 * cs.shape[1]
    c, s, x = cs[:, None, :, 0].double(), cs[:, None, :, 1].double(), x.abs()
    if halves:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y = torch.cat([a * c + b * s, a * s + b * c], -1)
    else:
        a, b = x[..., :R:2], x[..., 1:R:2]
        y = torch.stack([a * c + b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([y, x[..., R:]], -1)


def rotate(x, w, cs, eps, halves, dy=None, terms=0):
    """x [T, H, D]; w [D] or None; cs [T, R / 2, 2] of its rows. Dict of y, with dy also dx and dw: (value, bound)."""
    dt = x.dtype
    u, half = torch.finfo(dt).eps / 2, HALF[dt]
    x = x.double()
    r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) if w is not None else torch.ones_like(x[..., :1])
    xh = x * r
    wd = w.double() if w is not None else 1.0
    y = turn(xh * wd, cs, halves)
    res = dict(y=(y, F * _turn_abs(xh * wd, cs, halves) + u * (1 + F) * y.abs() + half))
    if dy is None:
        return res
    g, ga = turn(dy.double(), cs, halves, back=True), _turn_abs(dy.double(), cs, halves)
    if w is None:
        res["dx"] = (g, F * ga + u * (1 + F) * g.abs() + half)
        return res
    h, ha = g * wd, ga * wd.abs()
    dx = r * (h - xh * (h * xh).mean(-1, keepdim=True))
    mag = r * (ha + xh.abs() * (ha * xh.abs()).mean(-1, keepdim=True))
    res["dx"] = (dx, FB * mag + u * (1 + FB) * dx.abs() + half)
    dw = (g * xh).sum((0, 1))
    uw = torch.finfo(w.dtype).eps / 2
    res["dw"] = (dw, (20 + terms) * 2.0 ** -24 * (ga * xh.abs()).sum((0, 1)) + uw * 1.01 * dw.abs() + HALF[w.dtype])
    return res


def power(e):
    """2^e in float64, exact (torch's ldexp and exp2 are a last bit off for some e on the GPU)."""
    return (e.long() + 1023 << 52).view(torch.float64)


EXPONENTS = {torch.bfloat16: (-120, 120), torch.float16: (-13, 13)}


def held4(x, dtype):
    """The 4-bit values (float64) nearest to x [..., D] float32, and the exponents of their scales: by steps of a power of two,
    half of s below 2 s, s up to 4 s, 2 s above, ties to the even multiple."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    frac, e = torch.frexp(top)
    e = torch.where(frac > 0.875, e - 2, e - 3)
    e = torch.where(top == 0, -1000, e).clamp(*EXPONENTS[dtype])
    s = power(e)
    a = g.abs() / s
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.sign(g) * (torch.round(a / step) * step).clamp(max=6.0) * s).flatten(-2), e[..., 0]


MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def decode4(codes, scales):
    """float64 values of codes [..., D / 2] and scales [..., D / 32]."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=torch.float64, device=codes.device)
    x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
    return x * power(scales.long() - 127).repeat_interleave(32, -1)


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def page_table(keys, page, spare, dev, seed, width=None):
    """Pages of all sequences spread over a cache in any order, unused entries -1; (table, number of pages)."""
    need = [-(-m // page) for m in keys]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(keys), width or max(max(need), 1)), -1, dtype=torch.int32)
    for b, (at, n) in enumerate(zip(starts(need), need)):
        table[b, :n] = order[at:at + n]
    return table.to(dev), len(order)


def gathered(x, table, m, page):
    """Rows 0 .. m - 1 of one sequence, [m, Hk, D], from pages x [N, Hk, page, D]; table: its row."""
    if m == 0:
        return x.new_zeros(0, x.shape[1], x.shape[3])
    held = table[:-(-m // page)].long()
    return x[held].transpose(1, 2).flatten(0, 1)[:m]


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
