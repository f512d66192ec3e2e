"""The packed-sequence operators against plain 64-bit attention (packed_ref.py, which derives the bounds): lengths from nothing
to long, grouped heads, masks that leave rows empty, padding full of NaN, key ranges, streams, graphs, determinism."""
import math

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _api():
    import self_trainable_or_free_attn_amd as api
    return api


def _workspace(B, Tq, Tk, H, Hk, D):
    from self_trainable_or_free_attn_amd import _lib
    return _lib.lib().es_packed_fwd_workspace(B, Tq, Tk, H, Hk, D)


def _cu(lens, dev):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


def _inputs(lens, keys, H, Hk, D, dtype, dev, seed, pad=0, buckets=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)
    Tq, Tk = sum(lens) + pad, sum(keys) + pad
    t = dict(q=(1.5 * rnd(Tq, H, D)).to(dtype), k=rnd(Tk, Hk, D).to(dtype), v=rnd(Tk, Hk, D).to(dtype),
             dout=rnd(Tq, H, D).to(dtype))
    if buckets:
        t["bias"] = rnd(buckets, H)
    if pad:      # rows behind the last sequence hold anything
        for n in ("k", "v"):
            t[n][Tk - pad:] = math.nan
        t["q"][Tq - pad:] = math.nan
        t["dout"][Tq - pad:] = math.nan
    return t


def _clean(x):
    return torch.nan_to_num(x)


def _case(lens, keys, H, Hk, D, dtype, causal, dev, train=False, pad=0, table=None, seed=0, scale=None):
    api = _api()
    t = _inputs(lens, keys, H, Hk, D, dtype, dev, seed, pad, 0 if table is None else int(table.max()) + 1)
    scale_ = scale or 1 / math.sqrt(D)
    want = ref.packed(_clean(t["q"]), _clean(t["k"]), _clean(t["v"]), lens, keys, causal, scale_, t.get("bias"), table,
                      _clean(t["dout"]) if train else None)
    names = [n for n in ("q", "k", "v", "bias") if n in t]
    if train:
        for n in names:
            t[n].requires_grad_()
    out, lse = api.packed_attention(t["q"], t["k"], t["v"], _cu(lens, dev), _cu(keys, dev), causal=causal, scale=scale,
                                    bias=t.get("bias"), buckets=table, return_lse=True)
    ref.check("out", out.detach(), *want["out"])
    ref.check("lse", lse, *want["lse"])
    if train:
        for n, g in zip(names, torch.autograd.grad(out, [t[n] for n in names], t["dout"])):
            assert g.dtype == t[n].dtype
            ref.check("d" + n, g, *want["d" + n])


TYPES = [(64, BF), (128, BF), (64, FP), (128, FP)]
RAGGED = [
    ([1], [1]), ([0, 5, 0, 33, 1, 0], [0, 5, 0, 33, 1, 0]), ([64, 128, 127, 129, 65], [64, 128, 127, 129, 65]),
    ([3, 40, 200], [0, 7, 150]),                 # fewer keys than queries: rows without keys under a causal mask
    ([1, 17, 130], [300, 100, 131]), ([5, 0, 2], [0, 9, 63]),
]


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("H, Hk", [(2, 2), (6, 2), (8, 1)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens, keys", RAGGED)
def test_forward(dev, D, dtype, H, Hk, causal, lens, keys):
    _case(lens, keys, H, Hk, D, dtype, causal, dev, pad=9, seed=1)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("lens, keys, H, Hk", [
    ([1500, 700], [2500, 1700], 3, 1),                           # ranges of wide tiles
    ([1, 1, 1], [5000, 64, 1029], 10, 2),                       # ranges of single tokens
    ([33, 2, 300], [4100, 2500, 70], 5, 5),                     # narrow and wide tiles in one launch
    ([2, 1, 1, 600], [0, 3500, 1, 600], 4, 2),
    ([1], [40000], 16, 2),
])
@pytest.mark.parametrize("causal", [False, True])
def test_key_ranges(dev, D, dtype, lens, keys, H, Hk, causal):
    assert _workspace(len(lens), sum(lens), sum(keys), H, Hk, D) > 0
    _case(lens, keys, H, Hk, D, dtype, causal, dev, seed=2)


@pytest.mark.parametrize("D, dtype, T, H, Hk", [(128, BF, 2200, 64, 16), (64, FP, 4300, 64, 32)])
def test_whole_tiles(dev, D, dtype, T, H, Hk):
    assert _workspace(2, T, T, H, Hk, D) == 0
    _case([T - 130, 130], [T - 130, 130], H, Hk, D, dtype, True, dev, seed=3)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_many_heads(dev, D, dtype, causal, bias):
    """Grids that fill the GPU take tiles of 128 rows, smaller ones (the other tests) of 64."""
    table = _api().relative_buckets(16, 60, device=dev) if bias else None
    _case([300, 1, 70, 0, 129], [300, 1, 200, 5, 129], 128, 128, D, dtype, causal, dev, table=table, pad=2, seed=48)


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_many_sequences(dev, B, pad):
    lens = [(7 * i) % 23 for i in range(B)]
    keys = [(11 * i) % 40 for i in range(B)]
    _case(lens, keys, 3, 1, 64, BF, True, dev, pad=pad, seed=4, train=True)


def test_many_sequences_with_key_ranges(dev):
    lens = [1 + (i % 3 == 0) for i in range(150)]
    keys = [(i * i * 7) % 900 for i in range(150)]
    _case(lens, keys, 4, 1, 128, FP, True, dev, pad=2, seed=5)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("H, Hk", [(2, 2), (6, 2), (7, 1)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens, keys", RAGGED + [([700, 333], [700, 333])])
def test_backward(dev, D, dtype, H, Hk, causal, lens, keys):
    _case(lens, keys, H, Hk, D, dtype, causal, dev, train=True, pad=5, seed=6)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("lens, keys, H, Hk, pad", [([1500], [1500], 8, 1, 0), ([700, 5, 600], [650, 0, 1100], 6, 1, 3),
                                                    ([1030], [70], 3, 3, 1), ([900, 901], [900, 901], 5, 1, 0)])
@pytest.mark.parametrize("causal", [False, True])
def test_row_ranges(dev, D, dtype, lens, keys, H, Hk, pad, causal):
    """Few key tiles against many rows: the KV owner's rows in ranges."""
    from self_trainable_or_free_attn_amd import _lib
    Tq, Tk = sum(lens) + pad, sum(keys) + pad
    assert _lib.lib().es_packed_bwd_workspace(len(lens), Tq, Tk, H, Hk, D, 0, 0, causal) > 8 * Tq * H + 16
    _case(lens, keys, H, Hk, D, dtype, causal, dev, train=True, pad=pad, seed=22)


@pytest.mark.parametrize("H, Hk", [(100, 1), (65, 1), (256, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_more_heads_than_a_tile_has_rows(dev, H, Hk, causal):
    _case([5, 1, 30], [9, 1, 30], H, Hk, 64, BF, causal, dev, train=True, seed=42)
    _case([1, 2], [2000, 70], H, Hk, 128, FP, causal, dev, seed=43)


def test_row_ranges_with_a_bias(dev):
    table = _api().relative_buckets(16, 60, device=dev)
    _case([1200, 300], [1200, 300], 2, 1, 64, BF, False, dev, train=True, table=table, seed=23)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("H, Hk", [(2, 2), (6, 3), (4, 1)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens, keys", [([1], [1]), ([0, 70, 200, 3], [0, 70, 200, 3]), ([40, 5], [300, 0]), ([600], [450])])
def test_bias(dev, D, dtype, H, Hk, causal, lens, keys):
    table = _api().relative_buckets(32, 128, bidirectional=not causal, device=dev)
    if H // Hk * table.numel() > 784:
        table = _api().relative_buckets(16, 60, bidirectional=not causal, device=dev)
    _case(lens, keys, H, Hk, D, dtype, causal, dev, train=True, pad=4, table=table, seed=7)


@pytest.mark.parametrize("table", [[0], [1, 0, 2], [0, 0, 0, 1, 1], list(range(195))])
def test_bias_tables(dev, table):
    """Tables of the caller's own: a single entry, unordered and unused buckets, one bucket a distance up to the limit."""
    t = torch.tensor(table, dtype=torch.int32, device=dev)
    _case([150, 80], [150, 330], 4, 1, 64, BF, False, dev, train=True, table=t, seed=8)


def test_bias_over_key_ranges(dev):
    table = _api().relative_buckets(32, 128, bidirectional=False, device=dev)
    _case([1, 40], [3000, 1200], 2, 2, 128, BF, True, dev, table=table, seed=9)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_scores_of_any_size(dev, dtype):
    """A large scale (one key takes all), a small one (every key the same), and scores far below zero."""
    for scale in (3.0, 1e-6):
        _case([130, 1], [130, 1500], 2, 1, 64, dtype, True, dev, train=scale < 1, seed=10, scale=scale)
    api = _api()
    t = _inputs([70], [70], 2, 2, 64, dtype, dev, 11)
    low = torch.full((1, 2), -60000.0, device=dev)
    one = torch.zeros(1, dtype=torch.int32, device=dev)
    out = api.packed_attention(t["q"], t["k"], t["v"], bias=low, buckets=one)
    want = ref.packed(t["q"], t["k"], t["v"], [70], [70], False, 0.125)
    # (scores of -60000 keep 2^-8 of their last bits in float32: the probabilities are off by up to that in the exponent)
    value, bound = want["out"]
    ref.check("out", out, value, bound + 2.0 ** -7 * value.abs().amax() * 4)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H, Hk", [(2, 2), (4, 2)])
def test_bias_that_masks(dev, D, dtype, causal, H, Hk):
    """Buckets of -inf: keys without weight, and rows (all of one head's, some of another's) without any key."""
    table = _api().relative_buckets(16, 60, device=dev)
    lens = [150, 1, 70]
    t = _inputs(lens, lens, H, Hk, D, dtype, dev, 40, buckets=16)
    t["bias"][:, 1] = -math.inf
    t["bias"][2:6, 0] = -math.inf
    t["bias"][:3, 0] = -math.inf        # (the first rows of a causal sequence then see nothing)
    t["bias"][8, 0] = -math.inf
    want = ref.packed(t["q"], t["k"], t["v"], lens, lens, causal, 1 / math.sqrt(D), t["bias"], table, t["dout"])
    names = ("q", "k", "v", "bias")
    leaves = [t[n].requires_grad_() for n in names]
    out, lse = _api().packed_attention(*leaves[:3], _cu(lens, dev), causal=causal, bias=leaves[3], buckets=table,
                                       return_lse=True)
    ref.check("out", out, *want["out"])
    ref.check("lse", lse, *want["lse"])
    for n, x in zip(names, torch.autograd.grad(out, leaves, t["dout"])):
        ref.check("d" + n, x, *want["d" + n])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("low", [-1e6, -1e9, -3.4028234663852886e38, 1e12])
@pytest.mark.parametrize("R", [0, 4])
def test_bias_of_any_size(dev, dtype, low, R):
    """One value for all keys cancels, whatever it is. Held to 2^17 (189097 in log2 units, where float32 has steps of 2^-6), it
    rounds a score by up to 2^-7, which puts a probability off by up to 2^-7 ln 2 and the row's sum by as much: 2^-6 of
    sum p |v| <= max |v| together. The stored LSE adds its own half step 2^-8 (natural) and twice that of 2^-7 (log2), so the
    backward's probabilities are off by less than 2^-5."""
    L, D = 90, 64
    t = _inputs([L], [L], 2, 2, D, dtype, dev, 41)
    bias, table = torch.full((1, 2), low, device=dev), torch.zeros(2 * R + 1, dtype=torch.int32, device=dev)
    want = ref.packed(t["q"], t["k"], t["v"], [L], [L], True, 0.125, None, None, t["dout"])
    leaves = [t[n].requires_grad_() for n in "qkv"]
    out = _api().packed_attention(*leaves, causal=True, bias=bias, buckets=table)
    value, bound = want["out"]
    ref.check("out", out, value, bound + 2.0 ** -6 * t["v"].detach().abs().max().double())
    dq, dk, dv = torch.autograd.grad(out, leaves, t["dout"])
    value, bound = want["dv"]
    s = 0.125 * torch.einsum("ihd,jhd->hij", t["q"].detach().double(), t["k"].detach().double())
    p = torch.softmax(s.masked_fill(torch.ones(L, L, device=dev, dtype=torch.bool).triu(1), -math.inf), -1)
    moved = (p.transpose(1, 2) @ t["dout"].abs().double().transpose(0, 1).contiguous()).transpose(0, 1)
    ref.check("dv", dv, value, bound + 2.0 ** -5 * moved)
    assert dq.isfinite().all() and dk.isfinite().all()


def test_batch_form_equals_packed_form(dev):
    api = _api()
    g = torch.Generator(device=dev).manual_seed(12)
    q = torch.randn(3, 50, 6, 64, device=dev, generator=g).to(BF).requires_grad_()
    k = torch.randn(3, 70, 2, 64, device=dev, generator=g).to(BF).requires_grad_()
    v = torch.randn(3, 70, 2, 64, device=dev, generator=g).to(BF).requires_grad_()
    out, lse = api.packed_attention(q, k, v, causal=True, return_lse=True)
    o2, l2 = api.packed_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), _cu([50] * 3, dev), _cu([70] * 3, dev),
                                  causal=True, return_lse=True)
    assert out.shape == q.shape and lse.shape == q.shape[:3]
    assert torch.equal(out.flatten(0, 1), o2) and torch.equal(lse.flatten(0, 1), l2)
    d = torch.randn(out.shape, device=dev, generator=g).to(BF)
    a = torch.autograd.grad(out, [q, k, v], d)
    b = torch.autograd.grad(o2, [q, k, v], d.flatten(0, 1))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    one = api.packed_attention(q[0], k[0], v[0], causal=True)
    assert torch.equal(one, out[0])
    assert api.packed_attention(q[:0], k[:0], v[:0]).shape == (0, 50, 6, 64)
    assert api.packed_attention(q[:, :0], k, v).shape == (3, 0, 6, 64)
    empty = api.packed_attention(q, k[:, :0], v[:, :0], return_lse=True)
    assert not empty[0].any() and (empty[1] == -math.inf).all()
    gq, gk = torch.autograd.grad(empty[0], [q, k], torch.ones_like(empty[0]))
    assert not gq.any() and not gk.any()


def test_inputs_that_start_anywhere(dev):
    """Views one value into a storage: contiguous, but not at the 16 bytes that the kernels load."""
    api = _api()
    t = _inputs([60], [60], 2, 2, 64, BF, dev, 40)

    def shifted(x):
        y = torch.empty(x.numel() + 1, device=dev, dtype=x.dtype)[1:].view(x.shape)
        return y.copy_(x)

    a = [t[n].clone().requires_grad_() for n in "qkv"]
    b = [shifted(t[n]).requires_grad_() for n in "qkv"]
    oa, ob = api.packed_attention(*a, causal=True), api.packed_attention(*b, causal=True)
    assert b[0].data_ptr() % 16 and torch.equal(oa, ob)
    ga, gb = torch.autograd.grad(oa, a, t["dout"]), torch.autograd.grad(ob, b, shifted(t["dout"]))
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))
    s = _shared(2, 1, 10, 8, [1, 2], 2, 2, 64, BF, dev, 41)
    with pytest.raises(RuntimeError, match="aligned"):
        api.shared_prefix_attention(s["q"], s["kp"], s["vp"], shifted(s["k"]), s["v"], s["lens"])


def test_strided_inputs_and_gradients(dev):
    """Views of one projection, a gradient that is an expanded view, a bias in the token type."""
    api = _api()
    g = torch.Generator(device=dev).manual_seed(13)
    qkv = torch.randn(100, 3, 2, 64, device=dev, generator=g).to(BF).requires_grad_()
    cu = _cu([30, 70], dev)
    out = api.packed_attention(*qkv.unbind(1), cu)
    out.sum(dtype=torch.float32).backward()
    parts = [x.detach().clone().requires_grad_() for x in qkv.unbind(1)]
    o2 = api.packed_attention(*parts, cu)
    assert torch.equal(out, o2)
    for x, y in zip(torch.autograd.grad(o2, parts, torch.ones_like(o2)), qkv.grad.unbind(1)):
        assert torch.equal(x, y)
    w = torch.randn(8, 2, device=dev, generator=g).to(BF).requires_grad_()
    table = api.relative_buckets(8, 20, device=dev)
    o3 = api.packed_attention(*parts, cu, bias=w, buckets=table)
    gw, = torch.autograd.grad(o3, [w], torch.ones_like(o3))
    assert gw.dtype == BF and gw.shape == w.shape
    o4 = api.packed_attention(*parts, cu, bias=w.detach().float(), buckets=table)
    assert torch.equal(o3, o4)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_gradients_against_differences(dev, dtype):
    """sum(out * dout) of the 64-bit attention along random directions, central differences, against the kernels' gradients:
    off by at most the gradients' bounds along the direction and the differences' own h^2."""
    table = _api().relative_buckets(8, 30, device=dev)
    lens = [60, 9]
    t = _inputs(lens, lens, 4, 2, 64, dtype, dev, 14, buckets=8)
    want = ref.packed(t["q"], t["k"], t["v"], lens, lens, False, 0.125, t["bias"], table, t["dout"])
    names = ["q", "k", "v", "bias"]
    leaves = {n: t[n].clone().requires_grad_() for n in names}
    out = _api().packed_attention(leaves["q"], leaves["k"], leaves["v"], _cu(lens, dev), bias=leaves["bias"], buckets=table)
    grads = torch.autograd.grad(out, [leaves[n] for n in names], t["dout"])
    g = torch.Generator(device=dev).manual_seed(15)

    def value(x):
        total = 0.0
        for a, n in ((0, 60), (60, 9)):
            i = torch.arange(n, device=dev)
            at = table.long()[(i[None] - i[:, None]).clamp(-(table.numel() // 2), table.numel() // 2) + table.numel() // 2]
            for h in range(4):
                s = 0.125 * x["q"][a:a + n, h] @ x["k"][a:a + n, h // 2].t() + x["bias"][:, h][at]
                total = total + (torch.softmax(s, -1) @ x["v"][a:a + n, h // 2] * t["dout"][a:a + n, h].double()).sum()
        return total

    for n, grad in zip(names, grads):
        for _ in range(3):
            d = torch.randn(grad.shape, device=dev, generator=g).double()
            x = {m: t[m].double() for m in names}
            h, diffs = 1e-3, []
            for step in (h, 2 * h):
                up, down = dict(x), dict(x)
                up[n], down[n] = x[n] + step * d, x[n] - step * d
                diffs.append((value(up) - value(down)) / (2 * step))
            off = (diffs[1] - diffs[0]).abs()            # three times the h^2 term
            got = (grad.double() * d).sum()
            assert (got - diffs[0]).abs() <= (want["d" + n][1] * d.abs()).sum() + off + 1e-7


def test_same_bits_every_time(dev):
    table = _api().relative_buckets(32, 128, device=dev)
    lens, keys = [300, 1, 130], [300, 2000, 130]
    t = _inputs(lens, keys, 6, 3, 128, BF, dev, 16, buckets=32)
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v", "bias")]
    runs = []
    for _ in range(4):
        out, lse = _api().packed_attention(*leaves[:3], _cu(lens, dev), _cu(keys, dev), bias=leaves[3], buckets=table,
                                           return_lse=True)
        runs.append([out.detach(), lse, *torch.autograd.grad(out, leaves, t["dout"])])
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


def test_wrong_running_lengths_stay_in_bounds(dev):
    """Lengths past the tensors are cut off, negative ones count as none."""
    t = _inputs([40], [60], 2, 2, 64, BF, dev, 17)
    for cu in ([0, 30, 10 ** 9], [0, 35, 20, 40], [-5, 10, 40], [0, 0, 0]):
        c = torch.tensor(cu, dtype=torch.int32, device=dev)
        out = _api().packed_attention(t["q"].requires_grad_(), t["k"], t["v"], c, c)
        torch.autograd.grad(out, [t["q"]], t["dout"])
        torch.cuda.synchronize()
    c = torch.tensor([0, 30, 10 ** 9], dtype=torch.int32, device=dev)
    out = _api().packed_attention(t["q"], t["k"], t["v"], c, c)
    want = _api().packed_attention(t["q"], t["k"], t["v"], _cu([30, 10], dev), _cu([30, 30], dev))
    assert torch.equal(out, want)


def test_one_row_of_nan_stays_alone(dev):
    t = _inputs([200], [200], 2, 1, 64, BF, dev, 18)
    clean = _api().packed_attention(t["q"], t["k"], t["v"], causal=True)
    t["q"][77] = math.nan
    out = _api().packed_attention(t["q"], t["k"], t["v"], causal=True)
    rows = torch.arange(200, device=dev) != 77
    assert torch.equal(out[rows], clean[rows]) and out[77].isnan().all()


def test_rows_past_four_gigabytes(dev):
    """Keys whose byte offsets pass 32 bits: the last sequence, and one sequence that spans the border; two of the heads are
    compared."""
    H, D, T = 32, 128, 540_000                      # 8 KB a row: 4.4 GB each for k and v
    g = torch.Generator(device=dev).manual_seed(19)
    k = torch.empty(T, H, D, device=dev, dtype=BF)
    v = torch.empty_like(k)
    for x in (k, v):
        for a in range(0, T, 60_000):
            x[a:a + 60_000] = torch.randn(min(60_000, T - a), H, D, device=dev, generator=g).to(BF)
    lens, keys = [1, 2, 70], [500_000, 39_930, 70]
    q = torch.randn(73, H, D, device=dev, generator=g).to(BF)
    out, lse = _api().packed_attention(q, k, v, _cu(lens, dev), _cu(keys, dev), causal=True, return_lse=True)
    for h in (0, 31):
        hs = slice(h, h + 1)
        want = ref.packed(q[:, hs], k[:, hs], v[:, hs], lens, keys, True, 1 / math.sqrt(D))
        ref.check("out", out[:, hs], *want["out"])
        ref.check("lse", lse[:, hs], *want["lse"])


def test_streams_and_graphs(dev):
    """A call on a side stream, two graphs whose replays alternate with eager work, and other lengths in a captured call."""
    api = _api()
    lens, keys = [1, 1, 40], [900, 130, 700]
    t = _inputs(lens, keys, 4, 2, 64, BF, dev, 20)
    cu_q, cu_k = _cu(lens, dev), _cu(keys, dev)
    eager = lambda: api.packed_attention(t["q"], t["k"], t["v"], cu_q, cu_k, causal=True)
    want = eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = eager()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(eager())
        graphs.append(g)
    for keys2 in (keys, [1000, 30, 700], [0, 1029, 701]):
        cu_k.copy_(_cu(keys2, dev))
        want = eager()
        for _ in range(2):
            for g, o in zip(graphs, outs):
                o.fill_(7.0)
                g.replay()
                torch.cuda.synchronize()
                assert torch.equal(o, want)
                assert torch.equal(eager(), want)


def test_two_streams_at_once(dev):
    """Calls with key and row ranges, whose workspaces hold partial sums, side by side on two streams."""
    api = _api()
    ts = [_inputs([600], [5000], 8, 1, 128, BF, dev, 44 + i) for i in range(2)]
    step = lambda t: (lambda out, leaves: [out.detach(), *torch.autograd.grad(out, leaves, t["dout"])])(
        *(lambda x: (api.packed_attention(*x, causal=True), x))([t[n].detach().requires_grad_() for n in "qkv"]))
    want = [step(t) for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ts]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(ts[i]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(x, y) for x, y in zip(r, w))


def test_ranges_in_a_graph(dev):
    """A captured step with key ranges and row ranges, replayed with other lengths between eager ones."""
    api = _api()
    t = _inputs([1500], [5000], 8, 1, 128, BF, dev, 46)
    cu_q, cu_k = _cu([1500, 0], dev), _cu([5000, 0], dev)

    def step():
        leaves = [t[n].detach().requires_grad_() for n in "qkv"]
        out = api.packed_attention(*leaves, cu_q, cu_k, causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, t["dout"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for lens, keys in (([1500, 0], [5000, 0]), ([700, 800], [4200, 800]), ([1, 1400], [4000, 900])):
        cu_q.copy_(_cu(lens, dev))
        cu_k.copy_(_cu(keys, dev))
        want = step()
        for _ in range(2):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)), lens


def test_no_queries(dev):
    """Keys without a query: zero gradients for them, and for the bias."""
    api = _api()
    t = _inputs([0], [70], 4, 2, 64, BF, dev, 47, buckets=8)
    table = api.relative_buckets(8, 30, device=dev)
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v", "bias")]
    out = api.packed_attention(*leaves[:3], _cu([0], dev), _cu([70], dev), bias=leaves[3], buckets=table)
    for x, y in zip(torch.autograd.grad(out, leaves, t["dout"]), leaves):
        assert x.shape == y.shape and not x.any()


def test_training_step_in_a_graph(dev):
    api = _api()
    lens = [200, 1, 70]
    table = api.relative_buckets(8, 30, device=dev)
    t = _inputs(lens, lens, 4, 2, 64, BF, dev, 21, buckets=8)
    cu = _cu(lens, dev)
    names = ("q", "k", "v", "bias")

    def step(x):
        leaves = [x[n].detach().requires_grad_() for n in names]
        out = api.packed_attention(*leaves[:3], cu, causal=True, bias=leaves[3], buckets=table)
        return [out.detach(), *torch.autograd.grad(out, leaves, t["dout"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(t)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(t)
    for i in range(3):
        t["q"].copy_(torch.randn_like(t["q"]))
        want = step(t)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i


# ------------------------------------------------------------------ shared prefix
def _shared(B, n, P, S, lens, H, Hk, D, dtype, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(dtype)
    t = dict(q=rnd(B, n, H, D) * 1.5, kp=rnd(P, Hk, D), vp=rnd(P, Hk, D), k=rnd(B, S, Hk, D), v=rnd(B, S, Hk, D),
             lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    for b, m in enumerate(lens):                     # unused cache rows hold anything
        t["k"][b, max(m, 0):] = math.nan
        t["v"][b, max(m, 0):] = math.inf
    return t


def _shared_check(t, out, lse, scale=None):
    (B, n, H, D), P, (_, S, Hk, _) = t["q"].shape, t["kp"].shape[0], t["k"].shape
    G = H // Hk
    for b, m in enumerate(t["lens"].tolist()):
        m = min(max(m, 0), S)
        keys, vals = torch.cat([t["kp"], t["k"][b, :m]]).double(), torch.cat([t["vp"], t["v"][b, :m]]).double()
        j = torch.arange(P + m, device=out.device)[None]
        seen = (j < P) | (j - P <= m - n + torch.arange(n, device=out.device)[:, None])
        for h in range(Hk):
            hs = slice(h * G, h * G + G)
            r = ref.attention(t["q"][b, :, hs].double().transpose(0, 1), keys[:, h], vals[:, h], seen,
                              scale or 1 / math.sqrt(D), dtype=t["q"].dtype)
            ref.check(f"out {b}", out[b, :, hs].transpose(0, 1), *r["out"])
            ref.check(f"lse {b}", lse[b, :, hs].transpose(0, 1), *r["lse"])


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("n, P, S, lens, H, Hk", [
    (1, 500, 256, [40, 1, 200], 8, 8), (1, 1, 1, [1], 2, 1), (1, 0, 64, [5, 64], 4, 2), (1, 77, 0, [0, 0], 4, 2),
    (3, 129, 70, [3, 0, 70, 2], 6, 2),               # fewer own keys than tokens: the first tokens see the prefix alone
    (1, 0, 9, [0, 4], 2, 2),                         # a row without any key
    (1, 5000, 300, [299, 300, 1, 17, 64, 65, 128, 8], 16, 2), (40, 700, 512, [512, 40, 41], 5, 5),
    (1, 2000, 100, [50] * 70, 4, 1), (2, 64, 3000, [3000, 2, 1999], 8, 1),
    (1, 300, 20, [25, -3], 4, 4),                    # lengths out of range are cut off
    (40, 300, 600, [600, 40, 77], 8, 2), (1, 0, 0, [0], 2, 2), (33, 65, 40, [40, 33], 4, 4),
    (1, 4000, 16, [16] * 130, 8, 2),
])
def test_shared_prefix(dev, D, dtype, n, P, S, lens, H, Hk):
    t = _shared(len(lens), n, P, S, lens, H, Hk, D, dtype, dev, 30)
    out, lse = _api().shared_prefix_attention(t["q"], t["kp"], t["vp"], t["k"], t["v"], t["lens"], return_lse=True)
    _shared_check(t, out, lse)


def test_shared_prefix_scale_streams_and_graph(dev):
    api = _api()
    t = _shared(3, 1, 600, 400, [400, 400, 400], 8, 2, 128, BF, dev, 31)
    call = lambda: api.shared_prefix_attention(t["q"], t["kp"], t["vp"], t["k"], t["v"], t["lens"], scale=0.2,
                                               return_lse=True)
    out, lse = call()
    _shared_check(t, out, lse, 0.2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    for lens in ([400, 1, 0], [3, 399, 64], [128, 129, 127]):      # a captured step, replayed as the caches grow
        t["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        want = call()
        for _ in range(2):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        _shared_check(t, *got, 0.2)


def test_shared_prefix_equals_packed(dev):
    """The same tokens through both operators: prefix and cache end to end as one packed sequence."""
    api = _api()
    t = _shared(4, 2, 300, 90, [90, 2, 33, 64], 6, 2, 64, FP, dev, 32)
    out, lse = api.shared_prefix_attention(t["q"], t["kp"], t["vp"], t["k"], t["v"], t["lens"], return_lse=True)
    lens = t["lens"].tolist()
    k = torch.cat([torch.cat([t["kp"], t["k"][b, :m]]) for b, m in enumerate(lens)])
    v = torch.cat([torch.cat([t["vp"], t["v"][b, :m]]) for b, m in enumerate(lens)])
    o2, l2 = api.packed_attention(t["q"].flatten(0, 1), k, v, _cu([2] * 4, dev), _cu([300 + m for m in lens], dev), causal=True,
                                  return_lse=True)
    # two float32 softmaxes of the same scores, each rounded once; probabilities are rounded against different maxima
    assert (lse.flatten(0, 1) - l2).abs().max() <= 2 * ref.F + 1e-5
    assert (out.flatten(0, 1).float() - o2.float()).abs().max() <= 4 * 2.0 ** -11 * v.float().abs().max()


def test_a_prompt_then_its_samples(dev):
    """The operators as they are used together: a prompt through packed_attention, whose keys become the prefix; then three
    tokens of two samples, one at a time, through shared_prefix_attention on growing caches; each equal to packed_attention
    over the whole history."""
    api = _api()
    H, Hk, D, P = 8, 2, 128, 210
    g = torch.Generator(device=dev).manual_seed(33)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(BF)
    q, k, v = rnd(P, H, D), rnd(P, Hk, D), rnd(P, Hk, D)
    want = ref.packed(q, k, v, [P], [P], True, 1 / math.sqrt(D))
    ref.check("prompt", api.packed_attention(q, k, v, causal=True), *want["out"])
    ck, cv = torch.full((2, 8, Hk, D), math.nan, device=dev, dtype=BF), torch.full((2, 8, Hk, D), math.nan, device=dev, dtype=BF)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    for step in range(3):
        qt, ck[:, step], cv[:, step] = rnd(2, 1, H, D), rnd(2, Hk, D), rnd(2, Hk, D)
        lens += 1
        out = api.shared_prefix_attention(qt, k, v, ck, cv, lens)
        for b in range(2):
            kk, vv = torch.cat([k, ck[b, :step + 1]]), torch.cat([v, cv[b, :step + 1]])
            want = ref.packed(qt[b], kk, vv, [1], [P + step + 1], True, 1 / math.sqrt(D))
            ref.check("token", out[b], *want["out"])
            ref.check("token", api.packed_attention(qt[b], kk, vv, causal=True), *want["out"])


def test_refusals_on_the_gpu(dev):
    api = _api()
    t = _shared(2, 1, 10, 8, [1, 2], 4, 2, 64, BF, dev, 34)
    with pytest.raises(ValueError, match="no backward"):
        api.shared_prefix_attention(t["q"].requires_grad_(), t["kp"], t["vp"], t["k"], t["v"], t["lens"])
    with torch.no_grad():
        api.shared_prefix_attention(t["q"], t["kp"], t["vp"], t["k"], t["v"], t["lens"])
    q = torch.zeros(4, 2, 64, device=dev, dtype=BF, requires_grad=True)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="cu_q is on cpu"):
        api.packed_attention(q, q, q, cu)
    out = api.packed_attention(q, q, q)
    gr, = torch.autograd.grad(out, [q], torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        gr.sum().backward()
    # the operators below refuse what would hand a kernel other memory than it expects
    from self_trainable_or_free_attn_amd import _lib
    op, x = _lib.ops().packed_attention, q.detach()
    cu = cu.to(dev)
    for bad in ((x.transpose(0, 1), x, x, None, None, None, None, 1), (x, x, x[:3], None, None, None, None, 1),
                (x, x, x.half(), None, None, None, None, 1), (x, x, x, None, cu, cu, None, 2),
                (x, x, x, None, cu.long(), None, None, 1), (x, x, x.cpu(), None, None, None, None, 1),
                (x, x, x, torch.zeros(4, 3, device=dev), None, None, cu[:1], 1),
                (x, x, x, torch.zeros(4, 2, device=dev), None, None, cu, 1),
                (x, x, x, torch.zeros(4, 2, device=dev), None, None, None, 1), (x, x, x, None, None, None, None, 0),
                (x, x, x, None, None, None, None, 3), (x.float(), x.float(), x.float(), None, None, None, None, 1)):
        with pytest.raises(RuntimeError):
            op(*bad, False, 1.0)


def test_compiled(dev):
    api = _api()
    lens = [100, 28]
    t = _inputs(lens, lens, 4, 2, 64, BF, dev, 35)
    cu = _cu(lens, dev)
    leaves = [t[n].requires_grad_() for n in "qkv"]

    def step(q, k, v):
        return api.packed_attention(q, k, v, cu, causal=True) * 2

    want = step(*leaves)
    got = torch.compile(step, backend="aot_eager")(*leaves)
    assert torch.equal(got, want)
    for x, y in zip(torch.autograd.grad(got, leaves, t["dout"]), torch.autograd.grad(want, leaves, t["dout"])):
        assert torch.equal(x, y)
