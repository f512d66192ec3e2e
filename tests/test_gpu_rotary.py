"""Norms of queries and keys with their rotation against plain 64-bit arithmetic (paged_ref.py, which derives the bounds): pairings,
partial rotations, layouts, positions, gradients, streams and graphs."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _api():
    import self_trainable_or_free_attn_amd as api
    return api


def _inputs(T, H, Hk, D, dtype, dev, seed, wtype=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)
    t = dict(q=(2 * rnd(T, H, D)).to(dtype), k=rnd(T, Hk, D).to(dtype), dq=rnd(T, H, D).to(dtype), dk=rnd(T, Hk, D).to(dtype))
    t["qw"], t["kw"] = ((1 + 0.3 * rnd(D)).to(wtype or dtype) for _ in "qk")
    return t


def _case(dev, T, H, Hk, D, dtype, R, halves, norm, seed, wtype=None, P=None, eps=1e-6, train=True):
    api = _api()
    t = _inputs(T, H, Hk, D, dtype, dev, seed, wtype)
    P = P or T
    table = api.rotary_table(P, R, device=dev) if R else None
    pos = torch.randint(0, P, (T,), generator=torch.Generator().manual_seed(seed)).to(dev, torch.int32) if P != T else None
    cs = torch.zeros(T, 0, 2, device=dev) if table is None else table if pos is None else table[pos.long()]
    leaves = [t["q"].requires_grad_(), t["k"].requires_grad_()]
    if norm:
        leaves += [t["qw"].requires_grad_(), t["kw"].requires_grad_()]
    out = api.norm_rotate(t["q"], t["k"], *(leaves[2:] or (None, None)), table, pos, eps=eps, halves=halves)
    grads = torch.autograd.grad(out, leaves, (t["dq"], t["dk"])) if train else ()
    for i, (n, heads) in enumerate((("q", H), ("k", Hk))):
        # terms that are added one by one: a lane's rows, 64 lane groups, a run of workgroups' sums, 16 runs
        terms = T * ((heads + 3) // 4) * 4 // min(T, 1024) + 64 + 64 + 16
        w = t[n + "w"].detach() if norm else None
        want = ref.rotate(t[n].detach(), w, cs, eps, halves, t["d" + n] if train else None, terms)
        assert out[i].dtype == dtype and out[i].is_contiguous()
        ref.check(n, out[i].detach(), *want["y"])
        if train:
            ref.check("d" + n, grads[i], *want["dx"])
        if train and norm:
            assert grads[2 + i].dtype == w.dtype
            ref.check(f"d{n}_weight", grads[2 + i], *want["dw"])


@pytest.mark.parametrize("D, dtype", [(64, BF), (128, BF), (64, FP), (128, FP)])
@pytest.mark.parametrize("part", [1, 0.5, 0, "16", "48"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_pairings(dev, D, dtype, part, halves, norm):
    R = int(part) if isinstance(part, str) else int(part * D)
    if R == 0 and not norm:
        pytest.skip("nothing to do")
    _case(dev, 37, 6, 2, D, dtype, R, halves, norm, seed=1)


@pytest.mark.parametrize("T, H, Hk", [(1, 1, 1), (1, 64, 8), (5, 3, 3), (33, 4, 1), (1000, 5, 2), (4097, 24, 8), (70001, 1, 1)])
@pytest.mark.parametrize("D, halves", [(64, False), (128, True)])
def test_sizes(dev, T, H, Hk, D, halves):
    _case(dev, T, H, Hk, D, BF, D, halves, True, seed=2, P=50 if T > 5 else None)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_float32_weights(dev, dtype):
    _case(dev, 300, 4, 2, 128, dtype, 64, True, True, seed=3, wtype=torch.float32)


@pytest.mark.parametrize("eps", [0.0, 1e-3, 10.0])
def test_eps(dev, eps):
    _case(dev, 50, 2, 2, 64, FP, 64, False, True, seed=4, eps=eps)


def test_rows_of_zeros_stay_zeros(dev):
    x = torch.zeros(7, 2, 128, device=dev, dtype=BF, requires_grad=True)
    k = torch.zeros(7, 1, 128, device=dev, dtype=BF, requires_grad=True)
    w = torch.ones(128, device=dev, dtype=BF)
    table = _api().rotary_table(7, 128, device=dev)
    q2, k2 = _api().norm_rotate(x, k, w, w, table)
    assert not q2.any() and not k2.any()
    dq, = torch.autograd.grad(q2, x, torch.ones_like(q2))
    assert torch.isfinite(dq).all()


@pytest.mark.parametrize("halves", [False, True])
def test_gradient_against_differences(dev, halves):
    """The derivative along a direction, from float64 differences of the definition, is what the gradients give."""
    D, T = 64, 9
    t = _inputs(T, 2, 2, D, FP, dev, 5, torch.float32)
    table = _api().rotary_table(T, 48, device=dev)
    leaves = [t[n].requires_grad_() for n in ("q", "k", "qw", "kw")]
    out = _api().norm_rotate(t["q"], t["k"], t["qw"], t["kw"], table, halves=halves)
    grads = torch.autograd.grad(out, leaves, (t["dq"], t["dk"]))
    g = torch.Generator(device=dev).manual_seed(6)
    for n, (x, w, dx, dw, dy) in dict(q=(t["q"], t["qw"], grads[0], grads[2], t["dq"]),
                                      k=(t["k"], t["kw"], grads[1], grads[3], t["dk"])).items():
        def loss(x, w):
            return (ref.turn(x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w, table, halves) * dy.double()).sum()
        for leaf, d in ((0, dx), (1, dw)):
            v = torch.randn(d.shape, device=dev, generator=g).double()
            a = [x.detach().double(), w.detach().double()]
            lo, hi, step = list(a), list(a), 1e-6
            lo[leaf], hi[leaf] = a[leaf] - step * v, a[leaf] + step * v
            want = (loss(*hi) - loss(*lo)) / (2 * step)
            # the gradient's own rounding (2^-11 of each value), and 1e-8 of the differences' terms
            bound = 2.0 ** -10 * (d.double() * v).abs().sum() + 1e-6 * dy.double().abs().sum()
            assert abs((d.double() * v).sum() - want) <= bound, (n, leaf)


def test_column_ranges_of_a_projection(dev):
    """Rows are read where they stand; a layout that the loads cannot take is copied; results are the same bits."""
    api, T, H, Hk, D = _api(), 40, 6, 2, 128
    table = api.rotary_table(T, D, device=dev)
    w = torch.linspace(0.5, 2, D, device=dev).to(BF)
    wide = torch.randn(T, (H + 2 * Hk) * D + 8, device=dev, generator=torch.Generator(device=dev).manual_seed(7)).to(BF)
    q, k = wide[:, :H * D].view(T, H, D), wide[:, H * D:(H + Hk) * D].view(T, Hk, D)
    want = api.norm_rotate(q.contiguous(), k.contiguous(), w, w, table)
    got = api.norm_rotate(q, k, w, w, table)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = torch.empty(T * H * D + 1, device=dev, dtype=BF)[1:].view(T, H, D).copy_(q)      # rows 2 bytes off
    assert torch.equal(api.norm_rotate(odd, k, w, w, table)[0], want[0])
    across = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(api.norm_rotate(across, k, w, w, table)[0], want[0])
    # gradients of column ranges reach the projection's rows
    wide.requires_grad_()
    q, k = wide[:, :H * D].view(T, H, D), wide[:, H * D:(H + Hk) * D].view(T, Hk, D)
    a, b = api.norm_rotate(q, k, w, w, table)
    (a.float().square().sum() + b.float().sum()).backward()
    assert wide.grad[:, :(H + Hk) * D].any() and not wide.grad[:, (H + Hk) * D:].any()


def test_batches_and_broadcast_gradients(dev):
    api, B, L, H, D = _api(), 3, 20, 4, 64
    t = _inputs(B * L, H, H, D, BF, dev, 8)
    q, k = t["q"].view(B, L, H, D), t["k"].view(B, L, H, D)
    table = api.rotary_table(L + 5, D, device=dev)
    got = api.norm_rotate(q, k, t["qw"], t["kw"], table)
    pos = torch.arange(L, device=dev, dtype=torch.int32).repeat(B)
    want = api.norm_rotate(t["q"], t["k"], t["qw"], t["kw"], table, pos)
    assert all(torch.equal(a.flatten(0, 1), b) for a, b in zip(got, want))
    assert torch.equal(api.norm_rotate(q, k, t["qw"], t["kw"], table, pos.view(B, L))[0], got[0])
    # an expanded gradient, and one output without any
    q = t["q"].requires_grad_()
    a, b = api.norm_rotate(q, t["k"], t["qw"], t["kw"], table, pos)
    g1, = torch.autograd.grad(a.sum(), q)
    a, b = api.norm_rotate(q, t["k"], t["qw"], t["kw"], table, pos)
    g2, = torch.autograd.grad(a, q, torch.ones_like(a))
    assert torch.equal(g1, g2)


def test_more_than_2_31_values(dev):
    """The last rows of a tensor whose offsets pass 32 bits, forward and backward, are what they are alone."""
    api, T, H, D = _api(), 136_000, 128, 128
    g = torch.Generator(device=dev).manual_seed(14)
    q = torch.empty(T, H, D, device=dev, dtype=BF)
    tail = torch.randn(50, H, D, device=dev, generator=g).to(BF)
    q[:-50] = 0
    q[-50:] = tail
    k = torch.zeros(T, 1, D, device=dev, dtype=BF)
    w = torch.ones(D, device=dev, dtype=BF)
    table = api.rotary_table(1000, D, device=dev)
    pos = torch.arange(T, device=dev, dtype=torch.int32) % 1000
    q.requires_grad_()
    out, _ = api.norm_rotate(q, k, w, w, table, pos)
    few = tail.clone().requires_grad_()
    want, _ = api.norm_rotate(few, k[-50:], w, w, table, pos[-50:].clone())
    assert torch.equal(out[-50:], want)
    dq, = torch.autograd.grad(out, q, torch.ones_like(out))
    dwant, = torch.autograd.grad(want, few, torch.ones_like(want))
    assert torch.equal(dq[-50:], dwant)


def test_gradients_of_broadcast_heads(dev):
    """One head's rows expanded to several, and a weight that queries and keys share."""
    api, T, D = _api(), 30, 64
    g = torch.Generator(device=dev).manual_seed(15)
    one = torch.randn(T, 1, D, device=dev, generator=g).to(BF).requires_grad_()
    w = torch.ones(D, device=dev, requires_grad=True)
    table = api.rotary_table(T, D, device=dev)
    q, k = api.norm_rotate(one.expand(T, 4, D), one, w, w, table)
    dy = torch.randn(T, 4, D, device=dev, generator=g).to(BF)
    dk = torch.randn(T, 1, D, device=dev, generator=g).to(BF)
    dx, dw = torch.autograd.grad((q, k), (one, w), (dy, dk))
    many, key = one.detach().expand(T, 4, D).contiguous().requires_grad_(), one.detach().clone().requires_grad_()
    wq, wk = (w.detach().clone().requires_grad_() for _ in "qk")
    each = torch.autograd.grad(api.norm_rotate(many, key, wq, wk, table), (many, key, wq, wk), (dy, dk))
    heads = each[0].double().sum(1, keepdim=True)
    total = heads + each[1].double()
    # the heads' sum and the keys' gradient beside it are each rounded to the token type (sums of five float32 values: 2^-21)
    bound = (2.0 ** -8 + 2.0 ** -21) * (heads.abs() + total.abs()) + 2.0 ** -21 * each[0].double().abs().sum(1, keepdim=True)
    ref.check("dx", dx, total, bound)
    ref.check("dw", dw, (each[2].double() + each[3].double()), 2.0 ** -23 * (each[2].double().abs() + each[3].double().abs()))


def test_positions_are_held_to_the_table(dev):
    api, D = _api(), 64
    x = torch.randn(4, 1, D, device=dev).to(BF)
    table = api.rotary_table(10, D, device=dev)
    ints = lambda *v: torch.tensor(v, device=dev, dtype=torch.int32)
    far = api.norm_rotate(x, x, table=table, positions=ints(-5, 10, 2 ** 31 - 1, 3))[0]
    assert torch.equal(far, api.norm_rotate(x, x, table=table, positions=ints(0, 9, 9, 3))[0])


def test_no_rows(dev):
    api = _api()
    q = torch.zeros(0, 4, 64, device=dev, dtype=BF, requires_grad=True)
    k = torch.zeros(0, 2, 64, device=dev, dtype=BF, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    a, b = api.norm_rotate(q, k, w, w, api.rotary_table(3, 64, device=dev))
    grads = torch.autograd.grad((a, b), (q, k, w), (torch.zeros_like(a), torch.zeros_like(b)))
    assert a.shape == q.shape and b.shape == k.shape and not grads[2].any()


def test_same_bits_twice_and_on_another_stream(dev):
    api = _api()
    t = _inputs(5000, 8, 2, 128, BF, dev, 9)
    table = api.rotary_table(5000, 128, device=dev)
    leaves = [t[n].requires_grad_() for n in ("q", "k", "qw", "kw")]

    def step():
        out = api.norm_rotate(t["q"], t["k"], t["qw"], t["kw"], table, halves=True)
        return (*out, *torch.autograd.grad(out, leaves, (t["dq"], t["dk"])))

    first = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured_training_step(dev):
    """A step with its gradients in a graph, replayed with other values, eager work between the replays."""
    api = _api()
    t = _inputs(300, 4, 2, 64, BF, dev, 10)
    table = api.rotary_table(300, 64, device=dev)

    def step():
        leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "qw", "kw")]
        out = api.norm_rotate(*leaves, table)
        return (*(x.detach() for x in out), *torch.autograd.grad(out, leaves, (t["dq"], t["dk"])))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for seed in (11, 12, 13):
        for n, x in _inputs(300, 4, 2, 64, BF, dev, seed).items():
            t[n].copy_(x)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_captured_step_of_leaves_of_another_stream(dev):
    """Leaves that an eager graph holds are refused in a capture, taken again once it is gone, and without gradients at once."""
    api = _api()
    t = _inputs(40, 4, 2, 64, BF, dev, 14)
    table = api.rotary_table(40, 64, device=dev)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "qw", "kw")]
    eager = api.norm_rotate(*leaves, table)
    want = [x.detach().clone() for x in eager]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="another stream"):
            api.norm_rotate(*leaves, table)
        with torch.no_grad():
            res = api.norm_rotate(*leaves, table)
        fresh = api.norm_rotate(*(x.detach().requires_grad_() for x in leaves), table)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(c.detach(), b) for a, b, c in zip(res, want, fresh))


def test_grid_table(dev):
    """Three axes: each point's rows turn by its own coordinates."""
    api, sizes, dims = _api(), (3, 4, 5), (16, 24, 24)
    table = api.rotary_table(sizes, dims, device=dev)
    x = torch.randn(60, 2, 64, device=dev).to(BF)
    got = api.norm_rotate(x, x, table=table)[0]
    f, r, c = 2, 1, 3
    row = (f * 4 + r) * 5 + c
    at = 0
    for n, (p, d) in zip("frc", zip((f, r, c), dims)):
        cs = torch.stack([torch.cos(a := p * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)), torch.sin(a)], -1)
        want = ref.turn(x[row:row + 1, :, at:at + d].double(), cs[None].to(dev), False)
        assert (got[row:row + 1, :, at:at + d].double() - want).abs().max() <= 2 ** -7 * x.abs().max(), n
        at += d
