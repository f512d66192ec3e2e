"""Appending to paged caches of 16 and 4 bits and reading rows back, against plain 64-bit arithmetic (paged_ref.py)."""
import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _api():
    import self_trainable_or_free_attn_amd as api
    return api


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _noise(cache, g):
    """Fills a cache with anything."""
    for x in cache:
        if x is None:
            continue
        if x.dtype is torch.uint8:
            x.copy_(torch.randint(100, 140, x.shape, generator=g, device=x.device, dtype=torch.uint8))
        else:
            x.copy_(torch.randn(x.shape, generator=g, device=x.device))
    return cache


def _values(cache, dtype):
    """(k, v) of a whole cache in float64."""
    if cache.k_scales is None:
        return cache.k.double(), cache.v.double()
    return ref.decode4(cache.k, cache.k_scales), ref.decode4(cache.v, cache.v_scales)


def _case(dev, lens, keys, H, Hk, D, dtype, page, bits, R, halves, norm, seed, pad=0, cache=None, holes=(), x=None):
    """Appends, checks the new rows, that every other row kept its bits, and that paged_rows returns what is held."""
    api = _api()
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)
    T = sum(lens) + pad
    wide = (1.5 * rnd(T, H + 2 * Hk, D)).to(dtype) if x is None else x
    if pad:
        wide[T - pad:] = math.nan
    q, k, v = wide[:, :H], wide[:, H:H + Hk], wide[:, H + Hk:]
    qw, kw = ((1 + 0.3 * rnd(D)).to(dtype) for _ in "qk") if norm else (None, None)
    table = api.rotary_table(max(max(keys), 1), R, device=dev) if R else None
    pages, num = ref.page_table(keys, page, 2, dev, seed)
    for b, i in holes:
        pages[b, i] = num + 7 if b % 2 else -3
    cache = _noise(cache or api.paged_cache(num, Hk, D, page_size=page, bits=bits, dtype=dtype, device=dev), g)
    before = [None if c is None else c.clone() for c in cache]
    cu, total = _ints(ref.starts(lens), dev), _ints(keys, dev)
    out = api.append_paged(cache, k, v, pages, total, cu, q=q if H else None, q_weight=qw if H else None, k_weight=kw,
                           table=table, halves=halves)
    held = _values(cache, dtype)
    touched = torch.zeros(num, page, dtype=torch.bool, device=dev)
    rows_k, rows_v = api.paged_rows(cache, pages, total, cu, rows=T, dtype=dtype)
    want_rows = [torch.zeros(T, Hk, D, device=dev, dtype=torch.float64) for _ in "kv"]
    if H:
        assert out.is_contiguous() and out.shape == q.shape
        assert not out[T - pad:].any() if pad else True
    for b, (at, n, m) in enumerate(zip(ref.starts(lens), lens, keys)):
        for i0 in range(n):
            if m - n + i0 < 0 and H:
                assert not out[at + i0].any()
        skip = max(n - m, 0)                  # tokens of negative positions
        pos = torch.arange(m - n + skip, m, device=dev)
        sl = slice(at + skip, at + n)
        cs = table[pos] if R else torch.zeros(len(pos), 0, 2, device=dev)
        if H:
            ref.check("q", out[sl], *ref.rotate(q[sl], qw, cs, 1e-6, halves)["y"])
        number = pages[b].long()[pos // page]
        keep = (number >= 0) & (number < num)
        number, row = number[keep], (pos % page)[keep]
        touched[number, row] = True
        sl = torch.arange(at + skip, at + n, device=dev)[keep]
        want = ref.rotate(k[sl], kw, cs[keep], 1e-6, halves)["y"]
        if bits == 16:
            ref.check("k", held[0][number, :, row], *want)
            assert torch.equal(held[1][number, :, row], v[sl].double())
        else:
            for i, x32 in ((0, want[0].float()), (1, v[sl].float())):
                vals, e = ref.held4(x32, dtype)
                assert torch.equal(cache[2 + i][number, :, row].long() - 127, e.long()), "scales"
                assert torch.equal(held[i][number, :, row], vals), "values"
        for i in (0, 1):
            want_rows[i][sl] = held[i][number, :, row]
    assert torch.equal(rows_k.double(), want_rows[0]) and torch.equal(rows_v.double(), want_rows[1])
    for c, old in zip(cache, before):
        if c is not None:
            assert torch.equal(c.transpose(1, 2)[~touched], old.transpose(1, 2)[~touched]), "a row that no token is held in"
    return cache, out


RAGGED = [([1], [1]), ([1, 1, 1, 1], [129, 1, 77, 300]), ([0, 5, 0, 33, 1, 0], [0, 5, 9, 40, 200, 3]), ([64, 16, 17], [64, 32, 300])]


@pytest.mark.parametrize("D, dtype", [(64, BF), (128, BF), (64, FP), (128, FP)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens, keys", RAGGED)
@pytest.mark.parametrize("halves", [False, True])
def test_append(dev, D, dtype, bits, lens, keys, halves):
    _case(dev, lens, keys, 6, 2, D, dtype, 16, bits, D, halves, True, seed=1, pad=3)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("R, halves, norm", [(0, False, False), (0, True, True), (16, True, True), (48, True, False), (48, False, True),
                                             (64, True, True)])
@pytest.mark.parametrize("D", [64, 128])
def test_parts_of_the_turn(dev, bits, R, halves, norm, D):
    _case(dev, [9, 1], [40, 70], 3, 3, D, BF, 32, bits, R, halves, norm, seed=2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page", [16, 64, 256, 4096])
def test_page_sizes(dev, bits, page):
    _case(dev, [300, 1], [1000, 4097], 4, 1, 64, FP, page, bits, 64, True, True, seed=3)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Hk", [1, 2, 5, 9])
def test_without_queries(dev, bits, Hk):
    _case(dev, [3, 40], [30, 50], 0, Hk, 128, BF, 16, bits, 128, True, True, seed=4, pad=2)


@pytest.mark.parametrize("bits", [16, 4])
def test_tokens_without_a_place(dev, bits):
    """More new tokens than the sequence holds, pages that do not exist."""
    _case(dev, [20, 3, 40, 17], [7, 0, 90, 64], 2, 2, 64, BF, 16, bits, 64, False, True, seed=5, pad=1,
          holes=((0, 0), (2, 3), (3, 2)))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_many_sequences(dev, bits, B):
    _case(dev, [(7 * i) % 5 for i in range(B)], [(7 * i) % 5 + 11 * i % 60 for i in range(B)], 2, 1, 64, BF, 16, bits, 64, True,
          True, seed=6)


@pytest.mark.parametrize("bits", [16, 4])
def test_long_prompt(dev, bits):
    _case(dev, [5000, 700], [9000, 700], 8, 2, 128, BF, 64, bits, 128, True, True, seed=7)


def test_equal_counts_without_cu(dev):
    api, B, n, H, Hk, D = _api(), 5, 3, 4, 2, 64
    g = torch.Generator(device=dev).manual_seed(8)
    q, k, v = ((torch.randn(B, n, h, D, device=dev, generator=g)).to(BF) for h in (H, Hk, Hk))
    pages, num = ref.page_table([40] * B, 16, 0, dev, 8)
    lens, table = _ints([3, 40, 17, 16, 33], dev), api.rotary_table(40, D, device=dev)
    got = []
    for cu in (None, _ints(ref.starts([n] * B), dev)):
        cache = api.paged_cache(num, Hk, D, page_size=16, dtype=BF, device=dev)
        flat = [x if cu is None else x.flatten(0, 1) for x in (q, k, v)]
        out = api.append_paged(cache, flat[1], flat[2], pages, lens, cu, q=flat[0], table=table)
        got.append((out.view(B * n, H, D), *cache[:2], *api.paged_rows(cache, pages, lens, cu, rows=B * n)))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    # without weights and table keys and queries stay as they are
    cache = api.paged_cache(num, Hk, D, page_size=16, dtype=BF, device=dev)
    assert torch.equal(api.append_paged(cache, k, v, pages, lens, q=q), q)
    assert torch.equal(api.paged_rows(cache, pages, lens, rows=B * n)[0], k.flatten(0, 1))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_4_bit_values_and_their_borders(dev, dtype):
    """Every border of two codes, the values on either side of it, both signs, and scales over the whole range: 32 channels of
    one row are magnitudes of one exponent. Values come out exactly, by the definition."""
    D = 64
    lo, hi = ref.EXPONENTS[dtype]
    steps = torch.arange(0, 29, dtype=torch.float64) / 4                    # 0 .. 7 in quarters: every code and border
    rows = []
    for e in range(max(lo - 3, -24 if dtype is FP else -126), hi + 2):
        for top in (7.0, 6.0, 4.0, 3.75, 3.5625):                           # (3.5 and below belong to the next smaller scale)
            row = torch.cat([steps[steps <= top][-31:], torch.tensor([top])])
            row = torch.nn.functional.pad(row, (0, 32 - len(row)))
            rows.append(torch.cat([row, -row]) * 2.0 ** e)
    x = torch.stack(rows).to(dtype).to(dev)[:, None]
    x = x[torch.isfinite(x).all(-1).all(-1)]
    T = len(x)
    pages, num = ref.page_table([T], 16, 0, dev, 9)
    cache = _api().paged_cache(num, 1, D, page_size=16, bits=4, device=dev)
    _api().append_paged(cache, x, -x, pages, _ints([T], dev), _ints([0, T], dev))
    k, v = _api().paged_rows(cache, pages, _ints([T], dev), rows=T, dtype=dtype)
    want = ref.held4(x.float(), dtype)[0]
    assert torch.isfinite(want).all()
    assert torch.equal(k.double(), want) and torch.equal(v.double(), -want)


def test_4_bit_error(dev):
    """Off by at most half a step: a quarter of s below 2 s, half from there to 4 s, s up to 7 s."""
    T, D = 500, 128
    g = torch.Generator(device=dev).manual_seed(10)
    x = (torch.randn(T, 2, D, device=dev, generator=g) * torch.exp(2 * torch.randn(T, 2, 1, device=dev, generator=g))).to(BF)
    pages, num = ref.page_table([T], 32, 0, dev, 10)
    cache = _api().paged_cache(num, 2, D, page_size=32, bits=4, device=dev)
    _api().append_paged(cache, x, x, pages, _ints([T], dev), _ints([0, T], dev))
    k, v = _api().paged_rows(cache, pages, _ints([T], dev), rows=T)
    assert torch.equal(k, v)
    s = ref.power(ref.held4(x.float(), BF)[1]).repeat_interleave(32, -1)
    a = x.double().abs() / s
    assert bool(((k.double() - x.double()).abs() <= s * torch.where(a < 2, 0.25, torch.where(a < 4, 0.5, 1.0))).all())


def test_decoding_every_code(dev):
    """All 256 bytes at every scale whose values the type holds as normal numbers."""
    for dtype, (lo, hi) in ref.EXPONENTS.items():
        scales = torch.arange(lo + 127, hi + 128, dtype=torch.uint8, device=dev)
        n = len(scales) * 8
        num = -(-n // 16)
        codes = torch.zeros(num * 16, 1, 32, dtype=torch.uint8, device=dev)
        codes[:n] = torch.arange(256, dtype=torch.uint8, device=dev).view(8, 1, 32).repeat(len(scales), 1, 1)
        sc = torch.full((num * 16, 1, 2), 127, dtype=torch.uint8, device=dev)
        sc[:n] = scales.repeat_interleave(8)[:, None, None]
        paged = lambda x: x.view(num, 16, 1, -1).transpose(1, 2).contiguous()
        cache = _api().PagedCache(paged(codes), paged(codes), paged(sc), paged(sc))
        pages = torch.arange(num, dtype=torch.int32, device=dev)[None]
        k, v = _api().paged_rows(cache, pages, _ints([n], dev), rows=n, dtype=dtype)
        want = ref.decode4(codes, sc)[:n]
        assert torch.equal(k.double(), want) and torch.equal(v.double(), want), dtype


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_tokens_past_the_pages(dev, bits, n):
    """Sequences that have outgrown their rows of pages: tokens past them go nowhere, and their queries keep their positions."""
    api, page, D, width = _api(), 16, 64, 3
    cap, g = width * page, torch.Generator(device=dev).manual_seed(16)
    keys = [cap, cap + 1, cap + n // 2, cap + n, cap + n + 50, 2 ** 31 - 1]
    B = len(keys)
    q, k, v = (torch.randn(B * n, h, D, device=dev, generator=g).to(BF) for h in (4, 2, 2))
    pages = torch.randperm(B * width, device=dev, generator=g).to(torch.int32).view(B, width)
    cache = _noise(api.paged_cache(B * width, 2, D, page_size=page, bits=bits, device=dev), g)
    before = [None if c is None else c.clone() for c in cache]
    table = api.rotary_table(cap + n + 50, D, device=dev)
    out = api.append_paged(cache, k, v, pages, _ints(keys, dev), q=q, table=table)
    pos = torch.cat([torch.arange(m - n, m, device=dev) for m in keys])
    ref.check("q", out, *ref.rotate(q, None, table[pos.clamp(max=len(table) - 1)], 1e-6, False)["y"])
    new = pos < cap
    at = pages.long()[torch.arange(B, device=dev).repeat_interleave(n)[new], pos[new] // page]
    held = _values(cache, BF)
    want = v[new].double() if bits == 16 else ref.held4(v[new].float(), BF)[0]
    assert torch.equal(held[1][at, :, pos[new] % page], want)
    touched = torch.zeros(B * width, page, dtype=torch.bool, device=dev)
    touched[at, pos[new] % page] = True
    for c, old in zip(cache, before):
        if c is not None:
            assert torch.equal(c.transpose(1, 2)[~touched], old.transpose(1, 2)[~touched])
    rows_k, rows_v = api.paged_rows(cache, pages, _ints(keys, dev), rows=B * n, dtype=BF)
    assert torch.equal(rows_v[new].double(), want) and not rows_k[~new].any() and not rows_v[~new].any()


def test_layouts_of_a_cache(dev):
    """Rows of all heads side by side, keys and values in one allocation, pages far apart: the same contents."""
    api, Hk, D, page, keys = _api(), 3, 64, 16, [50, 20]
    lens = [50, 4]
    pages, num = ref.page_table(keys, page, 2, dev, 11)
    tokens = lambda: torch.zeros(num, page, Hk, D, dtype=BF, device=dev).transpose(1, 2)
    both = torch.zeros(num, 2, Hk, page, D, dtype=BF, device=dev)
    padded = [torch.zeros(num, Hk, page, D + 8, dtype=BF, device=dev)[..., :D] for _ in "kv"]
    got = []
    for cache in (api.paged_cache(num, Hk, D, page_size=page, dtype=BF, device=dev), api.PagedCache(tokens(), tokens()),
                  api.PagedCache(both[:, 0], both[:, 1]), api.PagedCache(*padded)):
        c, out = _case(dev, lens, keys, 6, Hk, D, BF, page, 16, D, True, True, seed=11, cache=cache)
        got.append((out, *api.paged_rows(c, pages, _ints(keys, dev), _ints(ref.starts(lens), dev), rows=54)))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("bits", [16, 4])
def test_cache_past_32_bits(dev, bits):
    """Pages whose rows start beyond 2^32 bytes."""
    api, Hk, D, page = _api(), 8, 128, 256
    held = Hk * page * (D * 2 if bits == 16 else D // 2)
    num = (1 << 32) // held + 40
    cache = api.paged_cache(num, Hk, D, page_size=page, bits=bits, dtype=BF, device=dev)
    x = torch.randn(300, Hk, D, device=dev).to(BF)
    pages = _ints([[num - 1, num - 20]], dev)
    api.append_paged(cache, x, x, pages, _ints([300], dev))
    k, _ = api.paged_rows(cache, pages, _ints([300], dev), rows=300)
    if bits == 16:
        assert torch.equal(k, x) and torch.equal(cache.k[num - 1], x[:256].transpose(0, 1))
    else:
        assert torch.equal(k.double(), ref.held4(x.float(), BF)[0])
        assert torch.equal(ref.decode4(cache.k[num - 20, :, :44], cache.k_scales[num - 20, :, :44]).transpose(0, 1), k[256:].double())


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_append(dev, bits):
    """A step of single tokens in a graph, replayed at other lengths and pages."""
    api, B, H, Hk, D, page = _api(), 6, 4, 2, 64, 16
    g = torch.Generator(device=dev).manual_seed(12)
    q, k, v = (torch.randn(B, h, D, device=dev, generator=g).to(BF) for h in (H, Hk, Hk))
    w, table = torch.ones(D, device=dev, dtype=BF), api.rotary_table(200, D, device=dev)
    pages, num = ref.page_table([100] * B, page, 0, dev, 12)
    lens = _ints([1] * B, dev)
    caches = [api.paged_cache(num, Hk, D, page_size=page, bits=bits, device=dev) for _ in "abc"]
    step = lambda c: api.append_paged(c, k, v, pages, lens, q=q, q_weight=w, k_weight=w, table=table)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(caches.pop())      # (a cache of its own: the capture itself writes nothing)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for n in (1, 17, 60, 61):
        lens.fill_(n)
        lens[2] = 0
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=dev, generator=g))
        graph.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(*caches) if a is not None)


def test_a_graph_that_saved_the_cache_sees_the_change(dev):
    api = _api()
    cache = api.paged_cache(2, 1, 64, page_size=16, device=dev)
    x = torch.randn(4, 1, 64, device=dev).to(BF)
    w = torch.ones(64, device=dev, dtype=BF, requires_grad=True)
    y = (cache.k * w).sum()
    api.append_paged(cache, x, x, _ints([[0]], dev), _ints([4], dev))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_under_inference_mode(dev):
    api = _api()
    with torch.inference_mode():
        cache = api.paged_cache(2, 1, 64, page_size=16, device=dev)
        x = torch.randn(4, 1, 64, device=dev).to(BF)
        api.append_paged(cache, x, x, _ints([[0]], dev), _ints([4], dev))
        assert torch.equal(api.paged_rows(cache, _ints([[0]], dev), _ints([4], dev), rows=4)[0], x)
