"""Attention over paged caches of 16 and 4 bits against plain 64-bit attention over what the cache holds (packed_ref.py, which
derives the bounds): lengths from nothing to long, page sizes, grouped heads, rows that see nothing, pages that do not exist, stale
rows full of NaN, tiles cut into pieces, streams, graphs, and a decoding loop of all operators together."""
import math

import pytest
import torch

import packed_ref
import paged_ref as ref

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _api():
    import self_trainable_or_free_attn_amd as api
    return api


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _filled(num, Hk, D, page, bits, dtype, dev, g):
    """A cache of random values."""
    cache = _api().paged_cache(num, Hk, D, page_size=page, bits=bits, dtype=dtype, device=dev)
    for x in cache[:2]:
        if bits == 4:
            x.copy_(torch.randint(0, 256, x.shape, device=dev, generator=g, dtype=torch.uint8))
        else:
            x.copy_(torch.randn(x.shape, device=dev, generator=g))
    for x in cache[2:] if bits == 4 else ():
        x.copy_(torch.randint(124, 128, x.shape, device=dev, generator=g, dtype=torch.uint8))
    return cache


def _spoil(cache, pages, keys, page):
    """What no key needs: pages that no sequence names, and rows past a sequence's last, as NaN (4 bits: scales past any type)."""
    num = cache.k.shape[0]
    used = torch.zeros(num, page, dtype=torch.bool, device=cache.k.device)
    for b, m in enumerate(keys):
        for i in range(-(-m // page)):
            p = int(pages[b, i])
            if 0 <= p < num:
                used[p, :min(page, m - i * page)] = True
    if cache.k_scales is None:
        for x in cache[:2]:
            x.transpose(1, 2)[~used] = math.nan
    else:
        for x in cache[2:]:
            x.transpose(1, 2)[~used] = 255


def _want(q, cache, pages, lens, keys, page, causal, scale, dtype):
    H, D = q.shape[1:]
    Hk = cache.k.shape[1]
    G, num = H // Hk, cache.k.shape[0]
    if cache.k_scales is None:
        held = [x.double() for x in cache[:2]]
    else:
        held = [ref.decode4(c, s) for c, s in zip(cache[:2], cache[2:])]
    dev = q.device
    out = [torch.zeros(q.shape, device=dev, dtype=torch.float64) for _ in "vb"]
    lse = [torch.full(q.shape[:2], x, device=dev, dtype=torch.float64) for x in (-math.inf, 0.0)]
    for b, (at, n, m) in enumerate(zip(ref.starts(lens), lens, keys)):
        table = pages[b].clamp(0, max(num - 1, 0))
        there = ((pages[b] >= 0) & (pages[b] < num)).repeat_interleave(page)[:m]
        i = torch.arange(n, device=dev)[:, None] + m - n
        j = torch.arange(m, device=dev)[None]
        seen = (j <= i if causal else torch.ones(n, m, dtype=torch.bool, device=dev)) & there
        for h in range(Hk):
            k, v = (ref.gathered(x[:, h:h + 1], table, m, page)[:, 0] for x in held)
            k, v = (torch.where(there[:, None], x, 0.0) for x in (k, v))
            hs = slice(h * G, h * G + G)
            r = packed_ref.attention(q[at:at + n, hs].double().transpose(0, 1), k, v, seen, scale, dtype=dtype)
            live = seen.any(1)
            # Float32 ends at 2^-126: a probability below that vanishes. They are taken against a maximum that is at most one power
            # of two above the row's largest score, so this is up to 2^-125 of the row's sum, times |v|, and as much again for an
            # output that small. (Values of a 4-bit cache are often zero: nothing larger stands beside such terms then.)
            r["out"] = (r["out"][0], r["out"][1] + 2.0 ** -125 * (v.abs().sum(0) + 1))
            for x in (0, 1):
                out[x][at:at + n, hs] = torch.where(live[:, None, None], r["out"][x].transpose(0, 1), 0.0)
                lse[x][at:at + n, hs] = torch.where(live[:, None], r["lse"][x].transpose(0, 1), -math.inf if x == 0 else 0.0)
    return out, lse


def _case(dev, lens, keys, H, Hk, D, dtype, page, bits, seed, causal=True, pad=0, holes=(), scale=None, width=None, cu=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(lens) + pad
    q = (1.5 * torch.randn(T, H, D, device=dev, generator=g)).to(dtype)
    if pad:
        q[T - pad:] = math.nan
    pages, num = ref.page_table(keys, page, 1, dev, seed, width)
    for b, i in holes:
        pages[b, i] = num if b % 2 else -1
    cache = _filled(num, Hk, D, page, bits, dtype, dev, g)
    _spoil(cache, pages, keys, page)
    out, lse = _api().paged_attention(q, cache, pages, _ints(keys, dev), _ints(ref.starts(lens), dev) if cu else None, causal=causal,
                                      scale=scale, return_lse=True)
    clean = type(cache)(*(None if x is None else torch.where(x == 255, 127, x) if x.dtype == torch.uint8 and i > 1
                          else torch.nan_to_num(x) if x.dtype != torch.uint8 else x for i, x in enumerate(cache)))
    want_out, want_lse = _want(torch.nan_to_num(q), clean, pages, lens, keys, page, causal, scale or D ** -0.5, dtype)
    packed_ref.check("out", out, *want_out)
    packed_ref.check("lse", lse, *want_lse)


TYPES = [(64, BF), (128, BF), (64, FP), (128, FP)]
RAGGED = [
    ([1], [1]), ([1, 1, 1, 1], [129, 1, 77, 300]), ([0, 5, 0, 33, 1, 0], [0, 5, 9, 33, 200, 3]),
    ([64, 128, 127, 129, 65], [64, 128, 127, 300, 65]),
    ([3, 40, 200, 2], [0, 7, 150, 0]),                 # fewer keys than new tokens: rows without keys under a causal mask
    ([1, 17, 130], [300, 100, 131]), ([16, 15, 33], [16, 47, 63]),
]


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H, Hk", [(2, 2), (6, 2), (8, 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens, keys", RAGGED)
def test_attention(dev, D, dtype, bits, H, Hk, causal, lens, keys):
    _case(dev, lens, keys, H, Hk, D, dtype, 16, bits, seed=1, causal=causal, pad=9)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 8, 16, 17, 32, 33])
def test_single_tokens_of_any_group(dev, D, dtype, bits, G):
    _case(dev, [1, 1, 1], [70, 33, 515], 2 * G, 2, D, dtype, 32, bits, seed=2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024, 4096])
def test_page_sizes(dev, bits, page):
    _case(dev, [1, 40, 1, 2], [1000, 777, 33, 5000], 4, 1, 64, BF, page, bits, seed=3)
    _case(dev, [1, 1, 1, 1], [1000, 777, 33, 5000], 4, 1, 128, FP, page, bits, seed=4)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens, keys, H, Hk", [
    ([1500, 700], [2500, 1700], 3, 1),                           # ranges of wide tiles
    ([1, 1, 1], [5000, 64, 1029], 10, 2),                       # of single tokens
    ([33, 2, 300], [4100, 2500, 70], 5, 5),                     # narrow and wide tiles in one launch
    ([2, 1, 1, 600], [0, 3500, 1, 600], 4, 2),
    ([1], [40000], 16, 2), ([1, 0, 1], [2049, 5000, 9000], 8, 8),
])
@pytest.mark.parametrize("causal", [False, True])
def test_key_ranges(dev, D, dtype, bits, lens, keys, H, Hk, causal):
    _case(dev, lens, keys, H, Hk, D, dtype, 16, bits, seed=5, causal=causal)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("bits", [16, 4])
def test_equal_counts_without_cu(dev, D, dtype, bits):
    """Drafted tokens: a few each, with and without running counts that say the same; as a batch."""
    api, B, n, H, Hk, page = _api(), 3, 4, 8, 2, 16
    _case(dev, [n] * B, [40, 1700, 4], H, Hk, D, dtype, page, bits, seed=6, cu=False)
    _case(dev, [n] * B, [40, 1700, 3], H, Hk, D, dtype, page, bits, seed=6)
    g = torch.Generator(device=dev).manual_seed(7)
    pages, num = ref.page_table([40, 100, 4], page, 0, dev, 7)
    cache = _filled(num, Hk, D, page, bits, dtype, dev, g)
    q = torch.randn(B, n, H, D, device=dev, generator=g).to(dtype)
    lens = _ints([40, 100, 4], dev)
    a, la = api.paged_attention(q, cache, pages, lens, return_lse=True)
    b, lb = api.paged_attention(q.flatten(0, 1), cache, pages, lens, return_lse=True)
    assert a.shape == q.shape and la.shape == q.shape[:3]
    assert torch.equal(a.flatten(0, 1), b) and torch.equal(la.flatten(0, 1), lb)


@pytest.mark.parametrize("D, dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("bits", [16, 4])
def test_many_heads(dev, D, dtype, bits):
    """Grids that fill the GPU: whole tiles."""
    _case(dev, [300, 1, 70, 0, 129], [300, 1, 200, 5, 1500], 128, 128, D, dtype, 64, bits, seed=8, pad=2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("B", [63, 64, 65, 200])
@pytest.mark.parametrize("most", [1, 3])
def test_many_sequences(dev, bits, B, most):
    lens = [(7 * i) % (most + 1) for i in range(B)]
    _case(dev, lens, [n + 11 * i % 40 + 60 * (i % 30 == 7) for i, n in enumerate(lens)], 3, 1, 64, BF, 16, bits, seed=9, pad=1)
    _case(dev, lens, [n + 11 * i % 40 + 3000 * (i % 30 == 7) for i, n in enumerate(lens)], 3, 1, 64, BF, 16, bits, seed=9)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("most", [1, 2])
@pytest.mark.parametrize("B", [300, 600])
def test_more_sequences_than_a_wave_reads_at_once(dev, bits, most, B):
    """255 at a time: single tokens in shares, more of them in ranges; a few long histories among short ones, some without keys."""
    lens = [(5 * i) % (most + 1) if most > 1 else 1 for i in range(B)]
    keys = [n + (13 * i) % 30 + (4000 if i % 97 == 5 else 0) if i % 11 else 0 for i, n in enumerate(lens)]
    _case(dev, lens, keys, 4, 2, 64, BF, 16, bits, seed=21, pad=2 if most > 1 else 0)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("lens", [[200] + [0] * 199, [0] * 30 + [7, 90] + [1] * 100, [33] + [1] * 40 + [0] * 32])
def test_few_sequences_have_most_of_the_tokens(dev, bits, G, lens):
    """No more tokens than sequences, so the call takes them for single ones, but some sequences have many: tiles of few rows whose
    pieces under a causal mask see a part of the keys, next to empty sequences."""
    for extra in (0, 3000):
        keys = [n + (extra if n > 1 else 5 * i % 70) if n else 0 for i, n in enumerate(lens)]
        for causal in (True, False):
            _case(dev, lens, keys, 2 * G, 2, 64, FP, 32, bits, seed=22, causal=causal, width=200)


@pytest.mark.parametrize("D, dtype", [(64, BF), (128, FP)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B", [1, 2, 15, 16, 63, 64, 255, 256])
def test_cuts_of_wide_tiles(dev, D, dtype, bits, causal, B):
    """Prompts, pieces and single tokens of every length: tiles that are cut into none to many pieces, of as many sequences as rows
    of lanes, waves and passes hold, the rows behind the last one among them."""
    for many in (False, True):
        n = lambda i: [700, 40, 1, 90][i % 4] if B < 60 or i % 40 < 2 else 1 + i % 3
        lens = [n(i) for i in range(B)]
        keys = [m + [0, 1500, 130, 5000][i % 4] // (1 if B < 60 or i % 20 == 3 else 50) if i % 9 < 8 else m // 2
                for i, m in enumerate(lens)]
        _case(dev, lens, keys, 6 if many else 1, 2 if many else 1, D, dtype, 32, bits, seed=23, causal=causal, pad=B % 3)


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(dev, seed):
    """Any mix of tokens, pieces and prompts, heads, pages and holes, tables of pages longer than needed (so that the call cuts)."""
    import random
    rng = random.Random(seed)
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    B = log(1, 90)
    single = rng.random() < 0.6
    lens = [1 if single or rng.random() < 0.7 else log(1, 300) for _ in range(B)]
    if rng.random() < 0.3:
        lens[rng.randrange(B)] = 0
    keys = [0 if rng.random() < 0.05 else max(0, n + log(1, 6000) - (rng.random() < 0.1) * n) for n in lens]
    Hk = rng.choice([1, 2, 3, 8, 40])
    H, D, page = Hk * rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 128]), rng.choice([16, 32, 64, 256])
    used = [(b, i) for b, m in enumerate(keys) for i in range(-(-m // page))]
    holes = rng.sample(used, min(len(used), rng.choice([0, 0, 3])))
    while sum(n * m for n, m in zip(lens, keys)) * H > 40_000_000:      # (the 64-bit result's time)
        i = max(range(B), key=lambda b: lens[b] * keys[b])
        lens[i] = max(1, lens[i] // 2)
        if lens[i] == 1:
            break
    _case(dev, lens, keys, H, Hk, D, rng.choice([BF, FP]), page, rng.choice([16, 4]), seed=100 + seed, causal=rng.random() < 0.8,
          pad=rng.choice([0, 3]), holes=holes, width=-(-max(max(keys), 1) // page) + rng.choice([0, 1, 100]))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [40, 1, 100, 20]])
@pytest.mark.parametrize("width", [None, 200])
def test_pages_that_do_not_exist(dev, bits, lens, width):
    """Their keys are left out: in the middle, at the ends, and all of a sequence's."""
    keys = [200, 40, 1500, 20]
    holes = [(0, 0), (0, 5), (1, 2), (2, 0), (2, 30), (2, 31), (2, 93), (3, 0), (3, 1)]
    for D, dtype in ((64, BF), (128, FP)):
        _case(dev, lens, keys, 4, 2, D, dtype, 16, bits, seed=10, holes=holes, width=width)


@pytest.mark.parametrize("bits", [16, 4])
def test_an_empty_cache(dev, bits):
    api = _api()
    cache = api.paged_cache(0, 2, 64, page_size=16, bits=bits, device=dev)
    q = torch.randn(3, 4, 64, device=dev).to(BF)
    for width in (0, 3, 100):
        pages = torch.zeros(3, width, dtype=torch.int32, device=dev)
        out, lse = api.paged_attention(q, cache, pages, _ints([5, 0, 40], dev), return_lse=True)
        assert not out.any() and bool((lse == -math.inf).all())
        x = torch.randn(3, 2, 64, device=dev).to(BF)
        assert torch.equal(api.append_paged(cache, x, x, pages, _ints([5, 1, 40], dev), q=q), q)    # (nowhere held, all the same)
        k, v = api.paged_rows(cache, pages, _ints([5, 0, 40], dev), rows=3)
        assert not k.any() and not v.any()
    out = api.paged_attention(q[:0], cache, torch.zeros(1, 3, dtype=torch.int32, device=dev), _ints([5], dev))
    assert out.shape == (0, 4, 64)


@pytest.mark.parametrize("bits", [16, 4])
def test_lengths_past_the_pages(dev, bits):
    """A length is held to what the row of pages names, and to nothing."""
    api = _api()
    g = torch.Generator(device=dev).manual_seed(11)
    cache = _filled(8, 1, 64, 16, bits, BF, dev, g)
    pages = _ints([[3, 1], [7, 2]], dev)
    q = torch.randn(2, 2, 64, device=dev, generator=g).to(BF)
    far = api.paged_attention(q, cache, pages, _ints([10 ** 9, -5], dev), return_lse=True)
    want = api.paged_attention(q, cache, pages, _ints([32, 0], dev), return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(far, want))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n, width", [(1, 2), (7, 2), (40, 2), (90, 3), (1, 100), (5, 90), (300, 90)])
def test_tokens_past_the_pages(dev, bits, causal, n, width):
    """Sequences that have outgrown their rows of pages: each token keeps its position and sees what is held."""
    api, page, H, D = _api(), 16, 4, 64
    cap = width * page
    g = torch.Generator(device=dev).manual_seed(15)
    lens, keys = [n] * 5, [cap, cap + 1, cap + n, cap + n + 50, cap + n // 2]
    cache = _filled(5 * width, 1, D, page, bits, BF, dev, g)
    pages = torch.randperm(5 * width, device=dev, generator=g).to(torch.int32).view(5, width)
    longer = torch.nn.functional.pad(pages, (0, -(-(n + 50) // page)), value=-1)
    q = torch.randn(5 * n, H, D, device=dev, generator=g).to(BF)
    out, lse = api.paged_attention(q, cache, pages, _ints(keys, dev), causal=causal, return_lse=True)
    want_out, want_lse = _want(q, cache, longer, lens, keys, page, causal, D ** -0.5, BF)
    packed_ref.check("out", out, *want_out)
    packed_ref.check("lse", lse, *want_lse)


@pytest.mark.parametrize("D, dtype", [(64, BF), (128, FP)])
@pytest.mark.parametrize("bits", [16, 4])
def test_large_and_small_scores(dev, D, dtype, bits):
    """Rows whose scores spread over thousands, and scores that are all alike."""
    _case(dev, [1, 30, 1], [900, 60, 3000], 4, 2, D, dtype, 16, bits, seed=12, scale=40.0)
    _case(dev, [1, 30, 1], [900, 60, 3000], 4, 2, D, dtype, 16, bits, seed=13, scale=1e-6)


def test_layouts_of_a_cache(dev):
    """Rows of all heads side by side, keys and values in one allocation, channels behind padding: the same bits."""
    api, Hk, D, page, num = _api(), 3, 64, 16, 30
    g = torch.Generator(device=dev).manual_seed(14)
    plain = _filled(num, Hk, D, page, 16, BF, dev, g)
    tokens = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in plain[:2]]
    both = torch.stack(plain[:2], 1)
    padded = [torch.nn.functional.pad(x, (0, 8), value=math.nan)[..., :D] for x in plain[:2]]
    pages = torch.randperm(num, device=dev, generator=g).to(torch.int32).view(2, 15)
    for lens, n in (([230, 100], 1), ([230, 100], 60)):
        q = torch.randn(2 * n, 6, D, device=dev, generator=g).to(BF)
        want = api.paged_attention(q, plain, pages, _ints(lens, dev), return_lse=True)
        for cache in (api.PagedCache(*tokens), api.PagedCache(both[:, 0], both[:, 1]), api.PagedCache(*padded)):
            got = api.paged_attention(q, cache, pages, _ints(lens, dev), return_lse=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("bits", [16, 4])
def test_cache_past_32_bits(dev, bits):
    """Pages that start beyond 2^32 bytes give what the same pages at the front give."""
    api, Hk, D, page = _api(), 8, 128, 256
    held = Hk * page * (D * 2 if bits == 16 else D // 2)
    num = (1 << 32) // held + 40
    big = api.paged_cache(num, Hk, D, page_size=page, bits=bits, dtype=BF, device=dev)
    g = torch.Generator(device=dev).manual_seed(15)
    small = _filled(3, Hk, D, page, bits, BF, dev, g)
    for x, y in zip(big, small):
        if x is not None:
            x[num - 3:] = y
    for n in (1, 50):
        q = torch.randn(n, 16, D, device=dev, generator=g).to(BF)
        a = api.paged_attention(q, big, _ints([[num - 1, num - 3, num - 2]], dev), _ints([700], dev), return_lse=True)
        b = api.paged_attention(q, small, _ints([[2, 0, 1]], dev), _ints([700], dev), return_lse=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [16, 4])
def test_same_as_packed_attention(dev, bits):
    """The rows that the cache gives back, attended to as packed sequences, give the same within both operators' bounds."""
    api, lens, keys, H, Hk, D, page = _api(), [5, 1, 60], [300, 1200, 60], 6, 2, 128, 32
    g = torch.Generator(device=dev).manual_seed(16)
    pages, num = ref.page_table(keys, page, 0, dev, 16)
    cache = _filled(num, Hk, D, page, bits, BF, dev, g)
    q = torch.randn(sum(lens), H, D, device=dev, generator=g).to(BF)
    cu_q, cu_k = _ints(ref.starts(lens), dev), _ints(ref.starts(keys), dev)
    k, v = api.paged_rows(cache, pages, _ints(keys, dev), cu_k, rows=sum(keys), dtype=BF)
    a, la = api.paged_attention(q, cache, pages, _ints(keys, dev), cu_q, return_lse=True)
    b, lb = api.packed_attention(q, k, v, cu_q, cu_k, causal=True, return_lse=True)
    want = packed_ref.packed(q, k, v, lens, keys, True, D ** -0.5)
    for x, l in ((a, la), (b, lb)):
        packed_ref.check("out", x, *want["out"])
        packed_ref.check("lse", l, *want["lse"])


@pytest.mark.parametrize("bits", [16, 4])
def test_same_bits_twice_and_side_by_side(dev, bits):
    """Two calls at once on two streams, each with a workspace of its own."""
    api, B, H, Hk, D, page = _api(), 12, 16, 2, 128, 16
    g = torch.Generator(device=dev).manual_seed(17)
    keys = [1 + 777 * i % 5000 for i in range(B)]
    pages, num = ref.page_table(keys, page, 0, dev, 17)
    cache = _filled(num, Hk, D, page, bits, BF, dev, g)
    qs = [torch.randn(B, H, D, device=dev, generator=g).to(BF) for _ in "ab"]
    lens = _ints(keys, dev)
    want = [api.paged_attention(q, cache, pages, lens, return_lse=True) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(api.paged_attention(q, cache, pages, lens, return_lse=True))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for i, (a, la) in enumerate(got):
        assert torch.equal(a, want[i % 2][0]) and torch.equal(la, want[i % 2][1])


def _prompt_layer(api, x, weights, cache, pages, lens, cu, table):
    """One layer's attention from its projection's rows: norm, rotation and append in a call, then attention over the cache."""
    H, Hk = weights["heads"]
    q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    q = api.append_paged(cache, k, v, pages, lens, cu, q=q, q_weight=weights["q"], k_weight=weights["k"], table=table, halves=True)
    return api.paged_attention(q, cache, pages, lens, cu, return_lse=True)


@pytest.mark.parametrize("bits", [16, 4])
def test_a_decoding_loop(dev, bits):
    """Prompts, then token by token with a captured step, all operators together: what comes out is the attention of the same tokens
    normed and rotated at once (16 bits; with 4, of what the cache holds of them)."""
    api, B, H, Hk, D, page, prompt, steps = _api(), 3, 8, 2, 64, 16, [37, 1, 16], 20
    g = torch.Generator(device=dev).manual_seed(18)
    total = [n + steps for n in prompt]
    x = torch.randn(sum(total), H + 2 * Hk, D, device=dev, generator=g).to(BF)
    weights = dict(heads=(H, Hk), **{n: (1 + 0.2 * torch.randn(D, device=dev, generator=g)).to(BF) for n in "qk"})
    table = api.rotary_table(100, D, device=dev)
    pages, num = ref.page_table(total, page, 1, dev, 18)
    cache = api.paged_cache(num, Hk, D, page_size=page, bits=bits, dtype=BF, device=dev)
    at = ref.starts(total)
    rows = torch.cat([torch.arange(a, a + n) for a, n in zip(at, prompt)]).to(dev)
    lens = _ints(prompt, dev)
    out, lse = torch.zeros(sum(total), H, D, device=dev, dtype=BF), torch.zeros(sum(total), H, device=dev)
    out[rows], lse[rows] = _prompt_layer(api, x[rows], weights, cache, pages, lens, _ints(ref.starts(prompt), dev), table)
    step = torch.zeros(B, H + 2 * Hk, D, device=dev, dtype=BF)
    spare = api.paged_cache(num, Hk, D, page_size=page, bits=bits, dtype=BF, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _prompt_layer(api, step, weights, spare, pages, lens, None, table)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_lse = _prompt_layer(api, step, weights, cache, pages, lens, None, table)
    for i in range(steps):
        here = torch.tensor([a + n + i for a, n in zip(at, prompt)], device=dev)
        step.copy_(x[here])
        lens.add_(1)
        graph.replay()
        out[here], lse[here] = got, got_lse
    # the whole sequences at once
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in total]).to(dev)
    q, k = api.norm_rotate(x[:, :H], x[:, H:H + Hk], weights["q"], weights["k"], table, pos, halves=True)
    hk, hv = api.paged_rows(cache, pages, lens, _ints(at, dev), rows=sum(total), dtype=BF)
    if bits == 16:
        assert torch.equal(hk, k) and torch.equal(hv, x[:, H + Hk:])
    want = packed_ref.packed(q, hk, hv, total, total, True, D ** -0.5)
    packed_ref.check("out", out, *want["out"])
    packed_ref.check("lse", lse, *want["lse"])


@pytest.mark.parametrize("bits", [16, 4])
def test_two_captured_graphs(dev, bits):
    """Each has its workspace; replays of both in turn, with eager calls between them."""
    api, B, H, Hk, D, page = _api(), 4, 8, 2, 128, 16
    g = torch.Generator(device=dev).manual_seed(19)
    pages, num = ref.page_table([3000] * B, page, 0, dev, 19)
    cache = _filled(num, Hk, D, page, bits, BF, dev, g)
    lens = _ints([1] * B, dev)
    qs = [torch.randn(B, H, D, device=dev, generator=g).to(BF) for _ in "ab"]
    call = lambda q: api.paged_attention(q, cache, pages, lens, return_lse=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(qs[0])
    torch.cuda.current_stream().wait_stream(s)
    graphs, res = [torch.cuda.CUDAGraph() for _ in qs], []
    for graph, q in zip(graphs, qs):
        with torch.cuda.graph(graph):
            res.append(call(q))
    for n in (5, 3000, 64, 1025):
        lens.copy_(_ints([n, max(n - 3, 0), 0, n // 2 + 1], dev))
        for graph in graphs:
            graph.replay()
        want = [call(q) for q in qs]
        torch.cuda.synchronize()
        for (a, la), (b, lb) in zip(res, want):
            assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_chunks_side_by_side(dev, bits):
    """Wide tiles in pieces: two graphs replayed with other lengths and counts, in turn and on two streams at once."""
    api, B, T, H, Hk, D, page = _api(), 4, 400, 6, 2, 64, 16
    g = torch.Generator(device=dev).manual_seed(24)
    pages, num = ref.page_table([4000] * B, page, 0, dev, 24)
    cache = _filled(num, Hk, D, page, bits, FP, dev, g)
    lens, cu = _ints([400, 0, 0, 0], dev), _ints([0, T, T, T, T], dev)
    qs = [torch.randn(T, H, D, device=dev, generator=g).to(FP) for _ in "ab"]
    call = lambda q: api.paged_attention(q, cache, pages, lens, cu, return_lse=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(qs[0])
    torch.cuda.current_stream().wait_stream(s)
    graphs, res = [torch.cuda.CUDAGraph() for _ in qs], []
    for graph, q in zip(graphs, qs):
        with torch.cuda.graph(graph):
            res.append(call(q))
    streams = [torch.cuda.Stream() for _ in qs]
    for counts, keys in (([400, 0, 0, 0], [400, 0, 0, 0]), ([1, 350, 1, 48], [4000, 360, 5, 3000]),
                         ([100, 100, 100, 90], [4000, 90, 2000, 1030]), ([0, 0, 0, 400], [7, 7, 7, 4000])):
        cu.copy_(_ints(ref.starts(counts), dev))
        lens.copy_(_ints(keys, dev))
        want = [call(q) for q in qs]
        for at_once in (False, True):
            for i, graph in enumerate(graphs):
                for x in res[i]:
                    x.fill_(7.0)
                streams[i].wait_stream(torch.cuda.current_stream())
                if not at_once:
                    graph.replay()
            if at_once:
                for stream, graph in zip(streams, graphs):
                    with torch.cuda.stream(stream):
                        graph.replay()
                for stream in streams:
                    torch.cuda.current_stream().wait_stream(stream)
            torch.cuda.synchronize()
            for (a, la), (b, lb) in zip(res, want):
                assert torch.equal(a, b) and torch.equal(la, lb)


def test_strided_queries(dev):
    api = _api()
    g = torch.Generator(device=dev).manual_seed(20)
    cache = _filled(8, 2, 64, 16, 16, BF, dev, g)
    pages, lens = _ints([[3, 1, 0], [7, 2, 5]], dev), _ints([40, 33], dev)
    wide = torch.randn(2, 4, 80, device=dev, generator=g).to(BF)
    want = api.paged_attention(wide[..., :64].contiguous(), cache, pages, lens)
    assert torch.equal(api.paged_attention(wide[..., :64], cache, pages, lens), want)
    odd = torch.empty(2 * 4 * 64 + 1, device=dev, dtype=BF)[1:].view(2, 4, 64).copy_(wide[..., :64])
    assert torch.equal(api.paged_attention(odd, cache, pages, lens), want)
