"""The arithmetic that the packed-sequence kernels derive their work from, as they run it: csrc/packed_rules.h compiled alone for the
host."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = r"""
#include "packed_rules.h"
using namespace es;
struct Inverse {
  float off;  // relative error of the reciprocal
  float operator()(float x) const { return 1.0f / x * (1.0f + off); }
};
extern "C" {
int c_divide(int d, int x) { return divide(fast_div(d), x); }
int c_first_tile(int M, int start, int G, int b) { return M == 64 ? first_tile<64>(start, G, b) : first_tile<128>(start, G, b); }
long long c_tile_numbers(int M, int B, int T, int G) { return M == 64 ? tile_numbers<64>(B, T, G) : tile_numbers<128>(B, T, G); }
// tokens of the rows first .. first + 63 of a tile whose first token starts at row 0; the two ways in which the kernels add up
void c_tokens(int G, int first, int* a, int* b) {
  const float inv = 1.0f / (float)G, half = (float)first + 0.5f;
  for (int i = 0; i < 64; ++i) a[i] = token_of((float)i + half, inv), b[i] = token_of((float)(first + i) + 0.5f, inv);
}
void c_cut(int tiles, int chunks, int rows, float per, float off, float* out) {
  const Cut c(tiles, chunks, rows, per, Inverse{off});
  out[0] = c.ranges, out[1] = c.size;
}
float c_parts(float x, float y, float off) { return parts(x, Inverse{off}(y)); }
float c_fair(float chunks, float inv_slots) { return fair_share(chunks, inv_slots); }
int c_begin(int chunks, int range, int ranges) { return range_begin(chunks, range, ranges); }
long long c_items(long long tiles, int Hk, int D) { return range_items(tiles, Hk, D); }
int c_resident(int D) { return resident(D); }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    src, lib = d / "rules.cpp", d / "rules.so"
    src.write_text(SHIM)
    # -ffp-contract=off: the products and sums round one by one, as written
    subprocess.run(["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-shared", "-fPIC",
                    "-I", os.path.join(ROOT, "self_trainable_or_free_attn_amd", "csrc"), str(src), "-o", str(lib)], check=True)
    so = ctypes.CDLL(str(lib))
    f, i, ll = ctypes.c_float, ctypes.c_int, ctypes.c_longlong
    so.c_cut.argtypes = [i, i, i, f, f, ctypes.POINTER(f)]
    so.c_parts.argtypes, so.c_parts.restype = [f, f, f], f
    so.c_fair.argtypes, so.c_fair.restype = [f, f], f
    so.c_items.argtypes, so.c_items.restype = [ll, i, i], ll
    so.c_tile_numbers.restype = ll
    return so


def test_division(rules):
    rng = random.Random(1)
    for d in list(range(1, 70)) + [100, 127, 128, 129, 1000, 2047, 4095, 4096]:
        near = [rng.randrange(2 ** 31) // d * d + e for _ in range(60) for e in (-1, 0)]
        for x in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1] + near:
            if 0 <= x < 2 ** 31:
                assert rules.c_divide(d, x) == x // d, (d, x)


def test_tokens_of_a_tile(rules):
    a, b = (ctypes.c_int * 64)(), (ctypes.c_int * 64)()
    rows = np.arange(64)
    for G in range(1, 4097):
        for first in {0, 1, G // 3, G // 2, G - 1}:
            rules.c_tokens(G, first, a, b)
            want = (first + rows) // G
            assert (np.frombuffer(a, np.int32) == want).all() and (np.frombuffer(b, np.int32) == want).all(), (G, first)


@pytest.mark.parametrize("M", [64, 128])
def test_every_tile_has_one_number(rules, M):
    """The last sequence whose numbers start at or below w holds tile number w: every tile, those of the rows behind the last
    sequence included, is found from exactly one number of the launch."""
    rng = random.Random(2)
    for _ in range(150):
        lens = [rng.choice([0, 1, rng.randint(0, 40), rng.randint(0, 900)]) for _ in range(rng.choice([1, 3, 64, 65, 130]))]
        G, pad = rng.choice([1, 2, 3, 5, 7, 8, 16]), rng.choice([0, 1, 700])
        B, start = len(lens), [0]
        for n in lens + [pad]:
            start.append(start[-1] + n)
        base = [rules.c_first_tile(M, start[b], G, b) for b in range(B + 1)]
        numbers = rules.c_tile_numbers(M, B, start[-1], G)
        tiles = [-(-(start[b + 1] - start[b]) * G // M) for b in range(B + 1)]
        found = []
        for w in range(numbers):
            b = max(i for i in range(B + 1) if base[i] <= w)
            if w - base[b] < tiles[b]:
                found.append((b, w - base[b]))
        assert found == [(b, t) for b in range(B + 1) for t in range(tiles[b])]


def test_range_items_fit_the_grid(rules):
    """Whichever chunk count the schedule search takes, with reciprocals off by up to 2^-23, the items are no more than the launch
    has, and the ranges of a tile cover its chunks once. The lists of one launch hold up to its tile numbers of tiles."""
    rng, out, f = random.Random(3), (ctypes.c_float * 2)(), np.float32
    for _ in range(1500):
        B, Hk, D = rng.choice([1, 2, 9, 64, 100]), rng.choice([1, 2, 3, 8, 40]), rng.choice([64, 128])
        G = rng.choice([1, 3, 8])
        lists = [(rng.choice([1, 1, rng.randint(0, 500)]) * G, rng.choice([0, 1, rng.randint(0, 70), rng.randint(0, 90000)])) for _ in range(B)]
        tiles, chunks = [-(-r // 128) for r, _ in lists], [-(-m // 64) for _, m in lists]
        inv_slots = f(Hk) / f(rules.c_resident(D))
        total = f(0)
        for t, c in zip(tiles, chunks):
            total = f(total + f(t) * f(c))
        fair = rules.c_fair(total, inv_slots)
        most = max([c for t, c in zip(tiles, chunks) if t], default=0)
        for off in (-2.0 ** -23, 0.0, 2.0 ** -23):
            near = int(rules.c_parts(most, fair, off))
            for n in range(max(near - 2, 1), near + 1):
                per = max(rules.c_parts(most, n, off), fair)
                items = 0
                for t, c, (rows, _) in zip(tiles, chunks, lists):
                    rules.c_cut(t, c, rows, per, off, out)
                    ranges = int(out[0])
                    assert ranges >= 1 and out[0] == ranges
                    items += t * ranges
                    cuts = [rules.c_begin(c, i, ranges) for i in range(ranges + 1)]
                    assert cuts[0] == 0 and cuts[-1] == c and cuts == sorted(cuts)
                    if t:   # (a border off by the reciprocal's rounding at most)
                        assert max(y - x for x, y in zip(cuts, cuts[1:])) <= out[1] + 1
                assert items <= rules.c_items(sum(tiles), Hk, D)
    assert rules.c_items(10, 8, 128) == 10 + rules.c_resident(128) // 8 + 1
