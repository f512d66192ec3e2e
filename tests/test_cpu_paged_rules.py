"""How attention over paged caches cuts wide launches, as the kernels derive it: csrc/paged_rules.h compiled alone for the host."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = r"""
#include "paged_rules.h"
using namespace es;
extern "C" {
void c_list(int rows, int nq, int len, int held, int group, int causal, int* out) {
  const WideList x = wide_list(rows, nq, len, held, ((rows < 128 ? rows : 128) - 1) / group + 1, causal);
  out[0] = x.rows, out[1] = x.tiles, out[2] = x.chunks, out[3] = x.behind, out[4] = x.first;
}
WideList list(const int* x) { return WideList{x[0], x[1], x[2], x[3], x[4]}; }
int c_within(const int* x, int group, int causal, int c) { return tiles_within(list(x), group, causal, c); }
int c_piece(const int* x, int per) { return piece_of(list(x), per); }
int c_pieces(int chunks, int piece) { return pieces_of(chunks, piece); }
int c_later(const int* x, int group, int causal, int piece) { return later_pieces(list(x), group, causal, piece); }
int c_at(const int* x, int group, int causal, int piece, int above, int i, int* out) {
  return piece_at(list(x), group, causal, piece, above, i, out[0], out[1]);
}
int c_number(const int* x, int group, int causal, int piece, int above, int tile, int level) {
  return piece_number(list(x), group, causal, piece, above, tile, level);
}
float c_time(float big, float size, float small, float mean, int cut, float start, float inv) {
  return wide_time(big, size, small, mean, cut, start, inv);
}
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    src, lib = d / "rules.cpp", d / "rules.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-shared", "-fPIC",
                    "-I", os.path.join(ROOT, "self_trainable_or_free_attn_amd", "csrc"), str(src), "-o", str(lib)], check=True)
    so = ctypes.CDLL(str(lib))
    f = ctypes.c_float
    so.c_time.argtypes, so.c_time.restype = [f, f, f, f, ctypes.c_int, f, f], f
    return so


def _chunks(n, length, held, group, causal):
    """Chunks that each tile of a list reads, row by row."""
    out = []
    for r0 in range(0, n * group, 128):
        last = (min(n * group, r0 + 128) - 1) // group
        seen = min(max(last + 1 - n + length, 0), held) if causal else held
        out.append(-(-seen // 64))
    return out


def _lists():
    rng = random.Random(7)
    log = lambda hi: int(2 ** rng.uniform(0, hi))
    for i in range(400):
        group = rng.choice([1, 1, 2, 3, 4, 5, 8, 16, 33, 128, 300])
        n = rng.choice([0, 1, 2, log(6), log(12), log(12)])
        length = rng.choice([0, n, n, n + 1, max(n - log(8), 0), n + log(14), log(14)])
        held = rng.choice([length, length, length, min(length, 16 * log(8)), 0])
        yield n, length, held, group, rng.random() < 0.8, rng.choice([4, 8, log(4) + 3, log(8) + 3])
    yield 5, 2 ** 31 - 1, 2 ** 30 - 16, 4, True, 1 << 16
    yield 1, 2 ** 30 - 16, 2 ** 30 - 16, 4096, True, 1 << 15
    yield 70000, 2 ** 31 - 1, 4096, 2, True, 8


@pytest.mark.parametrize("case", list(_lists()))
def test_pieces_cover_every_tile_once(rules, case):
    n, length, held, group, causal, per = case
    x = (ctypes.c_int * 5)()
    rules.c_list(n * group, n, length, held, group, causal, x)
    want = _chunks(n, length, held, group, causal)
    assert x[1] == len(want) and x[2] == (-(-held // 64))
    for c in {-1, 0, 1, 2, per - 1, per, per + 1, 2 * per, x[2] // 2, x[2] - 1, x[2], x[2] + 1}:
        assert rules.c_within(x, group, causal, c) == sum(w <= c for w in want), c
    if want:
        assert abs(x[4] - want[0]) <= 1 or x[4] >= want[0]
    piece = rules.c_piece(x, per)
    assert piece == max(per, 4 if n * group <= 32 else 8)
    pieces = [rules.c_pieces(w, piece) for w in want]
    assert all(p == max(1, -(-w // piece)) for p, w in zip(pieces, want))
    assert rules.c_later(x, group, causal, piece) == sum(pieces) - len(pieces)
    out = (ctypes.c_int * 2)()
    for above in {-1, 0, piece * 3 // 4}:
        items = {(t, 0) for t, w in enumerate(want) if w > above} | {(t, i) for t, p in enumerate(pieces) for i in range(1, p)}
        if len(items) > 5000:
            continue
        for i in range(len(items)):
            assert rules.c_at(x, group, causal, piece, above, i, out)
            at = (out[0], out[1])
            assert at in items, (i, at)
            items.remove(at)
            assert rules.c_number(x, group, causal, piece, above, *at) == i
        assert not items


def test_time(rules):
    time = lambda big, size, small, mean, cut: rules.c_time(big, size, small, mean, cut, 3.0, 1 / 64)
    assert time(64, 16, 0, 16, 0) == 19
    assert time(64, 16, 0, 16, 1) == 22
    assert time(65, 16, 0, 16, 0) == 38
    assert time(60, 16, 70, 16, 0) == 19                  # small ones in the four places that are left
    assert time(64, 16, 64, 16, 0) == 19 + 1 + 4          # behind the big ones
    assert time(0, 16, 128, 16, 0) == 2 + 4
    assert time(64, 16, 0, 6, 0) == pytest.approx(19 - 3.8)
