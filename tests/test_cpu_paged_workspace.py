"""The workspace of attention over paged caches: as large as the pieces that a call can cut, whatever its tokens and sequences, and
the numbers of those pieces (csrc/paged_rules.h compiled alone for the host)."""
import ctypes
import os
import random
import subprocess

import pytest

import test_cpu_paged_rules as rules_cases
from self_trainable_or_free_attn_amd import _lib

SHIM = rules_cases.SHIM + r"""
extern "C" int c_partial(int i, int level0, int cuts) { return partial_number(i, level0, cuts); }
extern "C" long long c_most(long long tiles, long long later) { return most_partials(tiles, later); }
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("partials")
    src, lib = d / "partials.cpp", d / "partials.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I",
                    os.path.join(rules_cases.ROOT, "self_trainable_or_free_attn_amd", "csrc"), str(src), "-o", str(lib)], check=True)
    so = ctypes.CDLL(str(lib))
    so.c_most.argtypes, so.c_most.restype = [ctypes.c_longlong] * 2, ctypes.c_longlong
    return so


def _most(Hk, D):
    """Twice the pieces that fill the GPU (256 CUs with two or three workgroups each) and one, of 128 rows of float32 with maximum
    and sum."""
    return 2 * ((768 if D == 64 else 512) // Hk + 1) * Hk * 128 * (D + 2) * 4


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("B, T, keys, H, Hk, D", [
    (1, 75600, 75600, 40, 8, 128), (1, 131072, 131072, 64, 8, 128), (1024, 2048, 8192, 32, 8, 128), (1, 32760, 32760, 24, 8, 64),
    (600, 1200, 4096, 16, 4, 128), (3, 900, 2048, 8, 1, 64), (5, 60000, 1 << 20, 40, 40, 128), (2, 4000, 5000, 600, 600, 64),
])
def test_does_not_grow_with_tokens_and_sequences(bits, B, T, keys, H, Hk, D):
    got = _lib.lib().es_paged_workspace(B, T, -(-keys // 64), 64, H, Hk, D, bits)
    assert 0 < got <= _most(Hk, D) + 8 * (B + 2)


def test_small_calls_take_no_more_than_their_tiles_can_be_cut_into():
    got = _lib.lib().es_paged_workspace(1, 100, 64, 64, 2, 2, 128, 16)
    assert got <= ((100 // 128 + 2) + 512 // 2 + 1) * 2 * 128 * 130 * 4 + 8 * 3


def test_random_shapes():
    rng = random.Random(3)
    log = lambda hi: int(2 ** rng.uniform(0, hi))
    for _ in range(500):
        B, Hk, D, page = log(10), rng.choice([1, 2, 3, 5, 8, 40]), rng.choice([64, 128]), 16 << rng.randrange(5)
        T, H, width = B * log(8), Hk * log(4), log(20 - page.bit_length())
        got = _lib.lib().es_paged_workspace(B, T, width, page, H, Hk, D, rng.choice([16, 4]))
        assert got <= _most(Hk, D) + 16 * (B + 770), (B, T, width, page, H, Hk, D)


@pytest.mark.parametrize("case", list(rules_cases._lists())[:200])
def test_partials_of_cut_tiles_are_numbered_without_gaps(rules, case):
    n, length, held, group, causal, per = case
    x = (ctypes.c_int * 5)()
    rules.c_list(n * group, n, length, held, group, causal, x)
    piece = rules.c_piece(x, per)
    tiles = rules_cases._chunks(n, length, held, group, causal)
    later = rules.c_later(x, group, causal, piece)
    cuts = sum(w > piece for w in tiles)
    if later > 5000:
        pytest.skip("more pieces than are worth a walk")
    assert cuts <= later and cuts + later <= rules.c_most(len(tiles), later)
    out = (ctypes.c_int * 2)()
    for above in {-1, per * 3 // 4}:
        level0 = sum(w > above for w in tiles)
        seen = []
        for i in range(level0 + later):
            assert rules.c_at(x, group, causal, piece, above, i, out)
            tile, level = out[0], out[1]
            if tiles[tile] <= piece:
                continue
            number = rules.c_partial(i, level0, cuts)
            assert number == rules.c_number(x, group, causal, piece, piece, tile, level)
            seen.append(number)
        assert sorted(seen) == list(range(cuts + later))
