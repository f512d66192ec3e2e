"""The tile that a share of single tokens begins in (csrc/paged_rules.h compiled alone for the host): always one of the sequence's."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = '#include "paged_rules.h"\nextern "C" int c_place(int y, int cost, int tiles) { return es::place_in(y, cost, tiles); }\n'


@pytest.fixture(scope="module")
def place(tmp_path_factory):
    d = tmp_path_factory.mktemp("places")
    (d / "places.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "self_trainable_or_free_attn_amd", "csrc"),
                    str(d / "places.cpp"), "-o", str(d / "places.so")], check=True)
    return ctypes.CDLL(str(d / "places.so")).c_place


def test_within_the_sequence(place):
    for tiles in (1, 2, 7):
        for cost in (1, 5, 80):
            for y in range(tiles * cost):
                assert place(y, cost, tiles) == y // cost


@pytest.mark.parametrize("y", [-1, -100, -2 ** 31, 2 ** 31 - 1, 10 ** 6])
@pytest.mark.parametrize("tiles", [0, 1, 3])
def test_costs_that_wrapped(place, y, tiles):
    """As decreasing counts can make them: no place before the first tile or behind the last."""
    got = place(y, 3, tiles)
    assert 0 <= got <= max(tiles - 1, 0)
