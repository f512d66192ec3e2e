"""The chunks that the first tile of a list reads, by which the work of wide launches is estimated (csrc/paged_rules.h)."""
import ctypes

import pytest

import test_cpu_paged_rules as cases
from test_cpu_paged_rules import rules  # noqa: F401  (the library of the rules)


@pytest.mark.parametrize("case", list(cases._lists()))
def test_first_tile_counts_as_what_it_reads(rules, case):  # noqa: F811
    """Neither as nothing nor as all keys: at most one chunk more than it reads, and no more than the last tile."""
    n, length, held, group, causal, _ = case
    x = (ctypes.c_int * 5)()
    rules.c_list(n * group, n, length, held, group, causal, x)
    want = cases._chunks(n, length, held, group, causal)
    if want:
        assert want[0] <= x[4] <= want[0] + 1 and x[4] <= x[2]
    if want and not causal:
        assert x[4] == want[0] == x[2]
