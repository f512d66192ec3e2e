"""Attention over paged caches of up to 1024 keys a sequence on grids that fill the GPU: whole tiles of 128 rows, without pieces.
(test_gpu_paged_attention.py has the smaller grids, whose tiles have 64 rows or fewer, and the longer tables.)"""
import pytest

import test_gpu_paged_attention as attention
from self_trainable_or_free_attn_amd import _lib

pytestmark = pytest.mark.gpu


def _case(dev, lens, keys, H, Hk, D, dtype, page, bits, seed, **kw):
    """The call takes this form by its sizes: no workspace, and more tiles of 128 rows than fill the GPU once."""
    B, T = len(lens), sum(lens) + kw.get("pad", 0)
    width = kw.get("width") or max(-(-m // page) for m in keys)
    assert width * page <= 1024 and _lib.lib().es_paged_workspace(B, T, width, page, H, Hk, D, bits) == 0
    assert T > B and (T * (H // Hk) // 128 + B + 1) * Hk > 768
    attention._case(dev, lens, keys, H, Hk, D, dtype, page, bits, seed, **kw)


@pytest.mark.parametrize("D, dtype", attention.TYPES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("causal", [True, False])
def test_many_heads(dev, D, dtype, bits, causal):
    _case(dev, [300, 1, 70, 0, 129], [300, 1, 200, 5, 1024], 128, 128, D, dtype, 64, bits, seed=1, causal=causal, pad=2)


@pytest.mark.parametrize("D, dtype", attention.TYPES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_of_grouped_heads(dev, D, dtype, bits, causal):
    """More keys than new tokens and fewer, tiles that end inside a token's heads, a missing page."""
    _case(dev, [700, 333, 1, 90, 40], [700, 1000, 900, 31, 0], 72, 24, D, dtype, 16, bits, seed=2, causal=causal, pad=1,
          holes=((0, 3), (1, 62), (2, 0)))


@pytest.mark.parametrize("D, dtype", attention.TYPES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("B", [63, 64, 90])
def test_many_sequences(dev, D, dtype, bits, B):
    """Up to 63 in order of their keys, more of them in their own."""
    lens = [(7 * i) % 5 if i % 20 else 140 for i in range(B)]
    keys = [n + (61 * i) % 800 if i % 9 else n // 2 for i, n in enumerate(lens)]
    _case(dev, lens, keys, 32, 16, D, dtype, 32, bits, seed=3, pad=B % 3, width=32)


@pytest.mark.parametrize("bits", [16, 4])
def test_equal_counts(dev, bits):
    _case(dev, [130] * 8, [130, 1000, 64, 1024, 129, 131, 0, 500], 64, 64, 64, attention.FP, 128, bits, seed=4, cu=False)
