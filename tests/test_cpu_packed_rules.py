"""Which calls of packed_attention cut their keys into ranges (seen by their workspace)."""
import pytest

from self_trainable_or_free_attn_amd import _lib


def _ranged(lens, keys, H, Hk, D):
    return _lib.lib().es_packed_fwd_workspace(len(lens), sum(lens), sum(keys), H, Hk, D) > 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, n, H, Hk", [(8, 512, 4, 4), (8, 512, 2, 2), (8, 512, 1, 1), (8, 512, 8, 8), (100, 64, 1, 1), (16, 256, 4, 4),
                                         (16, 256, 1, 1), (4, 1024, 4, 4), (50, 128, 2, 1)])
def test_batches_of_short_sequences_take_whole_tiles(D, B, n, H, Hk):
    """Sequences of up to 16 chunks of keys gain nothing from ranges, however many there are."""
    assert not _ranged([n] * B, [n] * B, H, Hk, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, m", [(32, 40), (32, 128), (8, 128), (8, 300), (4, 300), (2, 520), (64, 128), (64, 256), (128, 40)])
@pytest.mark.parametrize("H, Hk", [(8, 2), (32, 8)])
def test_tokens_over_short_caches_take_whole_tiles(D, B, m, H, Hk):
    assert not _ranged([1] * B, [m] * B, H, Hk, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens, keys, H, Hk", [
    ([1], [1100], 8, 2), ([1] * 8, [32760, 4097, 75600, 1209, 16384, 20011, 513, 9000], 40, 8), ([1] * 32, [8000] + [40] * 31, 8, 2),
    ([1] * 8, [4000] + [100] * 7, 32, 8), ([8000] + [64] * 7, None, 1, 1), ([6000] + [500] * 4, None, 2, 1), ([2000], None, 2, 1),
    ([64] * 4, [4000, 100, 100, 100], 8, 8), ([256, 512, 31, 1], [9000, 512, 4111, 2600], 24, 24)])
def test_long_sequences_are_cut(D, lens, keys, H, Hk):
    assert _ranged(lens, keys or lens, H, Hk, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, n, m", [(4, 64, 500), (2, 200, 900)])
def test_tokens_behind_short_histories_take_whole_tiles(D, B, n, m):
    assert not _ranged([n] * B, [m] * B, 8, 8, D)
