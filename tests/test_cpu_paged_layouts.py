"""Layouts of paged caches that the operators of paged.py take and refuse, on meta tensors. (The tests of the same name on the GPU
make the calls whose tensors the native operators check.)"""
import pytest
import torch

from self_trainable_or_free_attn_amd import PagedCache, append_paged, paged_attention, paged_rows

BF = torch.bfloat16


def strided(shape, strides, device="meta"):
    """A tensor of these strides over as much memory as they span."""
    size = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    return torch.zeros(size, dtype=BF, device=device).as_strided(shape, strides)


def _i(*shape):
    return torch.empty(*shape, dtype=torch.int32, device="meta")


def _calls(cache, n=2):
    """All calls with one sequence, whose tokens Python checks (a batch) on meta tensors."""
    Hk, D = cache.k.shape[1], cache.k.shape[3]
    x = torch.empty(1, n, Hk, D, dtype=BF, device="meta")
    return [lambda: append_paged(cache, x, x, _i(1, 1), _i(1)), lambda: paged_attention(x, cache, _i(1, 1), _i(1)),
            lambda: paged_rows(cache, _i(1, 1), _i(1), rows=n)]


# (pages, heads, rows of a page, channels) and strides; a dimension of one may have any stride
ONES = [((1, 2, 16, 64), (3, 1024, 64, 1)), ((8, 1, 16, 64), (1024, 5, 64, 1)), ((8, 1, 16, 64), (1024, 0, 64, 1)),
        ((1, 1, 32, 128), (7, 9, 136, 1)), ((1, 3, 16, 64), (1, 64, 192, 1))]


@pytest.mark.parametrize("shape, strides", ONES)
def test_dimensions_of_one_have_any_stride(shape, strides):
    for call in _calls(PagedCache(strided(shape, strides), strided(shape, strides))):
        call()


# rows that share values, though every stride is as long as a row
OVERLAPPING = [((8, 2, 16, 64), (256, 64, 128, 1)), ((8, 2, 16, 64), (1024, 128, 64, 1)), ((2, 3, 16, 64), (64, 96, 384, 1)),
               ((4, 2, 16, 128), (4096, 2048, 64, 1)), ((3, 2, 16, 64), (2048, 1024, 0, 1))]
APART = [((8, 2, 16, 64), (2048, 64, 128, 1)), ((8, 2, 16, 64), (64, 512, 1024, 1)), ((2, 3, 16, 64), (80, 160, 480, 1)),
         ((4, 2, 16, 128), (10000, 5000, 136, 1)), ((1, 2, 16, 64), (0, 64, 128, 1))]


@pytest.mark.parametrize("shape, strides", OVERLAPPING)
def test_rows_that_overlap_are_refused(shape, strides):
    for call in _calls(PagedCache(strided(shape, strides), strided(shape, strides))):
        with pytest.raises(ValueError, match="overlap"):
            call()


@pytest.mark.parametrize("shape, strides", APART)
def test_rows_apart_in_any_order(shape, strides):
    for call in _calls(PagedCache(strided(shape, strides), strided(shape, strides))):
        call()


def test_heads_without_channels_are_refused():
    q, cache = torch.empty(2, 2, 0, dtype=BF, device="meta"), PagedCache(*(torch.empty(8, 2, 16, 64, dtype=BF, device="meta"),) * 2)
    with pytest.raises(ValueError, match="head dim"):
        paged_attention(q, cache, _i(2, 3), _i(2))


def test_the_default_scale_needs_no_channels():
    """Tensors that claim to be on a GPU, whose calls only the native operator checks: no arithmetic of Python's fails before."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        t = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device="cuda")
        out = paged_attention(t(2, 2, 0), PagedCache(t(8, 2, 16, 64), t(8, 2, 16, 64)), t(2, 3, dtype=torch.int32),
                              t(2, dtype=torch.int32))
        assert out.shape == (2, 2, 0)
