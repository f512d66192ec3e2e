"""Layouts of paged caches that the operators of paged.py take and refuse, packed tokens (which the native operators check) and
batches (which Python checks first) alike."""
import pytest
import torch

import test_cpu_paged_layouts as cases
from self_trainable_or_free_attn_amd import PagedCache, append_paged, paged_attention, paged_rows

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("shape, strides", cases.ONES)
def test_dimensions_of_one_have_any_stride(dev, shape, strides):
    """Packed and as a batch, into a cache of this layout and into a contiguous one: the same bits."""
    num, Hk, page, D = shape
    g = torch.Generator(device=dev).manual_seed(1)
    odd = PagedCache(*(cases.strided(shape, strides, dev) for _ in "kv"))
    plain = PagedCache(*(torch.zeros(shape, dtype=BF, device=dev) for _ in "kv"))
    pages, lens = torch.tensor([[num - 1]], dtype=torch.int32, device=dev), torch.tensor([9], dtype=torch.int32, device=dev)
    q, k, v = (torch.randn(9, h, D, device=dev, generator=g).to(BF) for h in (2 * Hk, Hk, Hk))
    res = []
    for cache in (odd, plain):
        for flat in (lambda x: x, lambda x: x[None]):
            new = append_paged(cache, flat(k), flat(v), pages, lens, q=flat(q))
            res.append((new.flatten(0, -3), paged_attention(new, cache, pages, lens).flatten(0, -3),
                        *paged_rows(cache, pages, lens, rows=9), cache.k.clone(), cache.v.clone()))
    for other in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], other))
    assert torch.equal(odd.k[num - 1].transpose(0, 1)[:9], k) and torch.equal(odd.v[num - 1].transpose(0, 1)[:9], v)


@pytest.mark.parametrize("shape, strides", cases.OVERLAPPING)
def test_rows_that_overlap_are_refused(dev, shape, strides):
    cache = PagedCache(*(cases.strided(shape, strides, dev) for _ in "kv"))
    pages, lens = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    x = torch.zeros(2, shape[1], shape[3], dtype=BF, device=dev)
    for call in (lambda: append_paged(cache, x, x, pages, lens), lambda: paged_attention(x, cache, pages, lens),
                 lambda: paged_rows(cache, pages, lens, rows=2)):
        with pytest.raises(ValueError, match="overlap"):
            call()


@pytest.mark.parametrize("shape, strides", cases.APART)
def test_rows_apart_in_any_order(dev, shape, strides):
    num, Hk, page, D = shape
    g = torch.Generator(device=dev).manual_seed(2)
    odd = PagedCache(*(cases.strided(shape, strides, dev) for _ in "kv"))
    n = num * page - 3
    pages, lens = torch.randperm(num, device=dev, generator=g).to(torch.int32)[None], torch.tensor([n], dtype=torch.int32, device=dev)
    k, v = torch.randn(2, n, Hk, D, device=dev, generator=g).to(BF)
    append_paged(odd, k, v, pages, lens)
    rows = paged_rows(odd, pages, lens, rows=n)
    assert torch.equal(rows[0], k) and torch.equal(rows[1], v)


@pytest.mark.parametrize("scale", [None, 0.1])
def test_heads_without_channels_are_refused(dev, scale):
    cache = PagedCache(*(torch.zeros(8, 2, 16, 64, dtype=BF, device=dev) for _ in "kv"))
    pages, lens = torch.zeros(2, 3, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="head dim"):
        paged_attention(torch.zeros(2, 2, 0, dtype=BF, device=dev), cache, pages, lens, scale=scale)
