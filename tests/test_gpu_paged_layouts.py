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
