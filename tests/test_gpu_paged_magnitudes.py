"""Keys of any finite bf16 magnitude on their way into a cache of 4 bits: their norm is taken in 64 bits, so squares that float32
does not hold count as they are (paged_ref.py)."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R, halves", [(0, False), (1, False), (1, True), (0.5, True), (0.5, False)])
@pytest.mark.parametrize("scale, eps", [(2.0 ** 84, 1e-6), (2.0 ** 126, 1e-6), (2.0 ** 64, 0.0), (2.0 ** -84, 0.0), (2.0 ** -120, 0.0),
                                        (2.0 ** -70, 1e-30)])
def test_squares_that_float32_does_not_hold(dev, D, R, halves, scale, eps):
    import self_trainable_or_free_attn_amd as api
    g = torch.Generator(device=dev).manual_seed(1)
    lens, Hk, page = [40, 1, 23], 3, 16
    T, R = sum(lens), int(R * D)
    k, v = torch.randn(2, T, Hk, D, device=dev, generator=g).to(BF)
    k = torch.where(torch.rand(T, Hk, 1, device=dev, generator=g) < 0.8, k * scale, k)     # (some of ordinary size beside them)
    k[3, 0, 5] = scale                                                                     # (one large value, or one small one)
    k = k.clamp(-3e38, 3e38)
    w = (1 + 0.3 * torch.randn(D, device=dev, generator=g)).to(BF)
    table = api.rotary_table(max(lens), R, device=dev) if R else None
    pages, num = ref.page_table(lens, page, 1, dev, 1)
    cache = api.paged_cache(num, Hk, D, page_size=page, bits=4, device=dev)
    total = torch.tensor(lens, dtype=torch.int32, device=dev)
    cu = torch.tensor(ref.starts(lens), dtype=torch.int32, device=dev)
    api.append_paged(cache, k, v, pages, total, cu, k_weight=w, table=table, eps=eps, halves=halves)
    pos = torch.cat([torch.arange(n, device=dev) for n in lens])
    cs = table[pos] if R else torch.zeros(T, 0, 2, device=dev)
    want, e = ref.held4(ref.rotate(k, w, cs, eps, halves)["y"][0].float(), BF)
    assert bool(want.abs().amax(-1).gt(0).all())
    number = torch.cat([pages[b].long()[torch.arange(n, device=dev) // page] for b, n in enumerate(lens)])
    codes, scales = cache.k[number, :, pos % page], cache.k_scales[number, :, pos % page]
    assert torch.equal(scales.long() - 127, e.long())
    assert torch.equal(ref.decode4(codes, scales), want)
