"""What the operators of rotary.py and paged.py refuse of GPU tensors: the calls of test_cpu_paged.py, which the native operators
check by themselves, raise the same errors."""
import pytest
import torch

import test_cpu_paged as cases
from self_trainable_or_free_attn_amd import PagedCache, append_paged, norm_rotate, paged_attention, paged_cache, paged_rows, rotary_table

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _on(dev, x):
    """The tensor (cache) with the same layout on the GPU."""
    if isinstance(x, PagedCache):
        return PagedCache(*(_on(dev, t) for t in x))
    if not isinstance(x, torch.Tensor):
        return x
    size = 1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride())) if x.numel() else 0
    return torch.zeros(size, dtype=x.dtype, device=dev).as_strided(x.shape, x.stride())


@pytest.mark.parametrize("kw, error", cases.ROTATE_REFUSED)
def test_norm_rotate_refuses(dev, kw, error):
    kw = {n: _on(dev, x) for n, x in kw.items()}
    q = kw.pop("q", None)
    k = kw.pop("k", None)
    with pytest.raises(error):
        norm_rotate(torch.zeros(6, 4, 64, dtype=BF, device=dev) if q is None else q,
                    torch.zeros(6, 2, 64, dtype=BF, device=dev) if k is None else k, kw.pop("qw", None), kw.pop("kw", None),
                    kw.pop("table", None), kw.pop("positions", None), **kw)


def _places(dev, kw):
    return (kw.pop("pages", torch.zeros(3, 4, dtype=torch.int32, device=dev)),
            kw.pop("lens", torch.zeros(3, dtype=torch.int32, device=dev)), kw.pop("cu", None))


@pytest.mark.parametrize("kw, error", cases.APPEND_REFUSED)
def test_append_paged_refuses(dev, kw, error):
    kw = {n: _on(dev, x) for n, x in kw.items()}
    cache = kw.pop("cache", None) or paged_cache(8, 2, 64, page_size=16, device=dev)
    k = kw.pop("k", torch.zeros(6, 2, 64, dtype=BF, device=dev))
    v = kw.pop("v", torch.zeros_like(k))
    with pytest.raises(error):
        append_paged(cache, k, v, *_places(dev, kw), **kw)


@pytest.mark.parametrize("kw, error", cases.ATTEND_REFUSED)
def test_paged_attention_refuses(dev, kw, error):
    kw = {n: _on(dev, x) for n, x in kw.items()}
    cache = kw.pop("cache", None) or paged_cache(8, 2, 64, page_size=16, device=dev)
    q = kw.pop("q", torch.zeros(6, 4, 64, dtype=BF, device=dev))
    with pytest.raises(error):
        paged_attention(q, cache, *_places(dev, kw), **kw)


def test_derivatives_that_do_not_exist(dev):
    cache = paged_cache(8, 2, 64, page_size=16, device=dev)
    pages, lens = torch.zeros(3, 4, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    x = torch.zeros(3, 2, 64, dtype=BF, device=dev, requires_grad=True)
    for call in (lambda: append_paged(cache, x, x, pages, lens), lambda: paged_attention(x, cache, pages, lens)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()
    import torch.autograd.forward_ad as fw
    w = torch.ones(64, dtype=BF, device=dev)
    with fw.dual_level():
        d = fw.make_dual(x.detach(), torch.zeros_like(x))
        for call in (lambda: append_paged(cache, d, d, pages, lens), lambda: paged_attention(d, cache, pages, lens),
                     lambda: norm_rotate(d, d, w, w)):
            with pytest.raises(RuntimeError, match="derivative"):
                call()


def test_tensors_of_the_host_are_refused(dev):
    x = torch.zeros(3, 2, 64, dtype=BF, device=dev)
    pages, lens = torch.zeros(3, 4, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    cache = paged_cache(8, 2, 64, page_size=16, device=dev)
    for call in (lambda: append_paged(cache, x, x, pages.cpu(), lens), lambda: append_paged(cache, x, x.cpu(), pages, lens),
                 lambda: append_paged(paged_cache(8, 2, 64, page_size=16, device="cpu"), x, x, pages, lens),
                 lambda: paged_attention(x, cache, pages, lens.cpu()), lambda: paged_rows(cache, pages.cpu(), lens, rows=3),
                 lambda: norm_rotate(x, x, table=rotary_table(3, 64)), lambda: norm_rotate(x, x.cpu(), table=rotary_table(3, 64, device=dev))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kw, error", [
    (dict(rows=-1), ValueError), (dict(rows=1 << 30), ValueError), (dict(rows=4), ValueError), (dict(dtype=torch.float32), TypeError),
    (dict(dtype=torch.float16), TypeError), (dict(pages=torch.long), TypeError), (dict(lens=4), ValueError), (dict(cu=3), ValueError),
    (dict(bits=4, dtype=torch.float32), TypeError), (dict(bits=4, rows=4), ValueError), (dict(cut="k_scales"), ValueError),
    (dict(cut="k"), ValueError),
])
def test_paged_rows_refuses(dev, kw, error):
    cache = paged_cache(8, 2, 64, page_size=16, bits=4 if "cut" in kw else kw.get("bits", 16), device=dev)
    if "cut" in kw:
        cache = cache._replace(**{kw["cut"]: getattr(cache, kw["cut"])[..., :1].contiguous()})
    pages = torch.zeros(3, 4, dtype=kw.get("pages", torch.int32), device=dev)
    lens = torch.ones(kw.get("lens", 3), dtype=torch.int32, device=dev)
    cu = torch.zeros(kw["cu"], dtype=torch.int32, device=dev) if "cu" in kw else None
    with pytest.raises(error):
        paged_rows(cache, pages, lens, cu, rows=kw.get("rows", 3), dtype=kw.get("dtype"))
