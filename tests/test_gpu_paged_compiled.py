"""The operators of rotary.py and paged.py traced by torch.compile: the same bits as called directly, gradients included, and one
graph for any number of tokens."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _counted(count):
    from functorch.compile import make_boxed_func
    from torch._dynamo.backends.common import aot_autograd

    def counted(module, _):
        count.append(1)
        return make_boxed_func(module.forward)

    return aot_autograd(fw_compiler=counted, bw_compiler=counted)


def test_norm_rotate(dev):
    import self_trainable_or_free_attn_amd as api
    g = torch.Generator(device=dev).manual_seed(1)
    table = api.rotary_table(300, 64, device=dev)
    w = [(1 + 0.2 * torch.randn(64, device=dev, generator=g)).requires_grad_() for _ in "qk"]

    def step(q, k):
        return api.norm_rotate(q * 2, k, *w, table, halves=True)

    torch._dynamo.reset()
    count = []
    compiled = torch.compile(step, backend=_counted(count), dynamic=True)
    for n in (5, 33, 128, 300):
        q, k = (torch.randn(n, h, 64, device=dev, generator=g).to(BF).requires_grad_() for h in (6, 2))
        got, want = compiled(q, k), step(q, k)
        d = [torch.randn_like(x) for x in want]
        for a, b in zip((*got, *torch.autograd.grad(got, (q, k, *w), d)), (*want, *torch.autograd.grad(want, (q, k, *w), d))):
            assert torch.equal(a, b)
    assert len(count) == 2


@pytest.mark.parametrize("bits", [16, 4])
def test_a_layer(dev, bits):
    """Append, attention and the rows back, traced together."""
    import self_trainable_or_free_attn_amd as api
    g = torch.Generator(device=dev).manual_seed(2)
    page, Hk, H, D = 16, 2, 6, 64
    pages, num = ref.page_table([400] * 3, page, 1, dev, 2)
    caches = [api.paged_cache(num, Hk, D, page_size=page, bits=bits, device=dev) for _ in "ab"]
    table = api.rotary_table(400, D, device=dev)

    def step(cache, x, lens, cu):
        q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
        q = api.append_paged(cache, k, v, pages, lens, cu, q=q, table=table)
        return (*api.paged_attention(q, cache, pages, lens, cu, return_lse=True), *api.paged_rows(cache, pages, lens, cu,
                                                                                                  rows=x.shape[0]))

    torch._dynamo.reset()
    count = []
    compiled = torch.compile(step, backend=_counted(count), dynamic=True)
    lens = torch.zeros(3, dtype=torch.int32, device=dev)
    for new in ([40, 3, 70], [1, 1, 1], [100, 0, 33], [5, 250, 17]):
        lens = lens + torch.tensor(new, dtype=torch.int32, device=dev)
        cu = torch.tensor(ref.starts(new), dtype=torch.int32, device=dev)
        x = torch.randn(sum(new), H + 2 * Hk, D, device=dev, generator=g).to(BF)
        with torch.no_grad():
            got, want = (f(c, x, lens, cu) for f, c in zip((compiled, step), caches))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(*caches):
        assert a is None or torch.equal(a, b)
