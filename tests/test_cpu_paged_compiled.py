"""The operators of rotary.py and paged.py under torch.compile with symbolic sizes: one graph serves any number of tokens."""
import pytest
import torch

from self_trainable_or_free_attn_amd import append_paged, norm_rotate, paged_attention, paged_cache, paged_rows

BF = torch.bfloat16
COUNTS = (5, 17, 40, 96, 130, 1000)


def _t(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


def _i(*shape):
    return _t(*shape, dtype=torch.int32)


def _graphs(f, calls):
    """How many graphs `calls` of f take."""
    count = 0

    def backend(module, _):
        nonlocal count
        count += 1
        return module.forward

    torch._dynamo.reset()
    compiled = torch.compile(f, backend=backend, dynamic=True, fullgraph=True)
    for args in calls:
        want = f(*args)
        got = compiled(*args)
        for a, b in zip(*((x if isinstance(x, tuple) else (x,)) for x in (got, want))):
            assert a.shape == b.shape and a.dtype == b.dtype
    return count


CACHES = {bits: paged_cache(64, 2, 64, page_size=64, bits=bits, device="meta") for bits in (16, 4)}


@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_norm_rotate(positions, norm):
    table, w = _t(2000, 32, 2, dtype=torch.float32), _t(64) if norm else None

    def step(q, k, at):
        return norm_rotate(q * 2, k, w, w, table, at if positions else None)

    assert _graphs(step, [(_t(n, 4, 64), _t(n, 2, 64), _i(n)) for n in COUNTS]) == 1


def test_norm_rotate_of_batches():
    table, w = _t(2000, 32, 2, dtype=torch.float32), _t(64)

    def step(q, k):
        return norm_rotate(q * 2, k, w, w, table)

    # (batches of other sizes than the heads: torch takes equal sizes of a first call for one symbol)
    assert _graphs(step, [(_t(b, n, 4, 64), _t(b, n, 2, 64)) for n, b in zip(COUNTS, (7, 3, 6, 9, 11, 8))]) == 1


def test_norm_rotate_with_gradients():
    """Forward and backward traced together."""
    table, w = _t(2000, 32, 2, dtype=torch.float32), _t(64).requires_grad_()
    from functorch.compile import make_boxed_func
    from torch._dynamo.backends.common import aot_autograd
    count = 0

    def counted(module, _):
        nonlocal count
        count += 1
        return make_boxed_func(module.forward)

    def step(q, k):
        return norm_rotate(q * 2, k, w, w, table)

    torch._dynamo.reset()
    compiled = torch.compile(step, backend=aot_autograd(fw_compiler=counted, bw_compiler=counted), dynamic=True, fullgraph=True)
    for n in COUNTS:
        q, k = _t(n, 4, 64).requires_grad_(), _t(n, 2, 64).requires_grad_()
        out = compiled(q, k)
        grads = torch.autograd.grad(out, (q, k, w), [torch.empty_like(x) for x in out])
        assert [g.shape for g in grads] == [q.shape, k.shape, w.shape]
    assert count == 2


@pytest.mark.parametrize("bits", [16, 4])
def test_caches(bits):
    cache, pages, lens, cu = CACHES[bits], _i(3, 20), _i(3), _i(4)

    def attend(q):
        return paged_attention(q, cache, pages, lens, cu)

    def append(q, k):
        return append_paged(cache, k, k, pages, lens, cu, q=q)

    def rows(x):
        return paged_rows(cache, pages, lens, cu, rows=x.shape[0])

    assert _graphs(attend, [(_t(n, 4, 64),) for n in COUNTS]) == 1
    assert _graphs(append, [(_t(n, 4, 64), _t(n, 2, 64)) for n in COUNTS]) == 1
    assert _graphs(rows, [(_t(n),) for n in COUNTS]) == 1
