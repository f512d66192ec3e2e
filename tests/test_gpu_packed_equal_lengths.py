"""Batches of equal sequences without running lengths: whether keys are cut into ranges follows from the length of one."""
import math

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D, dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("B, n, m", [(8, 1, 600), (5, 130, 600), (4, 1, 3000), (3, 40, 2500)])
def test_equal_sequences(dev, D, dtype, B, n, m):
    import self_trainable_or_free_attn_amd as api
    from self_trainable_or_free_attn_amd import _lib
    H, Hk = 8, 2
    g = torch.Generator(device=dev).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(dtype)
    q, k, v = rnd(B, n, H, D), rnd(B, m, Hk, D), rnd(B, m, Hk, D)
    want = ref.packed(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), [n] * B, [m] * B, True, 1 / math.sqrt(D))
    out, lse = api.packed_attention(q, k, v, causal=True, return_lse=True)
    ref.check("out", out.flatten(0, 1), *want["out"])
    ref.check("lse", lse.flatten(0, 1), *want["lse"])
    if m > 1024:
        return
    # short ones are not cut: such a call needs no workspace, though one of the same sizes with running lengths may
    out, lse = torch.empty(B * n, H, D, device=dev, dtype=dtype), torch.empty(B * n, H, device=dev)
    _lib.call("es_packed_fwd" + ("_f16" if dtype is torch.float16 else ""), q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), None,
              None, None, None, 0, 0, out, lse, None, 0, B, B * n, B * m, H, Hk, D, 1, 1 / math.sqrt(D))
    ref.check("out", out, *want["out"])
    ref.check("lse", lse, *want["lse"])
