"""Gradients of packed_attention where the kernels sum delta themselves (rows of up to 512 keys, and every row with a bias), with
bounds that leave no room for the rounding of the output (packed_delta_ref.py)."""
import pytest
import torch

import packed_delta_ref as ref
import packed_ref

pytestmark = pytest.mark.gpu

TYPES = [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float16), (128, torch.float16)]


def _check(dev, q, k, v, do, bias, table, causal):
    import self_trainable_or_free_attn_amd as api
    (n, H, D), (m, Hk), dtype = q.shape, k.shape[:2], q.dtype
    leaves = [x.to(dev).requires_grad_() for x in (q, k, v, bias) if x is not None]
    do = do.to(dev)
    out = api.packed_attention(*leaves[:3], causal=causal, bias=leaves[3] if bias is not None else None, buckets=table)
    got = torch.autograd.grad(out, leaves, do)
    i, j = torch.arange(n, device=dev)[:, None] + m - n, torch.arange(m, device=dev)[None]
    seen = j <= i if causal else torch.ones(n, m, dtype=torch.bool, device=dev)
    if bias is not None:
        at = table.long()[(j - i).clamp(-(table.numel() // 2), table.numel() // 2) + table.numel() // 2]
    G = H // Hk
    q, k, v = (x.detach().double() for x in leaves[:3])
    for h in range(Hk):
        hs = slice(h * G, h * G + G)
        extra = leaves[3].detach()[:, hs].double().t()[:, at] if bias is not None else None
        w = ref.attention(q[:, hs].transpose(0, 1), k[:, h], v[:, h], do[:, hs].double().transpose(0, 1), seen, D ** -0.5, extra, dtype)
        packed_ref.check(f"dq of kv head {h}", got[0][:, hs].transpose(0, 1), *w["dq"])
        packed_ref.check(f"dk of kv head {h}", got[1][:, h], *w["dk"])
        if bias is not None:
            packed_ref.check(f"dbias of kv head {h}", got[3][:, hs], *ref.by_bucket(w["ds"], at, bias.shape[0]))


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("n, m, H, Hk, bias", [(512, 512, 2, 2, True), (1300, 1300, 1, 1, True), (300, 900, 4, 2, True), (70, 512, 6, 2, False),
                                               (512, 200, 2, 2, False), (3, 2, 2, 1, False)])
@pytest.mark.parametrize("causal", [False, True])
def test_delta_of_its_own(dev, D, dtype, n, m, H, Hk, bias, causal):
    import self_trainable_or_free_attn_amd as api
    g = torch.Generator().manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g)
    q, k, v, do = (1.5 * rnd(n, H, D)).to(dtype), rnd(m, Hk, D).to(dtype), rnd(m, Hk, D).to(dtype), rnd(n, H, D).to(dtype)
    table = api.relative_buckets(16, 60, device=dev) if bias else None
    _check(dev, q, k, v, do, rnd(16, H) if bias else None, table, causal)


@pytest.mark.parametrize("D, dtype", TYPES)
@pytest.mark.parametrize("n, m, H, Hk", [(400, 400, 2, 2), (400, 400, 4, 2), (130, 1400, 2, 1)])
def test_delta_is_not_taken_from_the_output(dev, D, dtype, n, m, H, Hk):
    """Bounds of dbias that delta from the stored output exceeds (shown in test_cpu_packed_delta.py)."""
    table = torch.arange(15, dtype=torch.int32, device=dev)
    _check(dev, *ref.telling_inputs(n, m, H, Hk, D, dtype), torch.zeros(15, H), table, False)
