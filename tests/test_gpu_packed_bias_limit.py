"""Bias values past the limit to which packed_attention holds them (+-131072): the scores are those of the limit, so a value that
is beyond it has no gradient, one at or inside it has."""
import math

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

LIMIT = 131072.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H, Hk", [(3, 3), (6, 3)])
@pytest.mark.parametrize("low", [LIMIT, 1.5 * LIMIT, 1e9, 3.4028234663852886e38])
@pytest.mark.parametrize("sign", [-1, 1])
def test_gradient_of_values_past_the_limit(dev, dtype, H, Hk, low, sign):
    """Three buckets by distance (behind, at, ahead of the query). Head 0: all at the limit or beyond, so a row's keys share its
    weight; head 1: one bucket there; head 2: none."""
    import self_trainable_or_free_attn_amd as api
    n, D = 90, 64
    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g)
    q, k, v, do = (rnd(n, h, D).to(dtype).to(dev) for h in (H, Hk, Hk, H))
    bias = rnd(3, H)
    bias[:, 0] = sign * low
    bias[0, 1] = sign * low
    bias = bias.to(dev)
    table = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, bias)]
    out = api.packed_attention(*leaves[:3], bias=leaves[3], buckets=table)
    got = torch.autograd.grad(out, leaves, do)[3]
    past = bias.abs() > LIMIT
    assert bool(past.any()) == (low > LIMIT)
    assert not got[past].any()
    want = ref.packed(q, k, v, [n], [n], False, D ** -0.5, bias.clamp(-LIMIT, LIMIT), table, do)["dbias"]
    if low == LIMIT:
        assert float(want[0][:, 0].abs().min()) > 0.1 and bool(got[:, 0].all())
    # scores of 2^17 (189097 in log2 units) have steps of 2^-6, so a probability of such a row is off by up to 2^-7 ln 2 as in its
    # sum, and once more for the stored LSE (2^-8 natural, 2^-7 log2): 2^-5 of p, and of sum p |dp - delta| for a sum of dS
    at = table.long()[(torch.arange(n, device=dev)[None] - torch.arange(n, device=dev)[:, None]).clamp(-1, 1) + 1]
    for h in range(H):
        x = [y.double() for y in (q[:, h], k[:, h // (H // Hk)], v[:, h // (H // Hk)], do[:, h])]
        s = D ** -0.5 * x[0] @ x[1].t() + bias[:, h].clamp(-LIMIT, LIMIT).double()[at]
        p = torch.softmax(s, -1)
        dp = x[3] @ x[2].t()
        moved = p * (dp - (p * dp).sum(-1, keepdim=True)).abs() + p * (p * dp.abs()).sum(-1, keepdim=True)
        large = bool((bias[:, h].abs() >= LIMIT).any())
        for b in range(3):
            if not past[b, h]:
                more = 2.0 ** -5 * float(moved[at == b].sum()) if large else 0.0
                ref.check(f"dbias {b} of head {h}", got[b, h], want[0][b, h], want[1][b, h] + more)
