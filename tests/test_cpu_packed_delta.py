"""The bounds of packed_delta_ref.py tell a backward that takes delta from the rounded output from one that sums it itself."""
import pytest
import torch

import packed_delta_ref as ref


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_bounds_exclude_delta_from_the_output(dtype, D):
    n = 400
    q, k, v, do = (x.transpose(0, 1) for x in ref.telling_inputs(n, n, 1, 1, D, dtype))
    at = (torch.arange(n)[None] - torch.arange(n)[:, None]).clamp(-7, 7) + 7
    seen, k, v = torch.ones(n, n, dtype=torch.bool), k[0], v[0]
    x = [y.double() for y in (q, k, v, do)]
    value, bound = ref.by_bucket(ref.attention(*x, seen, 0.125, None, dtype)["ds"], at, 15)
    # the same in float32, delta summed: inside
    p = torch.softmax(0.125 * q.float() @ k.float().t(), -1)
    dp = do.float() @ v.float().t()
    good = ref.by_bucket((p * (dp - (p * dp).sum(-1, keepdim=True)),) * 2, at, 15)[0]
    assert bool(((good.double() - value).abs() <= bound).all())
    # delta from the output as it is stored: outside
    delta = (do.double() * (p @ v.float()).to(dtype).double()).sum(-1, keepdim=True)
    wrong = ref.by_bucket(ref.attention(*x, seen, 0.125, None, dtype, delta=delta)["ds"], at, 15)[0]
    assert bool(((wrong - value).abs() > 5 * bound).all())
