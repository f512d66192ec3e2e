"""Derivatives that the packed-sequence operators do not have are refused in every mode of torch's, never left out."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from self_trainable_or_free_attn_amd import _lib, packed_attention, shared_prefix_attention

NAMES = ("q", "k_prefix", "v_prefix", "k", "v")


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, device="meta", dtype=dtype)


def _shared():
    kv, cache = _meta(5, 2, 64), _meta(3, 7, 2, 64)
    return [_meta(3, 2, 4, 64), kv, kv.clone(), cache, cache.clone()], _meta(3, dtype=torch.int32)


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("grad", [False, True])
def test_shared_prefix_refuses_a_tangent(which, grad):
    tensors, lens = _shared()
    with fw.dual_level(), torch.set_grad_enabled(grad):
        tensors[which] = fw.make_dual(tensors[which], torch.empty_like(tensors[which]))
        with pytest.raises(RuntimeError, match=f"no forward-mode derivative, and {NAMES[which]} has a tangent"):
            shared_prefix_attention(*tensors, lens)


@pytest.mark.parametrize("which", range(5))
def test_shared_prefix_refuses_function_transforms(which):
    tensors, lens = _shared()

    def f(x):
        return shared_prefix_attention(*tensors[:which], x, *tensors[which + 1:], lens)

    x = tensors[which]
    with pytest.raises(RuntimeError, match="has a tangent"):
        torch.func.jvp(f, (x,), (torch.empty_like(x),))
    with torch.no_grad(), pytest.raises(RuntimeError, match="has a tangent"):
        torch.func.jvp(f, (x,), (torch.empty_like(x),))
    with pytest.raises(ValueError, match="no backward"):
        torch.func.vjp(f, x)


@pytest.mark.parametrize("which", range(5))
def test_shared_prefix_operator_refuses_a_gradient(which):
    """The operator below the Python entry point, called directly."""
    tensors, lens = _shared()
    op = _lib.ops().shared_prefix_attention
    tensors[which].requires_grad_()
    with pytest.raises(RuntimeError, match=f"no backward, and {NAMES[which]} requires a gradient"):
        op(*tensors, lens, 0.125)
    with torch.no_grad():
        out, lse = op(*tensors, lens, 0.125)
    assert out.shape == tensors[0].shape and not out.requires_grad and lse.shape == (3, 2, 4)


def test_shared_prefix_without_derivatives_still_runs():
    tensors, lens = _shared()
    with fw.dual_level():      # (a level alone is no tangent)
        assert shared_prefix_attention(*tensors, lens).shape == tensors[0].shape
    with torch.inference_mode():
        assert shared_prefix_attention(*tensors, lens).shape == tensors[0].shape


def test_packed_refuses_a_tangent():
    q, k = _meta(10, 4, 64), _meta(10, 2, 64)
    with fw.dual_level(), pytest.raises(RuntimeError, match="jvp is not implemented"):
        packed_attention(fw.make_dual(q, torch.empty_like(q)), k, k)
