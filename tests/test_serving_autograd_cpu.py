"""What autograd is told about qk_norm_rope, append_kv and paged_attention: refusals, without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from attention.paged.cache import append_kv
from attention.paged.paged_attention import paged_attention
from attention.rotary.norm_rope import qk_norm_rope
from tests.test_serving_cpu import half, rope_args, step_args


def dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


@pytest.mark.parametrize("name", ["q", "k", "q_weight", "k_weight", "cos", "sin"])
def test_norm_rope_refuses_dual_tensors(name):
    """A tangent would be dropped silently."""
    args = rope_args(q_weight=half(64), k_weight=half(64))
    with forward_ad.dual_level():
        args[name] = dual(args[name])
        with pytest.raises(RuntimeError, match="forward-mode"):
            qk_norm_rope(**args)


@pytest.mark.parametrize("name", ["k", "v", "k_weight"])
def test_append_refuses_dual_tensors(name):
    args = step_args(k=half(3, 2, 64), v=half(3, 2, 64), k_weight=half(64))
    with forward_ad.dual_level(), torch.no_grad():
        args[name] = dual(args[name])
        with pytest.raises(RuntimeError, match="forward-mode"):
            append_kv(**args)


@pytest.mark.parametrize("name", ["q", "out"])
def test_attention_refuses_dual_tensors(name):
    args = step_args(q=half(3, 4, 64), out=half(3, 4, 64))
    with forward_ad.dual_level(), torch.no_grad():
        args[name] = dual(args[name])
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged_attention(**args)


def test_tensors_that_are_written_must_not_require_gradients():
    with pytest.raises(RuntimeError, match="out, which must not require"):
        paged_attention(**step_args(q=half(3, 4, 64), out=half(3, 4, 64).requires_grad_(True)))
    args = step_args(k=half(3, 2, 64), v=half(3, 2, 64))
    args["cache"].v_scales = args["cache"].v_scales.requires_grad_(True)
    with pytest.raises(RuntimeError, match="cache, which must not require"):
        append_kv(**args)
