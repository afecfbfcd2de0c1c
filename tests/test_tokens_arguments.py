"""CPU tests of what the losses over a large vocabulary accept and refuse, beside test_tokens."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from ppo_amd import tokens as K
from test_tokens import good

OPS = ["token_logprobs", "policy_loss", "preference_loss", "distillation_loss"]


def forms(op):
    """The entry point and, of a loss, its form that gives the gradient too."""
    return [getattr(K, op)] + ([getattr(K, op + "_and_grad")] if op != "token_logprobs" else [])


@pytest.mark.parametrize("op", OPS)
def test_logits_that_are_yet_to_be_negated_are_refused(op):
    for fn in forms(op):
        with pytest.raises(ValueError, match="yet to negate"):
            fn(**{**good(op), "logits": torch._neg_view(torch.zeros(2, 3, 7))})
        if fn is not forms(op)[0]:
            with pytest.raises(ValueError, match="yet to negate"):
                fn(**good(op), out=torch._neg_view(torch.zeros(2, 3, 7)))


FLOATS = {"token_logprobs": ["logits"], "policy_loss": ["logits", "old_logprobs", "advantages", "ref_logprobs"],
          "preference_loss": ["logits", "ref_logprobs"], "distillation_loss": ["logits", "teacher_logits"]}


@pytest.mark.parametrize("op,name", [(op, name) for op in OPS for name in FLOATS[op]])
def test_inputs_with_a_forward_mode_derivative_are_refused(op, name):
    """The results would carry none, which torch takes for zero."""
    for fn in forms(op):
        with forward_ad.dual_level():
            a = good(op)
            a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
            with pytest.raises(NotImplementedError, match=f"{name}.*forward-mode"):
                fn(**a)
            a[name] = forward_ad.unpack_dual(a[name]).primal
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                fn(**a)


@pytest.mark.parametrize("op", OPS[1:])
def test_out_with_a_forward_mode_derivative_is_refused(op):
    with forward_ad.dual_level():
        out = forward_ad.make_dual(torch.zeros(2, 3, 7), torch.ones(2, 3, 7))
        with pytest.raises(NotImplementedError, match="out.*forward-mode"):
            forms(op)[1](**good(op), out=out)
