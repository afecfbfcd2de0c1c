"""CPU tests of what the losses over a large vocabulary accept and refuse, beside test_tokens."""
import pytest
import torch

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
