"""CPU tests of what the losses over a large vocabulary accept and refuse, beside test_tokens."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from ppo_amd import _lib, tokens as K
from test_tokens import good, logits_struct

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


@pytest.mark.parametrize("op", OPS[1:])
@pytest.mark.parametrize("shape,view", [((3, 2, 7), lambda f: f.transpose(0, 1)), ((3, 2, 9), lambda f: f.transpose(0, 1)[..., 1:8]),
                                        ((3, 6, 7), lambda f: f[:, ::3].transpose(0, 1)), ((2, 9, 7), lambda f: f[:, ::3])])
def test_rows_of_out_in_either_order(op, shape, view):
    """Storage in which the positions come first, with room between the rows: the logits' own place or other memory."""
    a, out = good(op), view(torch.zeros(shape))
    with pytest.raises(RuntimeError, match="no CPU fallback"):      # all arguments have been accepted
        forms(op)[1](**a, out=out)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        forms(op)[1](**{**a, "logits": out}, out=out)


@pytest.mark.parametrize("op", OPS[1:])
@pytest.mark.parametrize("strides", [(7, 13, 1), (6, 14, 1), (13, 7, 1), (20, 7, 1), (7, 7, 1), (0, 7, 1), (7, 0, 1)])
def test_rows_of_out_that_overlap_in_either_order(op, strides):
    with pytest.raises(ValueError, match="overlap"):
        forms(op)[1](**good(op), out=torch.zeros(99).as_strided((2, 3, 7), strides))


@pytest.mark.parametrize("n_seq,n_tok,seq,tok,fits", [
    (2, 4, 40, 10, True), (2, 4, 10, 20, True), (2, 4, 11, 21, True), (2, 4, 10, 19, False), (2, 4, 9, 20, False), (2, 4, 10, 10, False),
    (3, 4, 10, 29, False), (3, 4, 10, 30, True), (3, 4, 1 << 62, 10, True), (3, 4, 10, 1 << 62, True), (1, 4, 0, 10, True),
    (1, 4, 0, 9, False), (4, 1, 10, 0, True), (4, 1, 9, 0, False), (1, 1, 0, 0, True), (1 << 15, 1 << 15, 1 << 62, 1 << 50, False),
    (2, 4, -40, 10, False), (2, 4, 10, -20, False)])
def test_c_abi_rows_of_the_gradient_in_either_order(n_seq, n_tok, seq, tok, fits):
    """Strides that do not fit are a bad argument; those that do are not, and the missing statistics or workspace are found next."""
    x = ctypes.byref(logits_struct(n_seq=n_seq, n_tok=n_tok, grad_seq_stride=seq, grad_tok_stride=tok))
    L, at = _lib.lib(), 1 << 20   # a pointer that is never followed
    terms = ctypes.byref(_lib.PolicyTerms(0.2, 0.2, 0.0, 0.0, 1.0, 1))
    want = -2 if fits else -1
    assert L.ppo_policy_loss(x, at, 1, None, at, at, 4, 1, None, terms, at, at, at, None, None, at, at, 0, None) == want
    assert L.ppo_distillation_loss(x, at, 1, at, 0, 4, None, 1, 1.0, at, at, None, at, at, 0, None) == want
    if n_seq % 2 == 0:
        assert L.ppo_preference_loss(x, at, 1, None, at, 0.1, 0.0, 1.0, at, at, None, None, at, at, 0, None) == want


@pytest.mark.parametrize("rows,shape,fits", [((3,), (1,), True), ((3,), (1, 1), True), ((3,), (3,), True), ((0,), (1,), True),
                                             ((3,), (2,), False), ((3,), (3, 1), False), ((3,), (1, 3), False), ((3,), (), False),
                                             ((2, 3), (2,), True), ((2, 3), (2, 1), True), ((2, 3), (1,), False),
                                             ((2, 3), (1, 1), False), ((1, 3), (1,), True), ((1, 3), (1, 1), True)])
def test_shapes_of_advantages(rows, shape, fits):
    z = torch.zeros(rows)
    for fn in forms("policy_loss"):
        with pytest.raises(RuntimeError if fits else ValueError, match="no CPU fallback" if fits else "advantages of shape"):
            fn(torch.zeros(*rows, 7), z.long(), z, torch.zeros(shape))
