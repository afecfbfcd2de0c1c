"""CPU-only tests of the losses over a large vocabulary: the oracle's gradients against central differences, and
what the C ABI and the Python entry points refuse before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import token_oracle as O
from ppo_amd import _lib, tokens as K


# ------------------------------------------------------------------------------------------ oracle
def differences(f, x, h=1e-5):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        g[i] = (f(a) - f(b)) / (2 * h)
    return g


def rows(seed, n=6, v=5):
    r = np.random.default_rng(seed)
    mask = np.array([1, 1, 0, 1, 0, 1], bool)[:n]
    return r, r.standard_normal((n, v)), r.integers(0, v, n), mask


@pytest.mark.parametrize("inv_t", [1.0, 0.5, 1.7])
def test_oracle_logprob_and_entropy_gradients_are_the_differences(inv_t):
    r, x, y, mask = rows(0)
    a, b = r.standard_normal(6), r.standard_normal(6)

    def f(z):
        lp, h = O.logprobs(z, y, mask, inv_t)
        return (a * lp).sum() + (b * h).sum()
    # central differences: h^2/6 of the third derivative (~1) + 2^-53 / h
    assert np.abs(O.logits_grad(x, y, mask, inv_t, a * mask, b * mask)[0] - differences(f, x)).max() < 1e-9


@pytest.mark.parametrize("reduction", ["sum", "token_mean", "sequence_mean"])
def test_oracle_policy_gradient_is_the_differences(reduction):
    r, x, y, mask = rows(1)
    lp, _ = O.logprobs(x, y, mask, 0.8)
    old, adv, ref = lp - np.array([.05, .5, 0, -.5, 0, .1]), np.array([1., 1, 9, -1, 9, -2]), lp + 0.3
    w = O.weights(mask, 2, 3, reduction, 1.5)
    f = lambda z: O.policy(z, y, old, adv, mask, ref, w, 0.2, 0.3, 0.1, 0.01, 0.8)[0]  # noqa: E731
    assert np.abs(O.policy(x, y, old, adv, mask, ref, w, 0.2, 0.3, 0.1, 0.01, 0.8)[1] - differences(f, x)).max() < 1e-8


def test_oracle_preference_gradient_is_the_differences():
    r, x, y, mask = rows(2, n=4)
    ref = r.standard_normal(2)
    f = lambda z: O.preference(z, y, mask[:4], ref, 2, 0.7, 0.1, 2.0)[0]  # noqa: E731
    assert np.abs(O.preference(x, y, mask[:4], ref, 2, 0.7, 0.1, 2.0)[1] - differences(f, x)).max() < 1e-9


def test_oracle_distillation_gradient_is_the_differences():
    r, x, y, mask = rows(3)
    index = np.array([[0, 2, -1], [1, 1, 4], [0, 1, 2], [-1, -1, -1], [2, 2, 2], [4, 0, 3]])
    teacher = r.standard_normal((6, 3))
    w = O.weights(mask, 2, 3, "token_mean", 1.0)
    f = lambda z: O.distillation(z, index, teacher, mask, w, 0.5)[0]  # noqa: E731
    assert np.abs(O.distillation(x, index, teacher, mask, w, 0.5)[1] - differences(f, x)).max() < 1e-9


# ------------------------------------------------------------------------------------------ C ABI refusals
def logits_struct(**more):
    d = dict(data=1 << 20, seq_stride=40, tok_stride=10, grad_seq_stride=40, grad_tok_stride=10, n_seq=2, n_tok=4, vocab=10,
             dtype=0, inv_temperature=1.0)
    d.update(more)
    return _lib.TokenLogits(**d)


BAD_LOGITS = [(dict(dtype=3), -1), (dict(vocab=0), -1), (dict(n_seq=-1), -1), (dict(inv_temperature=0.0), -1),
              (dict(inv_temperature=float("nan")), -1), (dict(inv_temperature=float("inf")), -1), (dict(data=None), -1),
              (dict(data=(1 << 20) + 2), -1), (dict(vocab=(1 << 26) + 1), -3), (dict(n_seq=1 << 20, n_tok=1 << 20), -3)]
BAD_GRADS = [(dict(grad_tok_stride=9), -1), (dict(grad_seq_stride=39), -1), (dict(grad_tok_stride=0), -1)]


@pytest.mark.parametrize("more,code", BAD_LOGITS)
def test_c_abi_refuses_logits(more, code):
    L, x = _lib.lib(), ctypes.byref(logits_struct(**more))
    at = 1 << 20   # a pointer that is never followed: every call is refused before a launch
    terms = ctypes.byref(_lib.PolicyTerms(0.2, 0.2, 0.0, 0.0, 1.0, 1))
    assert L.ppo_token_logprobs(x, at, 1, None, at, None, None, None, 0, None) == code
    assert L.ppo_token_logprobs_backward(x, at, 1, None, at, at, 4, 1, None, 0, 0, None, at, None) == code
    assert L.ppo_policy_loss(x, at, 1, None, at, at, 4, 1, None, terms, at, at, at, None, None, at, at, 1 << 40, None) == code
    assert L.ppo_preference_loss(x, at, 1, None, at, 0.1, 0.0, 1.0, at, at, None, None, at, at, 1 << 40, None) == code
    assert L.ppo_distillation_loss(x, at, 1, at, 0, 4, None, 1, 1.0, at, at, None, at, at, 1 << 40, None) == code
    assert L.ppo_distillation_backward(x, at, 1, at, 0, 4, None, at, None, at, None) == code
    assert L.ppo_token_logprobs(None, at, 1, None, at, None, None, None, 0, None) == -1


@pytest.mark.parametrize("more,code", BAD_GRADS)
def test_c_abi_refuses_overlapping_gradient_rows(more, code):
    L, x, at = _lib.lib(), ctypes.byref(logits_struct(**more)), 1 << 20
    assert L.ppo_token_logprobs_backward(x, at, 1, None, at, at, 4, 1, None, 0, 0, None, at, None) == code
    assert L.ppo_distillation_backward(x, at, 1, at, 0, 4, None, at, None, at, None) == code


def test_c_abi_refuses_other_arguments():
    L, x, at = _lib.lib(), ctypes.byref(logits_struct()), 1 << 20
    odd = ctypes.byref(logits_struct(n_seq=3, grad_seq_stride=40))
    terms = lambda **k: ctypes.byref(_lib.PolicyTerms(*({**dict(lo=.2, hi=.2, kl=0., ent=0., scale=1., red=1), **k}).values()))  # noqa: E731
    policy = lambda t=terms(), ref=None, ws=at, size=1 << 40, loss=at, old=at, stats=None, seeds=None: L.ppo_policy_loss(  # noqa: E731
        x, at, 1, None, old, at, 4, 1, ref, t, loss, at, at, stats, seeds, at, ws, size, None)
    need = L.ppo_token_workspace_bytes(2, 4)
    assert need > 0 and L.ppo_token_workspace_bytes(-1, 4) == 0 and L.ppo_token_workspace_bytes(1 << 40, 1 << 40) == 0
    assert policy(size=need - 1) == -2 and policy(ws=None) == -2
    assert policy(t=terms(red=3)) == -1 and policy(t=terms(kl=0.1)) == -1 and policy(loss=None) == -1 and policy(old=None) == -1
    assert policy(stats=at) == -1 and policy(t=None) == -1
    assert L.ppo_preference_loss(odd, at, 1, None, at, 0.1, 0.0, 1.0, at, at, None, None, None, at, 1 << 40, None) == -1
    assert L.ppo_preference_loss(x, at, 1, None, at, 0.1, 0.0, 1.0, at, at, None, None, None, at, need - 1, None) == -2
    assert L.ppo_preference_loss(x, at, 1, None, None, 0.1, 0.0, 1.0, at, at, None, None, None, at, need, None) == -1
    distill = lambda top, dtype=0, red=1, size=1 << 40, loss=at: L.ppo_distillation_loss(  # noqa: E731
        x, at, 1, at, dtype, top, None, red, 1.0, loss, at, None, None, at, size, None)
    assert distill(0) == -1 and distill(513) == -3 and distill(4, dtype=5) == -1 and distill(4, red=-1) == -1
    assert distill(4, size=need - 1) == -2 and distill(4, loss=None) == -1
    assert L.ppo_token_logprobs(x, None, 1, None, at, None, None, None, 0, None) == -1
    assert L.ppo_token_logprobs(x, at, 1, None, at, None, None, at, need - 1, None) == -2
    assert L.ppo_token_logprobs_backward(x, at, 1, None, None, at, 4, 1, None, 0, 0, None, at, None) == -1
    empty = ctypes.byref(logits_struct(n_seq=0, data=None))
    assert L.ppo_token_logprobs(empty, None, 1, None, None, None, None, None, 0, None) == 0


def test_constants_are_the_headers():
    import os
    import re
    text = open(os.path.join(os.path.dirname(_lib.HERE), "include", "ppo_hip.h")).read()
    value = lambda name: int(re.search(rf"#define {name} (\d+)", text).group(1))  # noqa: E731
    assert K.MAX_TEACHER_TOP == value("PPO_MAX_TEACHER_TOP")
    assert K._REDUCTIONS == {"sum": value("PPO_REDUCE_SUM"), "token_mean": value("PPO_REDUCE_TOKEN_MEAN"),
                             "sequence_mean": value("PPO_REDUCE_SEQUENCE_MEAN")}


# ------------------------------------------------------------------------------------------ Python refusals
def good(op, device="cpu"):
    """Arguments that an entry point accepts, by name."""
    z = lambda *s: torch.zeros(s, device=device)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int64, device=device)  # noqa: E731
    a = {"logits": z(2, 3, 7), "mask": torch.ones(2, 3, dtype=torch.bool, device=device)}
    if op == "distillation_loss":
        return {**a, "teacher_tokens": i(2, 3, 2), "teacher_logits": z(2, 3, 2)}
    a["tokens"] = i(2, 3)
    if op == "policy_loss":
        return {**a, "old_logprobs": z(2, 3), "advantages": z(2, 3), "ref_logprobs": z(2, 3)}
    return {**a, "ref_logprobs": z(2)} if op == "preference_loss" else a


z3 = torch.zeros(2, 3, 7)
REFUSED = [
    ("token_logprobs", dict(logits=z3[0, 0]), "logits must be"),
    ("token_logprobs", dict(logits=z3.double()), "type torch.float64"),
    ("token_logprobs", dict(logits=z3[..., :0]), "empty vocabulary"),
    ("token_logprobs", dict(logits=z3.transpose(1, 2)), "contiguous dimension"),
    ("token_logprobs", dict(tokens=torch.zeros(2, 4, dtype=torch.int64)), "tokens of shape"),
    ("token_logprobs", dict(tokens=torch.zeros(2, 3)), "tokens of type"),
    ("token_logprobs", dict(mask=torch.ones(2, 3)), "mask of type"),
    ("token_logprobs", dict(mask=torch.ones(3, 2, dtype=torch.bool)), "mask of shape"),
    ("token_logprobs", dict(temperature=0.0), "temperature"),
    ("token_logprobs", dict(temperature=float("nan")), "temperature"),
    ("policy_loss", dict(advantages=torch.zeros(2, 3, requires_grad=True)), "advantages requires grad"),
    ("policy_loss", dict(advantages=torch.zeros(3)), "advantages of shape"),
    ("policy_loss", dict(old_logprobs=torch.zeros(2, 3, dtype=torch.int64)), "old_logprobs of type"),
    ("policy_loss", dict(old_logprobs=torch.zeros(2)), "old_logprobs of shape"),
    ("policy_loss", dict(ref_logprobs=None, kl_coef=0.1), "kl_coef without"),
    ("policy_loss", dict(eps_clip=1.5), "clip range"),
    ("policy_loss", dict(eps_clip_high=-0.1), "clip range"),
    ("policy_loss", dict(reduction="mean"), "reduction"),
    ("preference_loss", dict(logits=z3[:1], tokens=torch.zeros(1, 3, dtype=torch.int64), mask=None,
                             ref_logprobs=torch.zeros(1)), "preferred sequences"),
    ("preference_loss", dict(ref_logprobs=torch.zeros(2, 3)), "ref_logprobs of shape"),
    ("preference_loss", dict(label_smoothing=1.0), "label_smoothing"),
    ("distillation_loss", dict(teacher_tokens=torch.zeros(2, 3, dtype=torch.int64)), "teacher_tokens must be"),
    ("distillation_loss", dict(teacher_tokens=torch.zeros(2, 3, 513, dtype=torch.int64)), "teacher_tokens must be"),
    ("distillation_loss", dict(teacher_logits=torch.zeros(2, 3, 3)), "teacher_logits of shape"),
    ("distillation_loss", dict(teacher_logits=torch.zeros(2, 3, 2).double()), "teacher_logits of type"),
    ("distillation_loss", dict(temperature=-1.0), "temperature"),
]


@pytest.mark.parametrize("op,more,text", REFUSED)
def test_python_refuses(op, more, text):
    for fn in [getattr(K, op)] + ([getattr(K, op + "_and_grad")] if op != "token_logprobs" else []):
        with pytest.raises(ValueError, match=text):
            fn(**{**good(op), **more})


@pytest.mark.parametrize("op", ["policy_loss", "preference_loss", "distillation_loss"])
def test_python_refuses_out(op):
    fn, a = getattr(K, op + "_and_grad"), good(op)
    a["logits"] = torch.zeros(2, 3, 7)
    for out, text in [(torch.zeros(2, 3, 8), "shape"), (torch.zeros(2, 3, 7).half(), "type"),
                      (torch.zeros(2, 7, 3).transpose(1, 2), "contiguous"), (torch.zeros(2, 1, 7).expand(2, 3, 7), "overlap"),
                      (torch.zeros(30).as_strided((2, 3, 7), (7, 7, 1)), "overlap")]:
        with pytest.raises(ValueError, match=text):
            fn(**a, out=out)
    store = torch.zeros(100)
    a["logits"] = store[:42].view(2, 3, 7)
    with pytest.raises(ValueError, match="shares memory with the logits"):
        fn(**a, out=store[7:49].view(2, 3, 7))
    with pytest.raises(ValueError, match="overlap"):
        a["logits"] = torch.zeros(1, 3, 7).expand(2, 3, 7)
        fn(**a, out=a["logits"])


@pytest.mark.parametrize("op", ["token_logprobs", "policy_loss", "preference_loss", "distillation_loss"])
def test_no_cpu_fallback(op):
    fns = [getattr(K, op)] + ([getattr(K, op + "_and_grad")] if op != "token_logprobs" else [])
    for fn in fns:
        for grad in (False, True):
            a = good(op)
            a["logits"].requires_grad_(grad)
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                fn(**a)


def test_gradient_storage_follows_the_logits_rows_where_that_is_cheap():
    full = torch.zeros(2, 5, 33)
    for view in (full[:, :-1], full[..., 1:], full[:, 1:]):
        g = K._ops.grad_like(view)
        assert g.shape == view.shape and g.stride() == view.stride()
    for view in (full[:, -1:], torch.zeros(1, 4, 33).expand(2, 4, 33), full.transpose(0, 1), torch.zeros(2, 0, 3), full):
        assert K._ops.grad_like(view).is_contiguous()
