"""GPU tests of the losses over a large vocabulary: layouts and inputs at the edges of what their documentation allows."""
import pytest
import torch

from test_gpu_tokens import K, make

pytestmark = pytest.mark.gpu


def negated(t):
    """t as a view that torch has yet to negate."""
    n = torch.imag(torch.complex(torch.zeros_like(t), -t).conj())
    assert n.is_neg() and torch.equal(n, t)
    return n


def test_lazily_negated_gradients_and_inputs():
    """Complex arithmetic after the log-probabilities gives gradients that are lazily negated views; so may be the numbers
    beside the logits."""
    x, y, m = make(23, 2, 6, 700, torch.float32)
    r = torch.Generator(device="cuda").manual_seed(3)
    g_lp, g_h = (torch.randn(2, 6, generator=r, device="cuda") for _ in range(2))
    x.requires_grad_(True)
    lp, h = K().token_logprobs(x, y, m)
    want = torch.autograd.grad([lp, h], x, [g_lp, g_h], retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad([lp, h], x, [negated(g_lp), negated(g_h)], retain_graph=True)[0], want)
    want = torch.autograd.grad(lp.sum(), x, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad((-torch.complex(g_lp, lp).conj().imag).sum(), x)[0], want)
    a = lambda f: K().policy_loss_and_grad(x, y, f(g_lp - 6), f(g_h), m, ref_logprobs=f(g_lp - 5), kl_coef=0.1)  # noqa: E731
    c = lambda f: K().preference_loss_and_grad(x, y, f(g_lp[:, 0]), m)  # noqa: E731
    e = lambda f: K().distillation_loss_and_grad(x, y[..., None], f(g_lp[..., None]), m)  # noqa: E731
    for fn in (a, c, e):
        for p, q in zip(fn(lambda t: t), fn(negated)):
            assert torch.equal(p, q)
    loss = lambda: K().policy_loss(x, y, g_lp - 6, g_h, m)[0]  # noqa: E731
    up = torch.tensor(0.5, device="cuda")
    assert torch.equal(torch.autograd.grad(loss(), x, negated(up))[0], torch.autograd.grad(loss(), x, up)[0])
