"""GPU tests of the losses over a large vocabulary: layouts and inputs at the edges of what their documentation allows."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_gpu_tokens import K, TYPES, all_three, calls, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,v", [(3, 4, 70), (2, 300, 1003), (2, 5, 33000), (1, 3, 70001), (2, 2, 140001), (3, 30, 140001)])
def test_a_row_without_entries_has_no_gradient_whatever_its_logits(b, t, v, dtype):
    """Rows whose teacher gave padding only: loss and gradient are 0 though the logits are NaN or infinite, in each form,
    and the other rows are as they are beside ordinary logits."""
    x, y, _ = make(v + t, b, t, v, dtype, masked=False)
    index = torch.stack([y, (y + 1) % v, y * 0 - 1], -1)
    values = torch.stack([y * 0.0, y * 0.0 - 1, y * 0.0 + 9], -1)
    none = torch.zeros(b, t, dtype=torch.bool, device="cuda")
    none[0, 0] = none[-1, -1] = True
    index[none] = -1
    bad = x.clone()
    bad[0, 0, v // 3] = math.nan
    bad[-1, -1] = -math.inf
    bad[-1, -1, v // 2] = math.inf
    results = []
    for logits in (x, bad):
        both = K().distillation_loss_and_grad(logits, index, values)
        place = logits.clone()
        over = K().distillation_loss_and_grad(place, index, values, out=place)
        leaf = logits.clone().requires_grad_(True)
        loss, each = K().distillation_loss(leaf, index, values)
        later = torch.autograd.grad(loss, leaf)[0]
        results.append([*both, *over, loss.detach(), each, later])
        for grad in (both[1], over[1], later):
            assert (grad[none] == 0).all()
        for each in (both[2], over[2], each):
            assert (each[none] == 0).all() and torch.isfinite(each).all()
    for a, c in zip(*results):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype,v", [(torch.float32, 7), (torch.bfloat16, 1001), (torch.float16, 4099), (torch.bfloat16, 70001)])
def test_gradient_over_logits_of_which_the_tokens_come_first(dtype, v):
    """Storage [tokens, sequences, vocabulary] seen as [sequences, tokens, vocabulary]: the same bits as in dense memory of
    the same alignment, in the logits' own place, in other memory of that order and in dense memory."""
    b, t = 4, 3
    x, y, m = make(v, b, t, v, dtype)
    first = torch.zeros(t, b, v + v % 2, dtype=dtype, device="cuda")      # rows on 4-byte boundaries at least
    view = lambda f: f[..., :v].transpose(0, 1)  # noqa: E731
    view(first).copy_(x)
    want = all_three(view(first), y, m)
    z = torch.full(y.shape, -2.0, device="cuda")
    index, values = torch.stack([y, (y + 1) % v], -1), torch.stack([z, z - 1], -1)
    for k, fn in enumerate([lambda a, o: K().policy_loss_and_grad(a, y, z, z, m, ref_logprobs=z, kl_coef=0.1, out=o),
                            lambda a, o: K().preference_loss_and_grad(a, y, z.sum(-1), m, out=o),
                            lambda a, o: K().distillation_loss_and_grad(a, index, values, m, out=o)]):
        own, other = first.clone(), torch.full_like(first, 7.0)
        for got in (fn(view(own), view(own)), fn(view(first), view(other))):
            for a, c in zip(want[k], got):
                assert torch.equal(a, c)
        assert torch.equal(view(own), want[k][1]) and (other[..., v:] == 7).all()


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


def test_incoming_gradients_with_a_forward_mode_derivative_are_refused():
    x, y, m = make(24, 2, 3, 500, torch.float32)
    for fn in calls(x, y, m):
        a = x.clone().requires_grad_(True)
        loss = fn(a)
        with forward_ad.dual_level():
            up = forward_ad.make_dual(torch.ones_like(loss), torch.ones_like(loss))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(loss, a, up, retain_graph=True)
        assert torch.isfinite(torch.autograd.grad(loss, a)[0]).all()


@pytest.mark.parametrize("shape", [(1,), (1, 1)])
@pytest.mark.parametrize("v", [5, 900, 70001])
def test_one_advantage_of_the_one_sequence(shape, v):
    x, y, m = make(9, 1, 7, v, torch.float32)
    x, y, m = x[0], y[0], torch.arange(7, device="cuda") != 2
    old, adv = torch.full((7,), -4.0, device="cuda"), torch.full(shape, -1.5, device="cuda")
    every = adv.reshape(1).expand(7)
    for a, c in zip(K().policy_loss_and_grad(x, y, old, adv, m), K().policy_loss_and_grad(x, y, old, every, m)):
        assert torch.equal(a, c)
    x.requires_grad_(True)
    a, c = (torch.autograd.grad(K().policy_loss(x, y, old, d, m)[0], x)[0] for d in (adv, every))
    assert torch.equal(a, c)


@pytest.mark.parametrize("v", [6, 900, 20003, 70001])
def test_divergence_at_an_impossible_token_is_infinite(v):
    """ln p = -inf, so d = ref - ln p is +inf and e^d - d - 1 is: not the difference of two infinities."""
    x, y, _ = make(5, 1, 5, v, torch.float32, masked=False)
    x[0, 2, y[0, 2]] = -math.inf
    z = torch.full((1, 5), -2.0, device="cuda")
    losses = [K().policy_loss_and_grad(x, y, z, z, ref_logprobs=z, kl_coef=0.1)[0],
              K().policy_loss(x, y, z, z, ref_logprobs=z, kl_coef=0.1)[0]]
    ref = z.clone()
    ref[0, 1] = -math.inf                         # a token that the reference policy rules out
    x[0, 2, y[0, 2]] = 1.0
    losses.append(K().policy_loss_and_grad(x, y, z, z, ref_logprobs=ref, kl_coef=0.1)[0])
    for loss in losses:
        assert float(loss) == math.inf


def test_c_abi_pair_of_which_the_label_is_certainly_wrong():
    """label_smoothing = 1: the rejected sequence is the better one, whatever the preferred one's probability."""
    from ppo_amd import _lib
    x, y, _ = make(8, 2, 3, 50, torch.float32, masked=False)
    x[0, 1, y[0, 1]] = -math.inf                  # the preferred sequence cannot happen: z = -inf, sigmoid(-z) = 1
    ref, loss, rewards = torch.zeros(2, device="cuda"), torch.ones((), device="cuda"), torch.zeros(2, device="cuda")
    L = _lib.lib()
    rows = _lib.TokenLogits(x.data_ptr(), x.stride(0), x.stride(1), 0, 0, 2, 3, 50, 0, 1.0)
    need = L.ppo_token_workspace_bytes(2, 3)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    code = L.ppo_preference_loss(ctypes.byref(rows), y.data_ptr(), 1, None, ref.data_ptr(), 0.1, 1.0, 1.0, loss.data_ptr(),
                                 rewards.data_ptr(), None, None, None, ws.data_ptr(), need,
                                 torch.cuda.current_stream().cuda_stream)
    assert code == 0 and float(rewards[0]) == -math.inf and float(loss) == 0.0
