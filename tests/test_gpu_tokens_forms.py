"""GPU tests of every form that the losses over a large vocabulary take, with random logits: rows and sizes on both sides
of each rule that chooses one, and gradients so large that they are stored past the caches.

Whole gradients are compared, with float64 on the GPU in groups of rows; the tolerances are those of test_gpu_tokens.  A
loss is a weighted sum of rows, each off by at most what its own terms are.
"""
import math

import numpy as np
import pytest
import torch

from oracle import token_oracle as O
from test_gpu_tokens import FAR, K, TINY, TYPES, close, f64, logp_tol, mean_tol, row_tol

pytestmark = pytest.mark.gpu

LO, HI, KL, ENT = 0.2, 0.25, 0.05, 0.02


# ------------------------------------------------------------------------------------------ float64 on the GPU
def softmax64(x, inv_t):
    z = x.double() * inv_t
    z = z - z.max(-1, keepdim=True).values
    logp = z - z.exp().sum(-1, keepdim=True).log()
    return logp.exp(), logp


def groups(n, v):
    step = max(1, (1 << 24) // v)
    return [slice(i, min(n, i + step)) for i in range(0, n, step)]


def logprobs64(x, y, on, inv_t):
    """ln p of y and the entropy of each row, 0 where it does not count: numpy."""
    lp, h = torch.zeros(len(y), dtype=torch.float64, device="cuda"), torch.zeros(len(y), dtype=torch.float64, device="cuda")
    for k in groups(*x.shape):
        p, logp = softmax64(x[k], inv_t)
        lp[k] = logp.gather(1, y[k, None])[:, 0]
        h[k] = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    return f64(lp * on), f64(h * on)


def check_gradient(got, x, want_of, off):
    """All of a gradient; want_of(rows) is the float64 one and the size of the terms that it is made of."""
    got, v = got.reshape(x.shape), x.shape[-1]
    eps = torch.finfo(got.dtype).eps
    for k in groups(*x.shape):
        want, size = want_of(k)
        err = (got[k].double() - want).abs()
        tol = want.abs() * eps / 2 + size * (3 * row_tol(v) + 2.0 ** -20 + FAR + off) + TINY[got.dtype]
        bad = ~(err <= tol)
        assert not bad.any(), (int(bad.sum()), float(err[bad].max()), (bad.nonzero()[:3] + torch.tensor([k.start, 0], device="cuda")).tolist())


def policy_want(x, y, on, inv_t, g_lp, g_h, wide):
    """The gradient from dloss/dlogp and dloss/dentropy; wide: the magnitude of what dloss/dlogp is the sum of."""
    g_lp, g_h, wide = (torch.from_numpy(np.asarray(a, np.float64)).cuda()[:, None] for a in (g_lp, g_h, wide))

    def want(k):
        p, logp = softmax64(x[k], inv_t)
        plnp = torch.where(p > 0, p * logp, 0.0)
        h = -plnp.sum(-1, keepdim=True)
        one = torch.zeros_like(p).scatter_(1, y[k, None], 1.0)
        g = inv_t * (g_lp[k] * (one - p) - g_h[k] * (plnp + p * h)) * on[k, None]
        return g, inv_t * (wide[k] * (one + p) + g_h[k].abs() * (plnp.abs() + p * h)) * on[k, None]
    return want


def teacher_want(x, index, q, w, inv_t):
    scale = torch.from_numpy(w / inv_t).cuda()[:, None]     # temperature^2 / temperature, times what the row counts

    def want(k):
        p, _ = softmax64(x[k], inv_t)
        mass = torch.zeros_like(p).scatter_add_(1, index[k].clamp(min=0), q[k])
        some = (q[k].sum(-1, keepdim=True) > 0).double()
        return scale[k] * (p - mass) * some, scale[k].abs() * (p + mass) * some
    return want


# ------------------------------------------------------------------------------------------ inputs
class Rows:
    """b * t rows of v logits, likely tokens, a mask of which one sequence is whole and (of three) one is empty; numbers
    beside them, ratios inside and outside of the clip range and none within 1e-3 of an edge."""
    def __init__(self, seed, b, t, v, dtype, inv_t=1.0, top=5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = np.random.default_rng(seed)
        n = b * t
        self.b, self.t, self.v, self.n, self.inv_t = b, t, v, n, inv_t
        self.x = torch.empty(b, t, v, dtype=dtype, device="cuda").normal_(0.0, 2.5, generator=g)
        flat = self.x.view(n, v)
        y = r.integers(0, v, n)
        y[: min(n, 2)] = [0, v - 1][: min(n, 2)]           # both ends of a row
        index = np.concatenate([y[:, None], r.integers(0, v, (n, top - 1))], 1)
        index[:, -1] = np.where(r.random(n) < 0.3, index[:, 0], index[:, -1])      # a token twice
        index[:, 1] = np.where(r.random(n) < 0.2, -1, index[:, 1])                 # and padding
        self.y, self.index = torch.from_numpy(y).cuda(), torch.from_numpy(index).cuda()
        near = math.log(v) + 2 - 2 * np.abs(r.standard_normal(n))
        flat.scatter_(1, self.y[:, None], torch.from_numpy(near[:, None]).to(dtype).cuda())
        mask = r.random((b, t)) < 0.8
        mask[0] = True
        if b > 2:
            mask[-1] = False
        self.mask = torch.from_numpy(mask).cuda()
        self.on = self.mask.view(n)
        self.values = torch.from_numpy(r.standard_normal((n, top)) * 2).to(dtype).cuda()
        self.lp, self.h = logprobs64(flat, self.y, self.on, inv_t)
        self.flat = flat
        self.off = 4 * float(logp_tol(self.lp, v).max()) + 2.0 ** -21
        d = r.choice([-0.6, -0.3, -0.1, -1e-3, 0.0, 1e-3, 0.1, 0.17, 0.29, 0.6], n) + r.uniform(-4e-4, 4e-4, n)
        self.old = (self.lp - d).astype(np.float32)
        self.adv = r.standard_normal(n).astype(np.float32)
        self.ref = (self.lp + r.choice([0.0, 1e-3, -0.2, 0.3, 1.5, -2.0], n)).astype(np.float32)

    def up(self, a, *more):
        return torch.from_numpy(a).cuda().view(self.b, self.t, *more)

    def close_rows(self, lp, h):
        close(lp.reshape(-1), self.lp, logp_tol(self.lp, self.v), "logprobs")
        close(h.reshape(-1), self.h, 2 * row_tol(self.v) * (1 + np.abs(self.h)) + 1e-6, "entropy")

    def check_logprobs(self):
        leaf = self.x.detach().requires_grad_(True)
        lp, h = K().token_logprobs(leaf, self.y.view(self.b, self.t), self.mask, temperature=1 / self.inv_t)
        self.close_rows(lp, h)
        with torch.no_grad():
            self.close_rows(*K().token_logprobs(leaf, self.y.view(self.b, self.t), self.mask, temperature=1 / self.inv_t))
        grad = torch.autograd.grad([lp, h], leaf, [self.up(self.adv), self.up(self.ref)])[0]
        check_gradient(grad, self.flat, policy_want(self.flat, self.y, self.on, self.inv_t, self.adv, self.ref, np.abs(self.adv)), 0.0)

    def check_policy(self, scale, in_place=False, reduction="token_mean"):
        on = f64(self.on)
        w = O.weights(on, self.b, self.t, reduction, scale)
        r, adv, d = np.exp(self.lp - self.old), self.adv.astype(np.float64), self.ref - self.lp
        s1, s2 = r * adv, np.clip(r, 1 - LO, 1 + HI) * adv
        each = -np.minimum(s1, s2) + KL * (np.expm1(d) - d) - ENT * self.h
        g = w * (np.where(s1 <= s2, -s1, 0.0) - KL * np.expm1(d))
        wide = w * np.maximum(np.abs(s1) + KL * np.exp(d), np.abs(g / np.where(w > 0, w, 1.0)))
        loss = float((w * each).sum())
        tol = mean_tol(w, (np.abs(adv) * 2 + KL * 10 + ENT * (1 + self.h)) * self.off) + 2.0 ** -23 * abs(loss) + 1e-12
        want = policy_want(self.flat, self.y, self.on, self.inv_t, g, -w * ENT, wide)
        args = (self.y.view(self.b, self.t), self.up(self.old), self.up(self.adv), self.mask)
        more = dict(ref_logprobs=self.up(self.ref), eps_clip=LO, eps_clip_high=HI, kl_coef=KL, entropy_coef=ENT,
                    temperature=1 / self.inv_t, reduction=reduction, scale=scale)
        leaf = self.x.detach().requires_grad_(True)
        one, lp, h = K().policy_loss(leaf, *args, **more)
        close(one, loss, tol, "loss")
        self.close_rows(lp, h)
        check_gradient(torch.autograd.grad(one, leaf)[0], self.flat, want, self.off)
        place = self.x.clone() if in_place else None
        two, grad, lp, h = K().policy_loss_and_grad(self.x if place is None else place, *args, **more, out=place)
        close(two, loss, tol, "loss")
        self.close_rows(lp, h)
        check_gradient(grad, self.flat, want, self.off)

    def check_preference(self, scale, in_place=False):
        r = np.random.default_rng(self.n)
        beta, pairs = 0.1, self.b // 2
        sums = self.lp.reshape(self.b, self.t).sum(1)
        ref = (sums + 3 * r.standard_normal(self.b)).astype(np.float32)
        rewards = beta * (sums - ref)
        z = rewards[:pairs] - rewards[pairs:]
        loss = scale * np.mean(np.logaddexp(0, -z))
        gz = scale * beta * (1 / (1 + np.exp(-z)) - 1) / pairs
        g = np.repeat(np.concatenate([gz, -gz]), self.t)
        tol = beta * self.t * (row_tol(self.v) + float(np.abs(self.lp).max()) * 2.0 ** -22)
        want = policy_want(self.flat, self.y, self.on, 1.0, g, 0 * g, np.abs(g))
        args = (self.y.view(self.b, self.t), torch.from_numpy(ref).cuda(), self.mask)
        leaf = self.x.detach().requires_grad_(True)
        one, got = K().preference_loss(leaf, *args, scale=scale)
        place = self.x.clone() if in_place else None
        two, grad, again = K().preference_loss_and_grad(self.x if place is None else place, *args, scale=scale, out=place)
        for some in (one, two):
            close(some, loss, 2 * scale * tol + 2.0 ** -23 * abs(loss), "loss")
        for some in (got, again):
            close(some, rewards, tol + np.abs(rewards) * 2.0 ** -24, "rewards")
        for some in (grad, torch.autograd.grad(one, leaf)[0]):
            check_gradient(some, self.flat, want, 2 * tol)

    def check_distillation(self, scale, in_place=False, reduction="token_mean"):
        top = self.index.shape[1]
        there = self.index >= 0
        q, logq = softmax64(torch.where(there, self.values.double(), -math.inf), self.inv_t)
        at = torch.empty_like(q)
        for k in groups(*self.flat.shape):
            at[k] = softmax64(self.flat[k], self.inv_t)[1].gather(1, self.index[k].clamp(min=0))
        each = f64(torch.where(q > 0, q * (logq - at), 0.0).sum(-1) * self.on) / self.inv_t ** 2
        w = O.weights(f64(self.on), self.b, self.t, reduction, scale)
        loss = float((w * each).sum())
        tol = (row_tol(self.v) + 60 * ((top + 8) * 2.0 ** -24 + 2.0 ** -22)) / self.inv_t ** 2
        want = teacher_want(self.flat, self.index, q, w, self.inv_t)
        args = (self.index.view(self.b, self.t, top), self.values.view(self.b, self.t, top), self.mask)
        more = dict(temperature=1 / self.inv_t, reduction=reduction, scale=scale)
        leaf = self.x.detach().requires_grad_(True)
        one, got = K().distillation_loss(leaf, *args, **more)
        place = self.x.clone() if in_place else None
        two, grad, again = K().distillation_loss_and_grad(self.x if place is None else place, *args, **more, out=place)
        for some in (one, two):
            close(some, loss, mean_tol(w, tol + np.abs(each) * 2.0 ** -22) + 2.0 ** -23 * abs(loss), "loss")
        for some in (got, again):
            close(some.reshape(-1), each, tol + np.abs(each) * 2.0 ** -23, "token losses")
        for some in (grad, torch.autograd.grad(one, leaf)[0]):
            check_gradient(some, self.flat, want, (top + 8) * 2.0 ** -24)

    def check_all(self, scale, in_place=False):
        self.check_logprobs()
        for reduction in ("token_mean", "sequence_mean"):
            self.check_policy(scale, in_place, reduction)
            self.check_distillation(scale, in_place, reduction)
        if self.b % 2 == 0 and self.inv_t == 1.0:
            self.check_preference(scale, in_place)


def test_the_float64_gradients_are_the_oracles():
    s = Rows(1, 3, 4, 50, torch.float32, inv_t=1.25)
    x, y, on = f64(s.flat), s.y.cpu().numpy(), s.on.cpu().numpy()
    lp, h = O.logprobs(x, y, on, s.inv_t)
    assert np.abs(lp - s.lp).max() < 1e-12 and np.abs(h - s.h).max() < 1e-12
    want = O.logits_grad(x, y, on, s.inv_t, s.adv, s.ref)[0]
    assert np.abs(f64(policy_want(s.flat, s.y, s.on, s.inv_t, s.adv, s.ref, s.adv)(slice(0, 12))[0]) - want).max() < 1e-12
    w = O.weights(on, 3, 4, "token_mean", 2.0)
    want = O.distillation(x, s.index.cpu().numpy(), f64(s.values), on, w, s.inv_t)[1]
    q = softmax64(torch.where(s.index >= 0, s.values.double(), -math.inf), s.inv_t)[0]
    assert np.abs(f64(teacher_want(s.flat, s.index, q, w, s.inv_t)(slice(0, 12))[0]) - want).max() < 1e-12


# ------------------------------------------------------------------------------------------ the rules' both sides
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [300, 2601, 9001, 20011])
@pytest.mark.parametrize("b,t", [(7, 73), (4, 128), (3, 171)])
def test_511_to_513_rows(b, t, v, dtype):
    """512 rows: forward passes give a row fewer threads and more rows to the chip."""
    Rows(v + b, b, t, v, dtype, inv_t=1.0 if b == 4 else 1.25).check_all(64.0)


@pytest.mark.parametrize("dtype,v", [(d, v) for d, size in ((torch.float32, 4), (torch.bfloat16, 2), (torch.float16, 2))
                                     for kb in (4, 16, 32, 64, 96, 128, 256) for v in (kb * 1024 // size - 1, kb * 1024 // size,
                                                                                      kb * 1024 // size + 1)] +
                         [(torch.bfloat16, 8191), (torch.float32, 8193), (torch.bfloat16, 131072 + 64), (torch.float32, 65536 + 4099)])
def test_row_lengths_at_which_the_form_changes(dtype, v):
    """A row of 4 (a wave), 16 (threads of a forward pass), 32 (of a backward pass), 64 and 128 (cut), 96 (vectors a thread)
    and 256 KB (held), a logit less and a logit more; rows that are cut, rows that are not, and many."""
    for b, t in ((1, 3), (2, 67)) + (((4, 135),) if v <= 16385 else ()):
        Rows(v + t, b, t, v, dtype).check_all(64.0)


@pytest.mark.parametrize("b,t", [(4, 16), (5, 13), (2, 64), (3, 43)])
@pytest.mark.parametrize("v,dtype", [(70001, torch.float32), (131072, torch.bfloat16), (70001, torch.float16)])
def test_long_rows_on_both_sides_of_the_number_that_is_cut(b, t, v, dtype):
    Rows(v + t, b, t, v, dtype).check_all(64.0, in_place=True)


# ------------------------------------------------------------------------------------------ gradients past the caches
@pytest.mark.parametrize("b,t,v,dtype", [(8, 6400, 2001, torch.float16), (4, 750, 17005, torch.float32), (6, 351, 50001, torch.bfloat16),
                                         (2, 351, 150001, torch.float16), (2, 400, 131072, torch.bfloat16)])
@pytest.mark.parametrize("op", ["logprobs", "policy", "preference", "distillation"])
def test_gradients_of_more_than_192_mb(op, b, t, v, dtype):
    """They are stored past the caches: rows of a wave, of a workgroup with 8 and 16 vectors a thread and longer than it
    holds, aligned and not, in memory of their own and over the logits."""
    assert b * t * v * torch.finfo(dtype).bits // 8 > 192 << 20
    s = Rows(v, b, t, v, dtype)
    if op == "logprobs":
        s.check_logprobs()
    else:
        for in_place in (False, True):
            getattr(s, "check_" + op)(1024.0 * b * t / 64 if op != "preference" else 1024.0, in_place)


# ------------------------------------------------------------------------------------------ whole logits
@pytest.mark.parametrize("v,dtype", [(5, torch.float32), (1000, torch.float32), (2049, torch.bfloat16), (50001, torch.bfloat16)])
def test_whole_logits_with_the_last_position_masked_off(v, dtype):
    """A step without the copies that a slice costs in the backward pass: all of a model's logits, tokens and mask shifted
    instead, the last position not counted.  Loss and gradient have the bits of the sliced form."""
    b, t = 4, 9
    g = torch.Generator(device="cuda").manual_seed(v)
    full = torch.empty(b, t + 1, v, dtype=dtype, device="cuda").normal_(0.0, 2.5, generator=g)
    ids = torch.randint(0, v, (b, t + 1), generator=g, device="cuda")
    mask = torch.rand(b, t + 1, generator=g, device="cuda") < 0.8
    adv = torch.randn(b, generator=g, device="cuda")
    last = torch.nn.functional.pad
    tokens, counts = last(ids[:, 1:], (0, 1)), last(mask[:, 1:], (0, 1))
    old = K().token_logprobs(full, tokens, counts)[0] - 0.05
    leaf = full.clone().requires_grad_(True)
    loss = K().policy_loss(leaf[:, :-1], ids[:, 1:], old[:, :-1], adv, mask[:, 1:], reduction="sequence_mean")[0]
    want = torch.autograd.grad(loss, leaf)[0]
    other = K().policy_loss(leaf, tokens, old, adv, counts, reduction="sequence_mean")[0]
    assert torch.equal(loss, other) and torch.equal(torch.autograd.grad(other, leaf)[0], want)
    assert (want[:, -1] == 0).all() and want.abs().max() > 0
    sliced = full.clone()
    one = K().policy_loss_and_grad(sliced[:, :-1], ids[:, 1:], old[:, :-1], adv, mask[:, 1:], out=sliced[:, :-1])
    two = K().policy_loss_and_grad(full, tokens, old, adv, counts, out=full)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1][:, :-1]) and (two[1][:, -1] == 0).all()
