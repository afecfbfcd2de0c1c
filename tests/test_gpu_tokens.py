"""GPU tests of the losses over a large vocabulary against the float64 oracle.

Tolerances.  A row's S = sum e_i is a sum of positive fp32 terms: at most CHAIN additions follow one another (a
thread's own terms, then about 20 to join), each off by at most 2^-24 of the running sum, and each term by 2^-22
(exp2 to two units in the last place, its argument u rounded twice: 2^-23 |u| ln 2, with e_i u_i small where |u| is
large; the terms that matter have |u| < 24, together below 24 * 2^-23 = 3e-6).  So ln S is off by at most
ROW = CHAIN * 2^-24 + 2^-22 + 3e-6.  A log-probability adds 2^-24 of itself (its rounding to fp32) and 2^-23 for the
rounded 1/temperature; a gradient's terms are off by 3 ROW + 2^-20 of their own magnitude (p, the entropy inside,
|u| up to 100 in p: 2^-23 * 100 * ln 2 = 8.3e-6 is added as FAR), and the gradient's rounding to its type is half a step.
"""
import math

import numpy as np
import pytest
import torch

from oracle import token_oracle as O

pytestmark = pytest.mark.gpu

FAR = 100 * 2.0 ** -23 * math.log(2.0)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}   # flushed, or half a subnormal step


def row_tol(v):
    return (max(128, v // 256) + 20) * 2.0 ** -24 + 2.0 ** -22 + 3e-6


def K():
    from ppo_amd import tokens
    return tokens


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, tol, what=""):
    got, want = f64(got) if isinstance(got, torch.Tensor) else np.asarray(got), np.asarray(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    with np.errstate(invalid="ignore"):
        bad = ~((got == want) | np.isnan(want) | (np.abs(got - want) <= tol))
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(np.abs(got - want))), np.argwhere(bad)[:3].tolist())


def close_grad(got, want, size, v, seeds_off=0.0):
    """seeds_off: relative error of what comes into the gradient (ratio, divergence)."""
    dtype = got.dtype
    got = got.reshape(-1, v)
    close(got, want, np.abs(want) * torch.finfo(dtype).eps / 2 + size * (3 * row_tol(v) + 2.0 ** -20 + FAR + seeds_off)
          + TINY[dtype], "grad")


def logp_tol(lp, v):
    return row_tol(v) + np.abs(np.where(np.isfinite(lp), lp, 0)) * (2.0 ** -24 + 2.0 ** -22)


def make(seed, b, t, v, dtype, masked=True, spread=2.5):
    """logits, tokens, mask on the GPU; likely tokens; the last sequence is empty where there are three, one is whole."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((b, t, v)) * spread
    y = r.integers(0, v, (b, t))
    np.put_along_axis(x, y[..., None], np.log(v) + 2 - 2 * np.abs(r.standard_normal((b, t, 1))), 2)
    mask = r.random((b, t)) < 0.7
    mask[0] = True
    if b > 2:
        mask[-1] = False
    x = torch.from_numpy(x).to(dtype).cuda()
    return x, torch.from_numpy(y).cuda(), torch.from_numpy(mask).cuda() if masked else None


def flat(x, y, m):
    v = x.shape[-1]
    return f64(x).reshape(-1, v), y.cpu().numpy().reshape(-1), None if m is None else m.cpu().numpy().reshape(-1)


def mean_tol(w, tol):
    return float((np.abs(w) * tol).sum())


SIZES = [(1, 1, 1), (2, 3, 2), (1, 1, 7), (3, 5, 64), (1, 4, 255), (4, 3, 1000), (2, 1, 2049), (3, 2, 4099), (2, 9, 8191),
         (1, 3, 16391), (2, 2, 50001)]
LARGE = [(1, 2, 131072, torch.bfloat16), (1, 1, 262144, torch.bfloat16), (1, 2, 70001, torch.float32),
         (2, 1, 150003, torch.float16), (1, 1, 300007, torch.float32)]
ALL = [(b, t, v, d) for b, t, v in SIZES for d in TYPES] + LARGE


# ------------------------------------------------------------------------------------------ log-probabilities
@pytest.mark.parametrize("b,t,v,dtype", ALL)
def test_logprobs_and_their_gradient(b, t, v, dtype):
    x, y, m = make(v + b, b, t, v, dtype)
    inv_t = [1.0, 0.5, 1.25][v % 3]
    fx, fy, fm = flat(x, y, m)
    lp, h = O.logprobs(fx, fy, fm, inv_t)
    r = np.random.default_rng(7)
    scale = 100.0 if dtype == torch.float16 else 1.0
    g_lp, g_h = (torch.from_numpy(scale * r.standard_normal((b, t)).astype(np.float32)).cuda() for _ in range(2))
    x.requires_grad_(True)
    for entropy in (True, False):
        got, ent = K().token_logprobs(x, y, m, temperature=1 / inv_t, entropy=entropy)
        close(got.reshape(-1), lp, logp_tol(lp, v), "logprobs")
        assert got.dtype == torch.float32 and (ent is None) == (not entropy)
        outs, seeds = ([got, ent], [g_lp, g_h]) if entropy else ([got], [g_lp])
        if entropy:
            close(ent.reshape(-1), h, 2 * row_tol(v) * (1 + np.abs(h)) + 1e-6, "entropy")
        grad = torch.autograd.grad(outs, [x], seeds)[0]
        assert grad.shape == x.shape and grad.dtype == dtype
        want, size = O.logits_grad(fx, fy, fm, inv_t, f64(g_lp).reshape(-1), f64(g_h).reshape(-1) * entropy)
        close_grad(grad, want, size, v)
        with torch.no_grad():
            again, _ = K().token_logprobs(x, y, m, temperature=1 / inv_t, entropy=entropy)
        close(again.reshape(-1), lp, logp_tol(lp, v), "logprobs")


@pytest.mark.parametrize("v", [33, 1000, 4099])
@pytest.mark.parametrize("dtype", TYPES)
def test_only_one_output_is_used(v, dtype):
    x, y, m = make(3, 2, 5, v, dtype)
    fx, fy, fm = flat(x, y, m)
    x.requires_grad_(True)
    for k in (0, 1):
        out = K().token_logprobs(x, y, m)[k]
        grad = torch.autograd.grad(out.sum(), x)[0]          # an expanded gradient comes in
        want, size = O.logits_grad(fx, fy, fm, 1.0, np.full(10, 1.0 - k), np.full(10, float(k)))
        close_grad(grad, want, size, v)


VIEWS = {
    "shifted": lambda f: f[:, :-1], "tail": lambda f: f[:, 1:], "padded vocabulary": lambda f: f[..., :-3],
    "vocabulary offset": lambda f: f[..., 5:], "every second": lambda f: f[:, ::2], "tokens first": lambda f: f.transpose(0, 1),
    "one sequence": lambda f: f[1], "last position": lambda f: f[:, -1:], "broadcast": lambda f: f[:1].expand(3, -1, -1),
    "one step": lambda f: f[:, 2],
}


@pytest.mark.parametrize("name", list(VIEWS))
@pytest.mark.parametrize("dtype,v", [(torch.float32, 77), (torch.bfloat16, 1001), (torch.float16, 4099)])
def test_views_of_logits(name, dtype, v):
    full, _, _ = make(11, 3, 5, v, dtype)
    full.requires_grad_(True)
    x = VIEWS[name](full)
    r = np.random.default_rng(5)
    w = x.shape[-1]
    y = torch.from_numpy(r.integers(0, w, x.shape[:-1]).astype(np.int32)).cuda()
    m = torch.from_numpy(r.random(x.shape[:-1]) < 0.8).cuda()
    fx, fy, fm = flat(x, y, m)
    lp, _ = O.logprobs(fx, fy, fm, 1.0)
    got, ent = K().token_logprobs(x, y, m)
    close(got.reshape(-1), lp, logp_tol(lp, w))
    grad = torch.autograd.grad(got.sum(), x)[0]
    n = len(fy)
    want, size = O.logits_grad(fx, fy, fm, 1.0, np.ones(n), np.zeros(n))
    close_grad(grad, want, size, w)
    # through the view to the whole tensor: broadcast rows add up, the rest is zero
    got, _ = K().token_logprobs(VIEWS[name](full), y, m)
    whole = f64(torch.autograd.grad(got.sum(), full)[0])
    probe = torch.zeros(full.shape, dtype=torch.float64, requires_grad=True)
    ref = torch.autograd.grad(VIEWS[name](probe), probe, torch.from_numpy(want.reshape(x.shape)))[0].numpy()
    eps = torch.finfo(dtype).eps
    assert np.abs(whole - ref).max() <= 4 * eps * max(1.0, np.abs(ref).max())   # three rounded rows added up in the type


def test_rows_that_do_not_count_are_not_used():
    b, t, v = 3, 4, 1003
    for dtype in TYPES:
        x, y, m = make(1, b, t, v, dtype)
        m[0, 1] = False
        bad = x.clone()
        bad[~m] = float("nan")
        wild = torch.where(m, y, torch.tensor([-100, 1 << 40, -(1 << 40), 5], device="cuda").repeat(b, 1))
        off = torch.where(m, torch.rand(b, t, device="cuda"), torch.tensor(float("nan"), device="cuda"))
        for args in [(x, y, torch.zeros_like(off).where(~m, off)), (bad, wild, off)]:
            logits, tok, side = args
            loss, grad, lp, h = K().policy_loss_and_grad(logits, tok, side - 7, side, m, ref_logprobs=side - 6, kl_coef=0.1,
                                                         entropy_coef=0.1)
            if logits is x:
                first = (loss, grad, lp, h)
        for a, c in zip(first, (loss, grad, lp, h)):
            assert torch.equal(a, c)
        assert (grad[~m] == 0).all() and (lp[~m] == 0).all() and (h[~m] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [40, 3000, 20003])
def test_impossible_tokens_and_extreme_logits(dtype, v):
    lowest, big = torch.finfo(dtype).min, torch.finfo(dtype).max
    x, y, _ = make(2, 1, 8, v, dtype)
    y[:] = 17
    x[0, 0, 3:9] = -math.inf                    # ruled out
    x[0, 1, 30:] = lowest                       # the same in other words
    x[0, 2] = lowest                            # uniform
    x[0, 3] = big                               # uniform
    x[0, 4, 17] = -math.inf                     # an impossible token was taken
    x[0, 5] = -math.inf
    x[0, 5, 17] = 1.0                           # the only possible one
    x[0, 6, :20] = big                          # all mass on twenty
    x[0, 7] += 1000.0 if dtype != torch.float16 else 100.0
    fx, fy, _ = flat(x, y, None)
    lp, h = O.logprobs(fx, fy, None, 1.0)
    x.requires_grad_(True)
    got, ent = K().token_logprobs(x, y)
    close(got.reshape(-1), lp, logp_tol(lp, v), "logprobs")
    close(ent.reshape(-1), h, 2 * row_tol(v) * (1 + np.abs(h)) + 1e-6, "entropy")
    grad = torch.autograd.grad([got, ent], [x], [torch.ones_like(got), torch.full_like(got, 0.5)])[0]
    want, size = O.logits_grad(fx, fy, None, 1.0, np.ones(8), np.full(8, 0.5))
    close_grad(grad, want, size, v)
    assert got[0, 4] == -math.inf and got[0, 5] == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,times", [(40, 1), (40, 30), (3000, 1), (20003, 20), (40001, 1), (40001, 20), (90001, 1), (140001, 18)])
def test_losses_of_extreme_logits(v, times, dtype):
    """Few and many rows, short and long ones, of logits so large or so low that the sums have to be taken exactly."""
    lowest, big = torch.finfo(dtype).min, torch.finfo(dtype).max
    x, y, _ = make(2, 1, 8, v, dtype)
    y[:] = 17
    x[0, 0, 3:9] = -math.inf
    x[0, 1, 30:] = lowest
    x[0, 2] = lowest
    x[0, 3] = big
    x[0, 5] = -math.inf
    x[0, 5, 17] = 1.0
    x[0, 6, :20] = big
    x[0, 7] += 1000.0 if dtype != torch.float16 else 100.0
    fx, fy, _ = flat(x, y, None)
    lp, h = O.logprobs(fx, fy, None, 1.0)
    old = (lp - 0.1).astype(np.float32)
    adv = np.array([1.0, -1.0, 0.5, -0.5, 2.0, 1.0, -2.0, 1.0], np.float32)
    w = np.full(8, 4.0 / 8)
    loss, grad, size, _ = O.policy(fx, fy, old, adv, None, None, w, 0.2, 0.2, 0.0, 0.02, 1.0)
    up = lambda a: torch.from_numpy(a).cuda()[None].repeat(times, 1)  # noqa: E731
    X, Y = x.repeat(times, 1, 1), y.repeat(times, 1)
    off = 4 * float(logp_tol(lp, v).max()) + 2.0 ** -21
    got = K().policy_loss_and_grad(X, Y, up(old), up(adv), entropy_coef=0.02, scale=4.0 * times)
    close(got[0], loss * times, times * mean_tol(w, (np.abs(adv) * 2 + 0.02 * (1 + h)) * off) + 2.0 ** -23 * abs(loss) * times, "loss")
    for t in (0, times - 1):
        close(got[2][t], lp, logp_tol(lp, v), "logprobs")
        close(got[3][t], h, 2 * row_tol(v) * (1 + np.abs(h)) + 1e-6, "entropy")
        close_grad(got[1][t], grad, size, v, off)
    index = torch.tensor([17, 2, 17, v - 1], device="cuda").repeat(times, 8, 1)
    index[:, 5, :] = 17                          # the teacher of the row with one possible token knows that one
    index[:, 0, 1] = 1
    index[:, 6, 3] = 1
    index[:, 1, 3] = 5
    values = torch.tensor([1.0, 0.5, 0.25, 0.0], device="cuda").repeat(times, 8, 1)
    fi, ft = index[0].cpu().numpy(), f64(values[0])
    loss, grad, size, each = O.distillation(fx, fi, ft, None, w, 1.0)
    got = K().distillation_loss_and_grad(X, index, values, scale=4.0 * times)
    tol = row_tol(v) + 60 * (12 * 2.0 ** -24 + 2.0 ** -22)
    close(got[0], loss * times, times * mean_tol(w, tol + np.abs(each) * 2.0 ** -22) + 2.0 ** -23 * abs(loss) * times, "loss")
    for t in (0, times - 1):
        close(got[2][t], each, tol + np.abs(each) * 2.0 ** -23, "token losses")
        close_grad(got[1][t], grad, size, v, 12 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES)
def test_bad_rows_are_nan_and_leave_the_others(dtype):
    b, t, v = 1, 7, 501
    x, y, _ = make(4, b, t, v, dtype)
    x[0, 1, 5] = float("nan")
    x[0, 2, 500] = math.inf
    x[0, 3] = -math.inf
    y[0, 4], y[0, 5] = v, -1
    x.requires_grad_(True)
    lp, h = K().token_logprobs(x, y)
    grad = torch.autograd.grad([lp, h], [x], [torch.ones_like(lp)] * 2)[0]
    assert torch.isnan(lp[0]).tolist() == [False, True, True, True, True, True, False]
    assert torch.isnan(h[0]).tolist() == [False, True, True, True, False, False, False]
    assert torch.isnan(grad[0]).any(-1).tolist() == [False, True, True, True, True, True, False]
    old = torch.full((b, t), -3.0, device="cuda")
    loss, g, lp2, _ = K().policy_loss_and_grad(x, y, old, old, reduction="sum")
    assert torch.isnan(loss) and torch.isnan(g[0]).any(-1).tolist() == torch.isnan(grad[0]).any(-1).tolist()
    assert torch.isnan(lp2).tolist() == torch.isnan(lp).tolist()


# ------------------------------------------------------------------------------------------ policy loss
def policy_inputs(seed, x, y, m, inv_t):
    """Ratios inside, above and below the clip range, none within 1e-3 of an edge (an error there may flip the gradient)."""
    r = np.random.default_rng(seed)
    fx, fy, fm = flat(x, y, m)
    lp, _ = O.logprobs(fx, fy, fm, inv_t)
    d = r.choice([-0.6, -0.3, -0.1, -1e-3, 0.0, 1e-3, 0.1, 0.17, 0.28, 0.6], len(lp)) + r.uniform(-4e-4, 4e-4, len(lp))
    old = (lp - d).astype(np.float32)
    adv = r.standard_normal(len(lp)).astype(np.float32)
    adv[r.random(len(lp)) < 0.1] = 0.0
    ref = (lp + r.choice([0.0, 1e-3, -0.2, 0.3, 1.5, -2.0], len(lp))).astype(np.float32)
    shape = tuple(y.shape)
    up = lambda a: torch.from_numpy(a.reshape(shape)).cuda()  # noqa: E731
    return fx, fy, fm, old, adv, ref, up(old), up(adv), up(ref)


@pytest.mark.parametrize("reduction", ["token_mean", "sequence_mean", "sum"])
@pytest.mark.parametrize("b,t,v,dtype", [s for s in ALL if s[2] in (2, 7, 255, 4099, 16391, 70001)])
@pytest.mark.parametrize("kl,ent", [(0.0, 0.0), (0.1, 0.0), (0.05, 0.02)])
def test_policy_loss(reduction, b, t, v, dtype, kl, ent):
    x, y, m = make(v, b, t, v, dtype, masked=t > 1)
    temp = 0.8
    inv_t = 1 / temp
    fx, fy, fm, old, adv, ref, old_t, adv_t, ref_t = policy_inputs(v, x, y, m, inv_t)
    scale = 64.0
    w = O.weights(fm, b, t, reduction, scale)
    loss, grad, size, _ = O.policy(fx, fy, old, adv, fm, ref, w, 0.2, 0.25, kl, ent, inv_t)
    lp, h = O.logprobs(fx, fy, fm, inv_t)
    more = dict(ref_logprobs=ref_t, eps_clip=0.2, eps_clip_high=0.25, kl_coef=kl, entropy_coef=ent, temperature=temp,
                reduction=reduction, scale=scale)
    off = 4 * float(logp_tol(lp, v).max()) + 2.0 ** -21      # of the ratio and of e^d, each a few roundings
    terms = np.abs(adv) * 2 + kl * 10 + ent * (1 + h)
    tol = mean_tol(w, terms * off) + 2.0 ** -23 * abs(loss) + 1e-12
    got = K().policy_loss_and_grad(x, y, old_t, adv_t, m, **more)
    close(got[0], loss, tol, "loss")
    close_grad(got[1], grad, size, v, off)
    close(got[2].reshape(-1), lp, logp_tol(lp, v))
    close(got[3].reshape(-1), h, 2 * row_tol(v) * (1 + np.abs(h)) + 1e-6)
    x.requires_grad_(True)
    out = K().policy_loss(x, y, old_t, adv_t, m, **more)
    close(out[0], loss, tol, "loss")
    close(out[1].reshape(-1), lp, logp_tol(lp, v))
    close(out[2].reshape(-1), h, 2 * row_tol(v) * (1 + np.abs(h)) + 1e-6)
    close_grad(torch.autograd.grad(out[0] * 3, x)[0], 3 * grad, 3 * size, v, off)
    with torch.no_grad():
        close(K().policy_loss(x, y, old_t, adv_t, m, **more)[0], loss, tol, "loss")


EDGES = [8, 9, 16, 17, 63, 65, 256, 257, 1023, 1024, 1025, 2047, 2048, 2049, 8192, 24575, 24576, 24577, 49151, 49152, 49153, 65535, 65536, 65537]


@pytest.mark.parametrize("v", EDGES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes_at_which_the_form_changes(v, dtype):
    """On both sides of each size at which rows are worked on in another way, 130 rows and 3: log-probabilities, entropy and the
    gradient of a policy loss that has all terms, from both forms of it."""
    for b, t in ((10, 13), (1, 3)):
        x, y, m = make(v + t, b, t, v, dtype)
        fx, fy, fm, old, adv, ref, old_t, adv_t, ref_t = policy_inputs(v, x, y, m, 1.0)
        w = O.weights(fm, b, t, "token_mean", 64.0)
        loss, grad, size, _ = O.policy(fx, fy, old, adv, fm, ref, w, 0.2, 0.2, 0.05, 0.02, 1.0)
        lp, h = O.logprobs(fx, fy, fm, 1.0)
        more = dict(ref_logprobs=ref_t, kl_coef=0.05, entropy_coef=0.02, scale=64.0)
        off = 4 * float(logp_tol(lp, v).max()) + 2.0 ** -21
        tol = mean_tol(w, (np.abs(adv) * 2 + 0.5 + 0.02 * (1 + h)) * off) + 2.0 ** -23 * abs(loss) + 1e-12
        got = K().policy_loss_and_grad(x, y, old_t, adv_t, m, **more)
        out = K().policy_loss(x.requires_grad_(True), y, old_t, adv_t, m, **more)
        for some in (got, (out[0], torch.autograd.grad(out[0], x)[0], out[1], out[2])):
            close(some[0], loss, tol, "loss")
            close_grad(some[1], grad, size, v, off)
            close(some[2].reshape(-1), lp, logp_tol(lp, v))
            close(some[3].reshape(-1), h, 2 * row_tol(v) * (1 + np.abs(h)) + 1e-6)


@pytest.mark.parametrize("shape", ["column", "vector", "expanded", "transposed", "half"])
def test_policy_advantages_of_other_layouts(shape):
    b, t, v = 3, 4, 301
    x, y, m = make(8, b, t, v, torch.float32)
    fx, fy, fm, old, adv, ref, old_t, adv_t, ref_t = policy_inputs(8, x, y, m, 1.0)
    per = torch.tensor([1.0, -0.5, 2.0], device="cuda")
    adv_t = {"column": per[:, None], "vector": per, "expanded": per[:, None].expand(b, t),
             "transposed": torch.arange(12.0, device="cuda").view(t, b).t(),
             "half": (torch.arange(12.0, device="cuda").view(b, t) - 4).half()}[shape]
    adv = f64(adv_t.reshape(b, -1).expand(b, t)).reshape(-1)
    w = O.weights(fm, b, t, "token_mean", 1.0)
    loss, grad, size, _ = O.policy(fx, fy, old, adv, fm, ref, w, 0.2, 0.2, 0.0, 0.0, 1.0)
    got = K().policy_loss_and_grad(x, y.int(), old_t, adv_t, m)
    off = 4 * float(logp_tol(old, v).max()) + 2.0 ** -21
    close(got[0], loss, mean_tol(w, 2 * np.abs(adv) * off) + 1e-7, "loss")
    close_grad(got[1], grad, size, v, off)
    assert torch.equal(K().policy_loss_and_grad(x, y, old_t, adv_t, m.to(torch.uint8))[1], got[1])


SEQS = [(1, 1), (1, 16), (1, 4000), (2, 1), (2, 15), (2, 17), (3, 33), (5, 64), (6, 255), (8, 500), (33, 7), (63, 65), (64, 16), (64, 64),
        (65, 3)]


@pytest.mark.parametrize("b,t,v", [(b, t, v) for v in (300, 2600, 21000) for b, t in SEQS if b * t * v < 3e7])
def test_means_over_sequences(b, t, v):
    """Every counted row's weight is 1 / (counted rows of its sequence * sequences with one): the gradient of the loss with
    respect to a row's log-probability, found at the token of a row of equal logits, where it is weight * (1 - 1/v)."""
    r = np.random.default_rng(b * 1000 + t)
    mask = r.random((b, t)) < r.choice([0.02, 0.5, 0.97], (b, 1))
    mask[0, -1] = True
    n = mask.sum(1)
    want = mask / np.maximum(n, 1)[:, None] / (n > 0).sum()
    x, m = torch.zeros(b, t, v, device="cuda"), torch.from_numpy(mask).cuda()
    y = torch.from_numpy(r.integers(0, v, (b, t))).cuda()
    one = torch.ones(b, t, device="cuda")
    old = one * -math.log(v)
    leaf = x.clone().requires_grad_(True)
    for sign, grad in ((-1, K().policy_loss_and_grad(x, y, old, one, m, reduction="sequence_mean")[1]),
                       (-1, torch.autograd.grad(K().policy_loss(leaf, y, old, one, m, reduction="sequence_mean")[0], leaf)[0]),
                       (-1, K().distillation_loss_and_grad(x, y[..., None], one[..., None], m, reduction="sequence_mean")[1]),
                       (-1, torch.autograd.grad(K().distillation_loss(leaf, y[..., None], one[..., None], m,
                                                                      reduction="sequence_mean")[0], leaf)[0])):
        got = sign * torch.take_along_dim(grad, y[..., None], 2)[..., 0] / (1 - 1 / v)
        close(got, want, want * (3 * row_tol(v) + 2.0 ** -20))


def test_many_rows_and_many_sequences():
    """More rows than workgroups, and masks counted in two launches."""
    for b, t, v in [(5000, 9, 33), (40000, 1, 5), (2, 20000, 9)]:
        x, y, m = make(6, b, t, v, torch.bfloat16)
        fx, fy, fm, old, adv, ref, old_t, adv_t, ref_t = policy_inputs(6, x, y, m, 1.0)
        off = 4 * float(logp_tol(old, v).max()) + 2.0 ** -21
        for reduction in ("token_mean", "sequence_mean", "sum"):
            w = O.weights(fm, b, t, reduction, 1.0)
            loss, grad, size, _ = O.policy(fx, fy, old, adv, fm, ref, w, 0.2, 0.2, 0.1, 0.0, 1.0)
            got = K().policy_loss_and_grad(x, y, old_t, adv_t, m, ref_logprobs=ref_t, kl_coef=0.1, reduction=reduction)
            close(got[0], loss, mean_tol(w, (2 * np.abs(adv) + 1) * off) + 2.0 ** -23 * abs(loss), "loss")
            close_grad(got[1], grad, size, v, off)


def test_nothing_counts():
    x, y, m = make(9, 2, 3, 50, torch.float32)
    m[:] = False
    z = torch.zeros(2, 3, device="cuda")
    for reduction in ("token_mean", "sequence_mean", "sum"):
        loss, grad, lp, h = K().policy_loss_and_grad(x, y, z, z, m, reduction=reduction)
        assert loss == 0 and (grad == 0).all() and (lp == 0).all() and (h == 0).all()
        loss, grad, each = K().distillation_loss_and_grad(x, y[..., None], z[..., None], m, reduction=reduction)
        assert loss == 0 and (grad == 0).all() and (each == 0).all()
    loss, grad, rewards = K().preference_loss_and_grad(x, y, torch.zeros(2, device="cuda"), m)
    assert abs(float(loss) - math.log(2)) < 2.0 ** -23 and (grad == 0).all() and (rewards == 0).all()


@pytest.mark.parametrize("shape", [(0, 3, 5), (2, 0, 5), (0, 5)])
def test_no_rows(shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    y = torch.zeros(shape[:-1], dtype=torch.int64, device="cuda")
    z = torch.zeros(shape[:-1], device="cuda")
    for m in (None, torch.ones(shape[:-1], dtype=torch.bool, device="cuda")):
        lp, h = K().token_logprobs(x, y, m)
        assert lp.shape == h.shape == y.shape
        assert torch.autograd.grad(lp.sum(), x)[0].shape == x.shape
        for reduction in ("token_mean", "sequence_mean", "sum"):
            loss = K().policy_loss(x, y, z, z, m, reduction=reduction)[0]
            assert loss == 0 and torch.autograd.grad(loss, x)[0].shape == x.shape
            assert K().policy_loss_and_grad(x, y, z, z, m, reduction=reduction)[0] == 0
            loss = K().distillation_loss(x, y[..., None], z[..., None], m, reduction=reduction)[0]
            assert loss == 0 and torch.autograd.grad(loss, x)[0].shape == x.shape
    if shape == (2, 0, 5):
        loss, grad, rewards = K().preference_loss_and_grad(x, y, torch.ones(2, device="cuda"))
        assert abs(float(loss) - math.log(2)) < 2.0 ** -23 and (rewards + 0.1).abs().max() < 1e-7


# ------------------------------------------------------------------------------------------ preference loss
@pytest.mark.parametrize("b,t,v,dtype", [(2, 1, 7, torch.float32), (2, 17, 2053, torch.float32), (6, 5, 255, torch.bfloat16),
                                         (4, 300, 64, torch.float16), (2, 3, 70001, torch.float32), (8, 2, 4099, torch.float16)])
@pytest.mark.parametrize("beta,smoothing", [(0.1, 0.0), (0.5, 0.1)])
def test_preference_loss(b, t, v, dtype, beta, smoothing):
    x, y, m = make(v + t, b, t, v, dtype)
    fx, fy, fm = flat(x, y, m)
    lp, _ = O.logprobs(fx, fy, fm, 1.0)
    r = np.random.default_rng(1)
    ref = (lp.reshape(b, t).sum(1) + 3 * r.standard_normal(b)).astype(np.float32)
    scale = 16.0
    loss, grad, size, rewards = O.preference(fx, fy, fm, ref, t, beta, smoothing, scale)
    ref_t = torch.from_numpy(ref).cuda()
    more = dict(beta=beta, label_smoothing=smoothing, scale=scale)
    got = K().preference_loss_and_grad(x, y, ref_t, m, **more)
    tol = beta * t * (row_tol(v) + float(np.abs(lp).max()) * 2.0 ** -22)      # of a reward, before its rounding
    close(got[2], rewards, tol + np.abs(rewards) * 2.0 ** -24, "rewards")
    close(got[0], loss, 2 * scale * tol + 2.0 ** -23 * abs(loss), "loss")
    close_grad(got[1], grad, size, v, 2 * tol)       # d sigmoid: at most 1/4 dz, relative to sigmoid at most dz
    x.requires_grad_(True)
    out = K().preference_loss(x, y, ref_t, m, **more)
    close(out[0], loss, 2 * scale * tol + 2.0 ** -23 * abs(loss), "loss")
    close(out[1], rewards, tol + np.abs(rewards) * 2.0 ** -24, "rewards")
    close_grad(torch.autograd.grad(out[0], x)[0], grad, size, v, 2 * tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,v", [(511, 50001), (2, 131072), (700, 900)])
def test_rewards_of_long_sequences(t, v, dtype):
    """A reward is a difference of sums of many log-probabilities, where a systematic error of theirs adds up: half a step
    of S (2^-24) is allowed for it, beside four times the spread of t independent errors of a step (2^-23)."""
    x, y, m = make(31, 4, t, v, dtype, masked=False)
    each = torch.stack([torch.log_softmax(q.double(), -1).gather(1, i[:, None])[:, 0] for q, i in zip(x, y)])
    ref = each.sum(1).float()
    want = each.sum(1) - ref.double()
    tol = t * 2.0 ** -24 + 4 * math.sqrt(t) * 2.0 ** -23
    for rewards in (K().preference_loss(x, y, ref, m, beta=1.0)[1], K().preference_loss_and_grad(x, y, ref, m, beta=1.0)[2]):
        close(rewards, f64(want), tol + 2.0 ** -24 * np.abs(f64(want)))


def test_preference_far_apart():
    """Rewards so far apart that a sigmoid is 0 or 1, and an impossible token."""
    x, y, _ = make(3, 4, 3, 90, torch.float32, masked=False)
    fx, fy, _ = flat(x, y, None)
    ref = torch.tensor([1e4, -1e4, -1e4, 1e4], device="cuda")
    loss, grad, size, rewards = O.preference(fx, fy, None, f64(ref), 3, 1.0, 0.0, 1.0)
    got = K().preference_loss_and_grad(x, y, ref, beta=1.0)
    close(got[0], loss, 1e-3, "loss")            # 1e4 * 2^-24 for each reward
    close_grad(got[1], grad, size, 90, 1e-3)
    x[2, 1, y[2, 1]] = -math.inf                 # a rejected sequence that cannot happen: the pair is decided
    loss, grad, rewards = K().preference_loss_and_grad(x, y, ref * 0, beta=1.0)
    assert math.isfinite(loss) and rewards[2] == -math.inf and (grad[0] == 0).all()


# ------------------------------------------------------------------------------------------ distillation
def teacher_of(seed, x, k, dtype):
    r = np.random.default_rng(seed)
    b, t, v = x.shape
    index = r.integers(0, v, (b, t, k))          # the same token twice, now and then
    if k > 2:
        index[..., -1] = index[..., 0]
        index[r.random(index.shape) < 0.15] = -1
        index[0, 0, :] = -1                      # a row without a teacher
    values = torch.from_numpy(np.sort(r.standard_normal((b, t, k)) * 2)[..., ::-1].copy()).to(dtype)
    if k > 4:
        values[..., 3] = -math.inf
    return torch.from_numpy(index).cuda(), values.cuda()


@pytest.mark.parametrize("b,t,v,dtype,k", [(1, 1, 1, torch.float32, 1), (2, 3, 7, torch.bfloat16, 5), (3, 4, 255, torch.float16, 64),
                                           (2, 3, 4099, torch.float32, 512), (3, 5, 16391, torch.bfloat16, 33),
                                           (1, 2, 70001, torch.float32, 100), (2, 2, 50001, torch.float16, 8),
                                           (1, 2, 300007, torch.bfloat16, 200)])
@pytest.mark.parametrize("temp,reduction", [(1.0, "token_mean"), (2.0, "sequence_mean"), (0.5, "sum")])
def test_distillation_loss(b, t, v, dtype, k, temp, reduction):
    x, _, m = make(v + k, b, t, v, dtype, masked=b > 1)
    index, values = teacher_of(k, x, k, TYPES[k % 3])
    fx = f64(x).reshape(-1, v)
    fm = None if m is None else m.cpu().numpy().reshape(-1)
    scale = 32.0
    w = O.weights(fm, b, t, reduction, scale)
    loss, grad, size, each = O.distillation(fx, index.cpu().numpy().reshape(-1, k), f64(values).reshape(-1, k), fm, w, 1 / temp)
    more = dict(temperature=temp, reduction=reduction, scale=scale)
    got = K().distillation_loss_and_grad(x, index, values, m, **more)
    # per entry q |ln p|: q to k + 8 roundings, ln p to logp_tol; |ln p| < 60 here
    tol = temp ** 2 * (row_tol(v) + 60 * ((k + 8) * 2.0 ** -24 + 2.0 ** -22))
    close(got[2].reshape(-1), each, tol + np.abs(each) * 2.0 ** -23, "token losses")
    close(got[0], loss, mean_tol(w, tol + np.abs(each) * 2.0 ** -22), "loss")
    close_grad(got[1], grad, size, v, (k + 8) * 2.0 ** -24)
    x.requires_grad_(True)
    out = K().distillation_loss(x, index.int(), values, m, **more)
    close(out[1].reshape(-1), each, tol + np.abs(each) * 2.0 ** -23, "token losses")
    close(out[0], loss, mean_tol(w, tol + np.abs(each) * 2.0 ** -22), "loss")
    close_grad(torch.autograd.grad(out[0], x)[0], grad, size, v, (k + 8) * 2.0 ** -24)


def test_distillation_bad_teacher_token():
    x, _, _ = make(5, 1, 3, 600, torch.bfloat16, masked=False)
    index = torch.tensor([[[1, 2], [600, 3], [5, 6]]], device="cuda")
    values = torch.ones(1, 3, 2, device="cuda")
    x.requires_grad_(True)
    loss, each = K().distillation_loss(x, index, values)
    assert torch.isnan(loss) and torch.isnan(each[0]).tolist() == [False, True, False]
    for grad in (K().distillation_loss_and_grad(x, index, values, reduction="sum")[1],
                 torch.autograd.grad(K().distillation_loss(x, index, values, reduction="sum")[0], x)[0]):
        assert torch.isnan(grad[0]).any(-1).tolist() == [False, True, False]


# ------------------------------------------------------------------------------------------ memory, streams, graphs
def all_three(x, y, m, out=None):
    """One call of each `_and_grad` form; the gradient of each in `out` if it is given (then it is copied)."""
    z = torch.full(y.shape, -2.0, device="cuda")
    keep = lambda r: tuple(t.clone() for t in r)  # noqa: E731
    index = torch.stack([y, (y + 1) % x.shape[-1]], -1)
    values = torch.stack([z, z - 1], -1)
    store = lambda: None if out is None else out()  # noqa: E731
    r = [keep(K().policy_loss_and_grad(x, y, z, z, m,
                                       ref_logprobs=z, kl_coef=0.1, out=store()))]
    return r + [keep(K().preference_loss_and_grad(x, y, z.sum(-1), m, out=store())),
                keep(K().distillation_loss_and_grad(x, index, values, m, out=store()))]


def same(a, b, exact=True):
    """The same bits; or, for rows that begin elsewhere relative to 16 bytes and are added up in another order, a result
    within two errors of a row and one rounding to the type."""
    if exact:
        assert torch.equal(a, b)
    else:
        a, b = a.double(), b.double()
        tol = 2 * (2.0 ** -24 + row_tol(200000)) * (1 + b.abs().max())
        step = 2.0 ** -7 * b.abs() if a.dim() == 3 else 0.0        # bfloat16's, the widest of the types
        assert ((a - b).abs() <= tol + step).all()


@pytest.mark.parametrize("v,dtype", [(5, torch.float32), (999, torch.float16), (4100, torch.bfloat16), (70001, torch.float32),
                                     (140001, torch.bfloat16)])
def test_gradient_in_place_and_in_other_memory(v, dtype):
    x, y, m = make(v, 4, 3, v, dtype)
    want = all_three(x, y, m)
    z = torch.full(y.shape, -2.0, device="cuda")
    pad = torch.full((4, 4, v + 3), 7.0, dtype=dtype, device="cuda")
    got = all_three(x, y, m, out=lambda: pad[:, 1:, 2:2 + v])
    for a, b in zip(want, got):
        for s, u in zip(a, b):
            assert torch.equal(s, u)
    assert (pad[:, 0] == 7).all() and (pad[..., :2] == 7).all() and (pad[..., -1] == 7).all()
    index = torch.stack([y, (y + 1) % v], -1)
    values = torch.stack([z, z - 1], -1)
    for k, fn in enumerate([lambda a: K().policy_loss_and_grad(a, y, z, z, m, ref_logprobs=z, kl_coef=0.1, out=a),
                            lambda a: K().preference_loss_and_grad(a, y, z.sum(-1), m, out=a),
                            lambda a: K().distillation_loss_and_grad(a, index, values, m, out=a)]):
        for view in (lambda f: f, lambda f: f[:, 1:, 2:2 + v]):
            a = view(torch.zeros((4, 3, v) if view(pad).shape == pad.shape else pad.shape, dtype=dtype, device="cuda"))
            a.copy_(x)
            r = fn(a)
            assert r[1].data_ptr() == a.data_ptr()
            for s, u in zip(want[k], r):
                same(s, u, exact=a.data_ptr() % 16 == x.data_ptr() % 16 and a.is_contiguous())


def test_overwritten_logits_are_noticed_by_autograd():
    x = torch.randn(2, 3, 20, device="cuda", requires_grad=True)
    logits = x * 1.0
    other = logits.exp()                 # exp keeps its result, square its argument
    square = logits.square()
    y, z = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, 3, device="cuda")
    K().policy_loss_and_grad(logits, y, z, z, out=logits)
    other.sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        square.sum().backward()


def calls(x, y, m):
    """The differentiable losses as functions of the logits."""
    z = torch.full(y.shape, -2.0, device="cuda")
    return [lambda a: K().token_logprobs(a, y, m)[0].sum(), lambda a: K().token_logprobs(a, y, m)[1].sum(),
            lambda a: K().policy_loss(a, y, z, z, m, ref_logprobs=z, kl_coef=0.1, entropy_coef=0.1)[0],
            lambda a: K().preference_loss(a, y, z.sum(-1), m)[0],
            lambda a: K().distillation_loss(a, y[..., None], z[..., None], m)[0]]


def test_autograd_corners():
    """Backward twice over a kept graph, a gradient of a gradient (refused, and only when it is asked for), logits changed
    in between (noticed), and saved tensors that leave the GPU in between."""
    x, y, m = make(15, 2, 5, 700, torch.float32)
    for fn in calls(x, y, m):
        a = x.clone().requires_grad_(True)
        loss = fn(a)
        one = torch.autograd.grad(loss, a, retain_graph=True)[0]
        two = torch.autograd.grad(loss * 2, a, create_graph=True)[0]
        assert torch.equal(one * 2, two.detach())
        with pytest.raises(RuntimeError, match="differentiated once"):
            two.sum().backward()
        b = x.clone().requires_grad_(True)
        c = b * 1.0
        loss = fn(c)
        c.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.autograd.graph.save_on_cpu():
            loss = fn(a)
        held = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]   # what was freed is written over
        assert torch.equal(torch.autograd.grad(loss, a)[0], one)
        del held
        with torch.inference_mode():
            assert torch.equal(fn(x), fn(x.clone()))
    with torch.inference_mode():
        a, z = x.clone(), torch.full(y.shape, -2.0, device="cuda")
        want = K().policy_loss_and_grad(x, y, z, z, m)[1]
        assert torch.equal(K().policy_loss_and_grad(a, y, z, z, m, out=a)[1], want) and torch.equal(a, want)


def test_gradients_on_a_side_stream():
    """A forward and a backward pass on a stream of its own, between work on the default stream."""
    x, y, m = make(16, 4, 30, 4099, torch.bfloat16)
    want = [torch.autograd.grad(fn(a), a)[0] for fn, a in ((f, x.clone().requires_grad_(True)) for f in calls(x, y, m))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [torch.autograd.grad(fn(a), a)[0] for fn, a in ((f, x.clone().requires_grad_(True)) for f in calls(x, y, m))]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16, torch.float16])
def test_other_types_beside_the_logits(dtype):
    x, y, m = make(17, 2, 4, 300, torch.float16)
    z = torch.linspace(-4, -1, 8, device="cuda").view(2, 4).to(dtype)
    a = K().policy_loss_and_grad(x, y, z, z, m, ref_logprobs=z, kl_coef=0.1)
    f = z.float()
    b = K().policy_loss_and_grad(x, y.int(), f, f.t().contiguous().t(), m.to(torch.uint8) * 7, ref_logprobs=f, kl_coef=0.1)
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    a, b = K().preference_loss_and_grad(x, y, z[:, 0], m), K().preference_loss_and_grad(x, y, f[:, 0], m)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


@pytest.mark.parametrize("v", [1, 6, 70, 500, 4099, 70001])
@pytest.mark.parametrize("temp", [1.0, 0.7])
def test_certain_tokens(v, temp):
    """All probability on one token: no log-probability above 0, no entropy below, in forward, loss and logging outputs."""
    r = np.random.default_rng(v)
    x = torch.full((4, 32, v), -math.inf)
    x[..., v // 2] = torch.from_numpy(20 * r.standard_normal((4, 32))).float()
    x, y = x.cuda(), torch.full((4, 32), v // 2).cuda()
    old, adv = torch.zeros(4, 32).cuda(), torch.ones(4, 32).cuda()
    for lp, ent in (K().token_logprobs(x, y, temperature=temp), K().policy_loss_and_grad(x, y, old, adv, temperature=temp)[2:],
                    K().policy_loss(x, y, old, adv, temperature=temp)[1:],
                    K().policy_loss_and_grad(x[:1, :1], y[:1, :1], old[:1, :1], adv[:1, :1], temperature=temp)[2:]):
        assert (lp <= 0).all() and (ent >= 0).all()
        assert lp.min() >= -row_tol(v) and ent.max() <= row_tol(v)


@pytest.mark.parametrize("dtype", TYPES)
def test_small_terms_of_long_rows_are_not_lost(dtype):
    """The mean error of ln p over 512 rows of 131072 logits with most of their terms far below the largest.  Added to
    S one by one, the small ones were lost: 6.5e-7.  At least 16 are added at once, so at most 1/16 of that is left: 4e-8;
    rounding ln p (below 64) is off by at most 2^-19 and by 2^-19 / sqrt 3 = 1.1e-6 in the square mean, 5e-8 in the mean of
    512, of which four are allowed."""
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = (2.5 * torch.randn(64, 8, 131072, generator=g, device="cuda")).to(dtype)
    y = torch.randint(0, 131072, (64, 8), generator=g, device="cuda")
    for entropy in (True, False):
        lp, _ = K().token_logprobs(x, y, temperature=0.5, entropy=entropy)
        want = torch.cat([torch.log_softmax(q.double() / 0.5, -1).gather(1, i[:, None])[:, 0][None] for q, i in zip(x, y)])
        assert abs((lp.double() - want).mean().item()) < 2.4e-7


def test_far_rows():
    """Offsets beyond 2^31 elements, in the logits and in the gradient."""
    v, far = 1003, (1 << 31) + 24
    x, y, m = make(12, 2, 3, v, torch.bfloat16, masked=False)
    want = K().policy_loss_and_grad(x, y, y.float() * -0.01, y.float() * 0.01)
    big = torch.empty(far + 4 * v, dtype=torch.bfloat16, device="cuda")
    view = big.as_strided((2, 3, v), (far, v, 1))
    view.copy_(x)
    once = K().policy_loss_and_grad(view, y, y.float() * -0.01, y.float() * 0.01)
    for a, b in zip(want, once):
        same(a, b, exact=False)
    got = K().policy_loss_and_grad(view, y, y.float() * -0.01, y.float() * 0.01, out=view)
    assert torch.equal(got[1], once[1]) and torch.equal(view, once[1])


def test_more_rows_than_a_launch():
    """Rows beyond the first 2^21 of a call, one in a million counted."""
    n, v = (1 << 21) + 3, 2049
    x = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    m = torch.zeros(n, dtype=torch.bool, device="cuda")
    at = torch.tensor([0, (1 << 21) - 1, 1 << 21, n - 1], device="cuda")
    m[at] = True
    x[at] = torch.randn(4, v, device="cuda").to(x.dtype)
    y = torch.arange(n, device="cuda") % v
    lp, h = K().token_logprobs(x, y, m)
    want, ent = O.logprobs(f64(x[at]), y[at].cpu().numpy(), None, 1.0)
    close(lp[at], want, logp_tol(want, v))
    close(h[at], ent, 2 * row_tol(v) * (1 + ent) + 1e-6)
    assert int((lp != 0).sum()) == 4
    z = torch.zeros(n, device="cuda")
    got = K().policy_loss_and_grad(x, y, lp, z + 1.0, m, out=x)
    assert abs(float(got[0]) + 1) < 1e-5 and int((got[1] != 0).any(-1).sum()) == 4


def test_same_bits_every_time_and_on_another_stream():
    for v, dtype in [(1000, torch.float32), (33000, torch.bfloat16)]:
        x, y, m = make(13, 4, 40, v, dtype)
        want = all_three(x, y, m)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one = all_three(x, y, m)
        two = all_three(x, y, m)
        torch.cuda.synchronize()
        for a, b, c in zip(want, one, two):
            for p, q, r in zip(a, b, c):
                assert torch.equal(p, q) and torch.equal(p, r)


def test_two_threads_at_once():
    """Calls from two threads, each on a stream of its own, whose workspaces and host code run at the same time."""
    import threading
    sets = [make(40 + k, 4, 40, v, dtype) for k, (v, dtype) in enumerate([(33000, torch.bfloat16), (140001, torch.float16)])]
    wants = [all_three(*s) for s in sets]
    torch.cuda.synchronize()
    gots = [[], []]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                gots[k].append(all_three(*sets[k]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for want, got in zip(wants, gots):
        assert len(got) == 10
        for one in got:
            for a, b in zip(want, one):
                for p, q in zip(a, b):
                    assert torch.equal(p, q)


def test_captured_graphs():
    """Each form captured and replayed with new inputs, eager work between; two graphs replayed on two streams."""
    v = 3001
    x, y, m = make(14, 4, 6, v, torch.bfloat16)
    z = torch.full(y.shape, -2.0, device="cuda")

    def work(x, y, m, z):
        leaf = x.detach().requires_grad_(True)
        loss, lp, h = K().policy_loss(leaf, y, z, z, m, ref_logprobs=z, kl_coef=0.1, entropy_coef=0.01, reduction="sequence_mean")
        grad = torch.autograd.grad(loss, leaf)[0]
        return [loss, lp, h, grad, *K().policy_loss_and_grad(x, y, z, z, m),
                *K().preference_loss_and_grad(x, y, z.sum(-1), m),
                *K().distillation_loss_and_grad(x, y[..., None], z[..., None], m), *K().token_logprobs(x, y, m)]

    held = []
    for _ in range(2):
        args = [t.clone() for t in (x, y, m, z)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(*args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work(*args)
        held.append((args, graph, outs, torch.cuda.Stream()))
    for step in range(3):
        wants = []
        for k, (args, graph, outs, stream) in enumerate(held):
            nx, ny, nm = make(20 + 2 * step + k, 4, 6, v, torch.bfloat16)
            for dst, src in zip(args, (nx, ny, nm, z - step)):
                dst.copy_(src)
            wants.append([t.clone() for t in work(*args)])
        torch.cuda.synchronize()
        for args, graph, outs, stream in held:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for want, (args, graph, outs, stream) in zip(wants, held):
            for a, b in zip(want, outs):
                assert torch.equal(a, b), step


def test_a_training_step_with_all_of_them():
    """A small token policy: log-probabilities of a rollout, then its update on the sum of the losses, by backward() and
    by the gradients given together; the gradients agree with autograd in float64 on the CPU."""
    torch.manual_seed(0)
    b, t, v, d = 4, 6, 517, 16
    w0, hid = torch.randn(v, d) * 0.3, torch.randn(b, t, d)
    tok = torch.randint(0, v, (b, t))
    mask = torch.rand(b, t) < 0.8
    adv, index, teach = torch.randn(b, 1), torch.randint(0, v, (b, t, 3)), torch.randn(b, t, 3)

    def cpu():
        w = w0.double().requires_grad_(True)
        logp = torch.log_softmax(hid.double() @ w.T, -1)
        at = logp.gather(2, tok[..., None])[..., 0] * mask
        old, ref = at.detach() - 0.1, at.detach() + 0.2
        r = (at - old).exp()
        n = mask.sum()
        k = ref - at
        pol = ((-torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv) + 0.1 * (k.exp() - k - 1)) * mask).sum() / n
        ent = (-(logp.exp() * logp).sum(-1) * mask).sum() / n
        rew = 0.1 * (at.sum(1) - (at.detach().sum(1) - torch.tensor([1.0, 2.0, 3.0, 5.0])))
        pre = -torch.nn.functional.logsigmoid(rew[:2] - rew[2:]).mean()
        q = torch.softmax(teach.double(), -1)
        dis = ((q * (q.log() - logp.gather(2, index))).sum(-1) * mask).sum() / n
        loss = pol - 0.01 * ent + pre + dis
        return loss.detach(), torch.autograd.grad(loss, w)[0], old, ref, at.detach().sum(1) - torch.tensor([1.0, 2.0, 3.0, 5.0])

    loss, grad, old, ref, sums = cpu()
    g = lambda a: a.cuda().float() if a.is_floating_point() else a.cuda()  # noqa: E731
    w = g(w0).requires_grad_(True)
    logits = torch.nn.functional.linear(g(hid), w)
    with torch.no_grad():
        lp, _ = K().token_logprobs(logits, g(tok), g(mask), entropy=False)
    assert (lp.cpu() - (old + 0.1) * mask).abs().max() < 1e-4
    args = (g(tok), g(old), g(adv), g(mask))
    pol, _, _ = K().policy_loss(logits, *args, ref_logprobs=g(ref), kl_coef=0.1, entropy_coef=0.01)
    pre, _ = K().preference_loss(logits, g(tok), g(sums), g(mask))
    dis, _ = K().distillation_loss(logits, g(index), g(teach), g(mask))
    got = torch.autograd.grad(pol + pre + dis, w, retain_graph=True)[0]
    # logits of 16 products in fp32 and gradients of 24 rows added in fp32: 1e-5 of the largest entry is 80 roundings
    assert (got.cpu() - grad).abs().max() < 1e-5 * grad.abs().max() and abs(float((pol + pre + dis).detach()) - float(loss)) < 1e-5
    total = K().policy_loss_and_grad(logits, *args, ref_logprobs=g(ref), kl_coef=0.1, entropy_coef=0.01)[1] \
        + K().preference_loss_and_grad(logits, g(tok), g(sums), g(mask))[1] \
        + K().distillation_loss_and_grad(logits, g(index), g(teach), g(mask))[1]
    assert (torch.autograd.grad(logits, w, total)[0].cpu() - grad).abs().max() < 1e-5 * grad.abs().max()


def test_the_gradient_takes_the_logits_place():
    """A model's step as the documentation shows it: the loss's gradient over the logits, a view, and backward from there."""
    torch.manual_seed(1)
    ids, mask = torch.randint(0, 901, (3, 9)).cuda(), torch.rand(3, 8).cuda() < 0.8
    model = torch.nn.Sequential(torch.nn.Embedding(901, 32), torch.nn.Tanh(), torch.nn.Linear(32, 901)).cuda()
    advantages = torch.randn(3, device="cuda")
    grads = []
    for in_place in (False, True):
        model.zero_grad()
        logits = model(ids)[:, :-1]
        with torch.no_grad():
            old = K().token_logprobs(logits, ids[:, 1:], mask)[0] - 0.05
        if in_place:
            logits.backward(K().policy_loss_and_grad(logits, ids[:, 1:], old, advantages, mask, out=logits.detach())[1])
        else:
            K().policy_loss(logits, ids[:, 1:], old, advantages, mask)[0].backward()
        grads.append([p.grad.clone() for p in model.parameters()])
    for a, b in zip(*grads):   # two forms of the same arithmetic: 2^-20 of the largest entry
        assert a.abs().max() > 0 and (a - b).abs().max() <= 2.0 ** -20 * a.abs().max()


@pytest.mark.parametrize("v", [6, 900])
def test_gradients_are_the_differences_of_the_losses(v):
    x, y, m = make(30, 2, 3, v, torch.float32)
    z = K().token_logprobs(x, y, m)[0] - 0.05
    index, values = y[..., None], z[..., None]
    fns = [lambda a: K().policy_loss(a, y, z, z, m, ref_logprobs=z + 0.5, kl_coef=0.1, entropy_coef=0.1, reduction="sum")[0],
           lambda a: K().preference_loss(a, y, z.sum(-1), m, beta=0.5)[0],
           lambda a: K().distillation_loss(a, index, values, m, reduction="sum")[0]]
    r = torch.Generator(device="cuda").manual_seed(1)
    way = torch.randn(x.shape, generator=r, device="cuda")
    for fn in fns:
        a = x.clone().requires_grad_(True)
        slope = (torch.autograd.grad(fn(a), a)[0].double() * way).sum()
        h = 2.0 ** -7
        diff = (fn(x + h * way).double() - fn(x - h * way).double()) / (2 * h)
        # h^2 / 6 of a third derivative of order |way|^3 ~ 10 per counted row, and 2^-24 of the loss / h
        assert abs(float(slope - diff)) < 2e-3 * (1 + abs(float(slope))), (float(slope), float(diff))
