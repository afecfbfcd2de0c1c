"""CPU restatement in float64 numpy of the losses over a large vocabulary (ppo_amd.tokens), from their formulas.

Rows are flat: logits [n, V], everything else [n]; gradients are those with respect to the logits.  Each function
also returns ``size``, per logit the sum of the magnitudes of the terms its gradient is made of, which is what a
rounding error of the terms is relative to."""
import numpy as np


def softmax(logits, inv_t):
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        x = np.asarray(logits, np.float64) * inv_t
        m = x.max(-1, keepdims=True)
        e = np.exp(x - m)
        s = e.sum(-1, keepdims=True)
        return e / s, x - m - np.log(s)


def xlogx(p, logp):
    """p ln p with 0 ln 0 = 0."""
    return np.where(p == 0, 0.0, p * np.where(p == 0, 0.0, logp))


def logprobs(logits, tokens, mask, inv_t):
    p, logp = softmax(logits, inv_t)
    n = np.arange(len(tokens))
    on = np.ones(len(tokens), bool) if mask is None else np.asarray(mask, bool)
    at = np.where(on, logp[n, np.where(on, tokens, 0)], 0.0)
    ent = np.where(on, -xlogx(p, logp).sum(-1), 0.0)
    return at, ent


def logits_grad(logits, tokens, mask, inv_t, g_lp, g_h):
    p, logp = softmax(logits, inv_t)
    on = np.ones(len(tokens), bool) if mask is None else np.asarray(mask, bool)
    at, ent = logprobs(logits, tokens, mask, inv_t)
    one = np.zeros_like(p)
    one[np.arange(len(tokens)), np.where(on, tokens, 0)] = 1.0
    g_lp, g_h = np.asarray(g_lp, np.float64)[:, None], np.asarray(g_h, np.float64)[:, None]
    plnp = xlogx(p, logp)
    grad = inv_t * (g_lp * (one - p) - g_h * (plnp + p * ent[:, None]))
    size = inv_t * (np.abs(g_lp) * (one + p) + np.abs(g_h) * (np.abs(plnp) + p * (np.abs(ent[:, None]))))
    return np.where(on[:, None], grad, 0.0), np.where(on[:, None], size, 0.0)


def weights(mask, n_seq, n_tok, reduction, scale):
    m = np.ones(n_seq * n_tok) if mask is None else np.asarray(mask, np.float64).reshape(-1)
    if reduction == "sum":
        return m * scale
    if reduction == "token_mean":
        return m * scale / max(1.0, m.sum())
    per = m.reshape(n_seq, n_tok).sum(1)
    return m * scale / np.repeat(np.maximum(per, 1.0), n_tok) / max(1, int((per > 0).sum()))


def policy(logits, tokens, old, adv, mask, ref, w, lo, hi, kl, ent_coef, inv_t):
    """-> loss, grad, size, dloss/dlogprob; w as weights() gives it."""
    at, ent = logprobs(logits, tokens, mask, inv_t)
    on = w != 0 if mask is None else np.asarray(mask, bool)
    old, adv = np.where(on, old, 0.0), np.where(on, adv, 0.0)
    r = np.exp(at - old)
    s1, s2 = r * adv, np.clip(r, 1.0 - lo, 1.0 + hi) * adv
    each = -np.minimum(s1, s2)
    g = np.where(s1 <= s2, -s1, 0.0)
    size = np.abs(s1)
    if kl:
        d = np.where(on, ref, 0.0) - at
        each = each + kl * (np.expm1(d) - d)
        g = g - kl * np.expm1(d)
        size = size + kl * np.exp(d)     # e^d - 1 is off by e^d times the error of d, also where d is 0
    each = each - ent_coef * ent
    w = np.where(on, w, 0.0)
    grad, gsize = logits_grad(logits, tokens, mask, inv_t, w * g, -w * ent_coef)
    wide = logits_grad(logits, tokens, mask, inv_t, w * np.maximum(size, np.abs(g)), w * ent_coef)[1]
    return float((w * np.where(on, each, 0.0)).sum()), grad, np.maximum(gsize, wide), w * g


def preference(logits, tokens, mask, ref, n_tok, beta, smoothing, scale):
    """-> loss, grad, size, rewards"""
    at, _ = logprobs(logits, tokens, mask, 1.0)
    rewards = beta * (at.reshape(-1, n_tok).sum(1) - ref)
    pairs = len(rewards) // 2
    z = rewards[:pairs] - rewards[pairs:]
    loss = scale * np.mean((1 - smoothing) * np.logaddexp(0, -z) + smoothing * np.logaddexp(0, z))
    sig = np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))
    gz = scale * beta * (sig - (1 - smoothing)) / pairs
    g = np.repeat(np.concatenate([gz, -gz]), n_tok)
    grad, size = logits_grad(logits, tokens, mask, 1.0, g, 0 * g)
    return float(loss), grad, size, rewards


def distillation(logits, index, teacher, mask, w, inv_t):
    """-> loss, grad, size, token losses; index [n, K], negative: padding"""
    p, logp = softmax(logits, inv_t)
    n, on = len(index), np.ones(len(index), bool) if mask is None else np.asarray(mask, bool)
    there = index >= 0
    t = np.where(there, np.asarray(teacher, np.float64) * inv_t, -np.inf)
    some = there.any(1)
    t[~some] = 0.0
    e = np.exp(t - t.max(1, keepdims=True)) * there
    q = e / np.where(some, e.sum(1), 1.0)[:, None]
    logq = np.log(np.where(q > 0, q, 1.0))
    at = logp[np.arange(n)[:, None], np.where(there, index, 0)]
    each = np.where(q > 0, q * (logq - np.where(q > 0, at, 0.0)), 0.0).sum(1) / inv_t ** 2
    each = np.where(on & some, each, 0.0)
    w = np.where(on & some, w, 0.0)
    mass = np.zeros_like(p)
    np.add.at(mass, (np.arange(n)[:, None].repeat(index.shape[1], 1), np.where(there, index, 0)), q)
    used = w != 0
    grad = np.where(used[:, None], w[:, None] / inv_t * (p - mass), 0.0)
    size = np.where(used[:, None], np.abs(w[:, None]) / inv_t * (p + mass), 0.0)
    return float((w * each).sum()), grad, size, each
