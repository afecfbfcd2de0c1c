"""Operators for policies over a large vocabulary (ppo_amd.tokens), as cases to be measured: their inputs, their
plain forms, the calls a user makes of them, the work they cannot do without and their values in 64 bits.

  logprobs      log-probability of given tokens and entropy: forward, or with gradients of both coming in
  policy        clipped surrogate with a KL term and an entropy term, and its gradient with respect to the logits
  preference    loss on pairs of a preferred and a rejected sequence, and its gradient
  distillation  divergence from a teacher's top logits, and its gradient

"form" says how the gradient is asked for: "forward" is the call without one, "autograd" the differentiable call
and its backward pass, "together" the call that gives loss and gradient at once.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS_CLIP = 0.2


def case_of(name, op, form, dtype, seqs, toks, vocab, **more):
    c = {"name": name, "op": op, "form": form, "dtype": dtype, "seqs": seqs, "toks": toks, "vocab": vocab,
         "masked": True,       # a mask of counted tokens is given; without it all of them count
         "shifted": False,     # logits are full[:, :-1]: the last position predicts nothing
         "banned": False,      # a range of the vocabulary is ruled out with -inf
         "temperature": 1.0, "reduction": "token_mean", "entropy": True, "kl_coef": 0.0, "entropy_coef": 0.0,
         "per_sequence": False,   # one advantage for each sequence
         "scale": 1024.0 if dtype == "float16" else 1.0,      # of loss and gradient, for what 16 bits can hold
         "top": 0}
    c.update(more)
    return c


def listed():
    return [
        # a sampler reports the log-probability of the one token that it has just drawn
        case_of("logprobs one token", "logprobs", "forward", "bfloat16", 1, 1, 131072, masked=False),
        # the behaviour policy's log-probabilities over a batch of finished rollouts, a vocabulary of odd size
        case_of("logprobs rollouts", "logprobs", "forward", "bfloat16", 8, 1023, 50001, shifted=True),
        # a reference policy in 32 bits over a very large vocabulary, log-probabilities only
        case_of("logprobs wide", "logprobs", "forward", "float32", 2, 64, 262144, entropy=False, masked=False),
        # a loss of the caller's own on log-probabilities and entropy, small odd sizes
        case_of("logprobs train", "logprobs", "autograd", "float32", 4, 129, 8191, banned=True),
        # one update of a small task: latency
        case_of("policy small", "policy", "together", "float32", 4, 16, 1000, kl_coef=0.05, entropy_coef=0.01),
        # an update step written with backward(), a group of answers with one advantage each
        case_of("policy groups", "policy", "autograd", "float16", 8, 255, 32768, kl_coef=0.04, entropy_coef=0.01,
                reduction="sequence_mean", per_sequence=True, temperature=0.7),
        # the same for long answers of a large policy, loss and gradient at once
        case_of("policy large", "policy", "together", "bfloat16", 4, 1024, 131072, kl_coef=0.05),
        # one short pair
        case_of("preference one pair", "preference", "autograd", "float32", 2, 17, 2053),
        # four pairs of long answers, a vocabulary of odd size
        case_of("preference pairs", "preference", "together", "bfloat16", 8, 511, 50001, shifted=True),
        # a single token distilled
        case_of("distillation one token", "distillation", "together", "float32", 1, 1, 4099, top=8, masked=False),
        # a student trained with backward() at a raised temperature
        case_of("distillation warm", "distillation", "autograd", "float16", 4, 250, 32000, top=50, temperature=2.0,
                reduction="sequence_mean"),
        # long sequences of a large student, loss and gradient at once
        case_of("distillation large", "distillation", "together", "bfloat16", 4, 512, 131072, top=64),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["logprobs", "policy", "policy", "preference", "distillation"])
    form = rng.choice(["forward", "forward", "autograd"] if op == "logprobs" else ["autograd", "together"])
    vocab = log(300, 262144)
    rows = log(1, min(8192, (1 << 28) // vocab))
    seqs = min(log(1, 64), rows)
    if op == "preference":
        seqs = 2 * max(1, seqs // 2)
    toks = max(1, rows // seqs)
    return {k: v for k, v in case_of(
        "", op, form, rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), seqs, toks, vocab,
        masked=rng.random() < 0.7, shifted=rng.random() < 0.3, banned=rng.random() < 0.3,
        temperature=1.0 if op == "preference" else rng.choice([1.0, 1.0, 0.7, 1.3, 2.0]),
        reduction=rng.choice(["token_mean", "sequence_mean", "sum"]), entropy=rng.random() < 0.6,
        kl_coef=rng.choice([0.0, 0.04]), entropy_coef=rng.choice([0.0, 0.01]), per_sequence=rng.random() < 0.5,
        top=rng.choice([1, 5, 16, 33, 64, 100]) if op == "distillation" else 0).items() if k != "name"}


def lengths(case):
    """How many tokens of each sequence count: ragged, the longest whole, one empty where there are three or more."""
    b, t = case["seqs"], case["toks"]
    if not case["masked"]:
        return [t] * b
    r = random.Random(b * 1000003 + t)
    got = [t] + [r.randint((t + 1) // 2, t) for _ in range(b - 1)]
    if b >= 3 and case["op"] != "preference":
        got[-1] = 0
    return got


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed) * 7919 + 17)
    b, t, v = case["seqs"], case["toks"], case["vocab"]
    inv = 1.0 / case["temperature"]
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=g, device=dev)  # noqa: E731
    full = torch.empty((b, t + (1 if case["shifted"] else 0), v), dtype=DTYPES[case["dtype"]], device=dev)
    full.normal_(0.0, 2.5, generator=g)
    logits = full[:, :t]
    # tokens avoid the ruled out range; their logits are such that they are likely ones, as sampled tokens are
    lo, many = v // 3, (max(1, v // 50) if case["banned"] else 0)
    if many:
        logits[..., lo:lo + many] = -math.inf
    k = max(1, case["top"])
    tokens = torch.randint(0, v - many - k * 2, (b, t, 1), generator=g, device=dev)
    steps = 1 + (uniform(b, t, k) < 0.3).long()
    tokens = tokens + steps.cumsum(-1) - steps[..., :1]     # k different tokens of each row
    tokens = tokens + many * (tokens >= lo).long()
    near = math.log(v) + 3.1 - 2.0 * normal(b, t, k).abs() - 0.05 * torch.arange(k, device=dev)
    logits.scatter_(2, tokens, near.to(logits.dtype))
    s = {"case": case, "logits": logits}
    if case["masked"]:
        n = torch.tensor(lengths(case), device=dev)[torch.randperm(b, generator=g, device=dev)]
        begin = (uniform(b) * (t - n + 1)).long().clamp_(max=t)
        at = torch.arange(t, device=dev)
        s["mask"] = (at >= begin[:, None]) & (at < (begin + n)[:, None])
    else:
        s["mask"] = None
    if case["op"] == "distillation":
        s["tokens"] = torch.where(uniform(b, t, k) < 0.05, -1, tokens)     # a teacher that gave fewer than k
        s["tokens"][..., 0] = tokens[..., 0]
        s["teacher"] = (near + 0.7 * normal(b, t, k)).sort(-1, descending=True).values.to(logits.dtype)
        return s
    s["tokens"] = tokens[..., 0].contiguous()
    if case["op"] == "logprobs":
        size = case["scale"] / (b * t)
        s["g_logprobs"], s["g_entropy"] = size * normal(b, t), 0.01 * size * normal(b, t)
        return s
    logp = torch.stack([torch.log_softmax(x.float() * inv, -1).gather(-1, y[:, None])[:, 0]
                        for x, y in zip(logits, s["tokens"])])
    if case["op"] == "preference":
        m = torch.ones_like(logp) if s["mask"] is None else s["mask"].float()
        s["ref"] = (logp.double() * m).sum(-1).float() + 4.0 * normal(b)
        return s
    # the policy has moved a little from the one that acted; no ratio lies on an edge of the clip range, where
    # the last bit of a log-probability would decide whether there is a gradient
    d = 0.15 * normal(b, t)
    for edge in (1.0 - EPS_CLIP, 1.0 + EPS_CLIP):
        d = torch.where((d.exp() - edge).abs() < 2e-3, d + 0.02, d)
    s["old"] = logp - d
    s["ref"] = logp + 0.3 * normal(b, t)
    s["advantages"] = normal(b, 1).expand(b, t) if case["per_sequence"] else normal(b, t)
    return s


# ------------------------------------------------------------------------------------------ the framework's calls
def run_own(s):
    from ppo_amd import tokens
    c, x = s["case"], s["logits"]
    if c["form"] == "autograd":
        x = x.detach().requires_grad_(True)
    if c["op"] == "logprobs":
        logp, ent = tokens.token_logprobs(x, s["tokens"], s["mask"], temperature=c["temperature"], entropy=c["entropy"])
        if c["form"] == "forward":
            return {"logprobs": logp, "entropy": ent}
        outs, seeds = ([logp, ent], [s["g_logprobs"], s["g_entropy"]]) if c["entropy"] else ([logp], [s["g_logprobs"]])
        return {"logprobs": logp, "entropy": ent, "grad": torch.autograd.grad(outs, [x], seeds)[0]}
    if c["op"] == "policy":
        more = dict(ref_logprobs=s["ref"] if c["kl_coef"] else None, eps_clip=EPS_CLIP, kl_coef=c["kl_coef"],
                    entropy_coef=c["entropy_coef"], temperature=c["temperature"], reduction=c["reduction"], scale=c["scale"])
        args = (x, s["tokens"], s["old"], s["advantages"], s["mask"])
        if c["form"] == "together":
            loss, grad, logp, ent = tokens.policy_loss_and_grad(*args, **more)
        else:
            loss, logp, ent = tokens.policy_loss(*args, **more)
            grad = torch.autograd.grad(loss, x)[0]
        return {"loss": loss, "grad": grad, "logprobs": logp, "entropy": ent}
    if c["op"] == "preference":
        args = (x, s["tokens"], s["ref"], s["mask"])
        more = dict(beta=0.1, label_smoothing=0.05, scale=c["scale"])
        if c["form"] == "together":
            loss, grad, rewards = tokens.preference_loss_and_grad(*args, **more)
        else:
            loss, rewards = tokens.preference_loss(*args, **more)
            grad = torch.autograd.grad(loss, x)[0]
        return {"loss": loss, "grad": grad, "rewards": rewards}
    args = (x, s["tokens"], s["teacher"], s["mask"])
    more = dict(temperature=c["temperature"], reduction=c["reduction"], scale=c["scale"])
    if c["form"] == "together":
        loss, grad, each = tokens.distillation_loss_and_grad(*args, **more)
    else:
        loss, each = tokens.distillation_loss(*args, **more)
        grad = torch.autograd.grad(loss, x)[0]
    return {"loss": loss, "grad": grad, "token_losses": each}


# ------------------------------------------------------------------------------------------ the plain forms
def plain_softmax(x):
    """exp(x - max) / sum and the logarithm of it, in 32 bits."""
    m = x.max(-1, keepdim=True).values
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    return e / total, x - m - total.log()


def plain_entropy(p, logp):
    return -torch.where(p > 0, p * logp, 0.0).sum(-1)


def plain_weights(case, mask, like):
    m = torch.ones_like(like) if mask is None else mask.float()
    if case["reduction"] == "sum":
        return m * case["scale"]
    if case["reduction"] == "token_mean":
        return m * case["scale"] / m.sum().clamp(min=1.0)
    n = m.sum(-1, keepdim=True)
    return m * case["scale"] / n.clamp(min=1.0) / (n > 0).sum().clamp(min=1)


def plain_grad(c, p, logp, ent, tokens, g_logp, g_ent, dtype):
    """The gradient with respect to the logits from those with respect to the tokens' log-probabilities and the entropy."""
    g = -p * g_logp[..., None]
    if g_ent is not None:
        g = g - torch.where(p > 0, p * (logp + ent[..., None]), 0.0) * g_ent[..., None]
    g.scatter_add_(2, tokens[..., None], g_logp[..., None])
    return (g / c["temperature"]).to(dtype)


def run_plain(s):
    c, mask = s["case"], s["mask"]
    dtype = s["logits"].dtype
    p, logp = plain_softmax(s["logits"].float() / c["temperature"])
    if c["op"] == "distillation":
        return plain_distillation(s, c, p, logp, mask, dtype)
    counted = 1.0 if mask is None else mask.float()
    at = logp.gather(2, s["tokens"][..., None])[..., 0] * counted
    if c["op"] == "preference":
        rewards = 0.1 * (at.double().sum(-1) - s["ref"].double())
        half = c["seqs"] // 2
        z = rewards[:half] - rewards[half:]
        soft = lambda u: u.clamp(min=0.0) + (1.0 + (-u.abs()).exp()).log()  # noqa: E731   ln(1 + e^u)
        loss = c["scale"] * (0.95 * soft(-z) + 0.05 * soft(z)).mean()
        gz = 0.1 * c["scale"] * (1.0 / (1.0 + (-z).exp()) - 0.95) / half
        g = torch.cat([gz, -gz]).float()[:, None].expand_as(at) * counted
        return {"loss": loss.float(), "grad": plain_grad(c, p, logp, None, s["tokens"], g, None, dtype),
                "rewards": rewards.float()}
    ent = plain_entropy(p, logp) * counted if c["op"] == "policy" or c["entropy"] else None
    if c["op"] == "logprobs":
        if c["form"] == "forward":
            return {"logprobs": at, "entropy": ent}
        g_ent = s["g_entropy"] * counted if c["entropy"] else None
        return {"logprobs": at, "entropy": ent,
                "grad": plain_grad(c, p, logp, ent, s["tokens"], s["g_logprobs"] * counted, g_ent, dtype)}
    w, a = plain_weights(c, mask, at), s["advantages"]
    r = (at - s["old"]).exp()
    inside = r.clamp(1.0 - EPS_CLIP, 1.0 + EPS_CLIP)
    active = (r * a <= inside * a).float()
    each = -torch.minimum(r * a, inside * a)
    g = -active * r * a
    if c["kl_coef"]:
        d = (s["ref"] - at).double()
        each = each + c["kl_coef"] * (d.exp() - d - 1.0).float()
        g = g + c["kl_coef"] * (1.0 - d.exp()).float()
    g_ent = None
    if c["entropy_coef"]:
        each = each - c["entropy_coef"] * ent
        g_ent = -c["entropy_coef"] * w
    return {"loss": (w * each).double().sum().float(), "logprobs": at, "entropy": ent,
            "grad": plain_grad(c, p, logp, ent, s["tokens"], w * g, g_ent, dtype)}


def plain_distillation(s, c, p, logp, mask, dtype):
    there = s["tokens"] >= 0
    at = s["tokens"].clamp(min=0)
    q, logq = plain_softmax(torch.where(there, s["teacher"].float() / c["temperature"], -math.inf))
    each = c["temperature"] ** 2 * torch.where(q > 0, q * (logq - logp.gather(2, at)), 0.0).sum(-1)
    w = plain_weights(c, mask, each)
    each = each * (1.0 if mask is None else mask.float())
    g = (p * (w * c["temperature"])[..., None]).scatter_add_(2, at, -q * (w * c["temperature"])[..., None])
    return {"loss": (w * each).double().sum().float(), "grad": g.to(dtype), "token_losses": each}


def run(state):
    return run_own(state) if own else run_plain(state)


# ------------------------------------------------------------------------------------------ work and values in 64 bits
def work(case):
    n, total = sum(lengths(case)), case["seqs"] * case["toks"]
    size = BYTES[case["dtype"]]
    small = total * {"logprobs": 16, "policy": 28, "preference": 8, "distillation": 4 + (8 + size) * case["top"]}[case["op"]]
    read = n * case["vocab"] * size
    written = 0 if case["form"] == "forward" else total * case["vocab"] * size
    return {"bytes": read + written + small, "flops": n * case["vocab"] * (5 if case["form"] == "forward" else 10)}


def exact(case, seed):
    s = prepare(case, seed)
    x = s["logits"].double().requires_grad_(case["form"] != "forward")
    logp = torch.nn.functional.log_softmax(x / case["temperature"], -1)
    b, t = case["seqs"], case["toks"]
    m = torch.ones((b, t), dtype=torch.float64, device=x.device) if s["mask"] is None else s["mask"].double()
    if case["reduction"] == "sum":
        w = m
    elif case["reduction"] == "token_mean":
        w = m / max(1.0, m.sum().item())
    else:
        n = m.sum(1, keepdim=True)
        w = m / torch.where(n > 0, n, 1.0) / max(1, int((n > 0).sum()))
    w = w * case["scale"]
    out = {}
    if case["op"] == "distillation":
        q = torch.softmax((s["teacher"].double() / case["temperature"]).masked_fill(s["tokens"] < 0, -math.inf), -1)
        picked = torch.take_along_dim(logp, s["tokens"].clamp(min=0), 2).masked_fill(s["tokens"] < 0, 0.0)
        each = case["temperature"] ** 2 * (-torch.special.entr(q).sum(-1) - (q * picked).sum(-1)) * m
        loss = (w * each).sum()
        out = {"loss": loss, "token_losses": each}
    else:
        at = torch.take_along_dim(logp, s["tokens"][..., None], 2).squeeze(2) * m
        if case["op"] == "preference":
            rewards = 0.1 * (at.sum(1) - s["ref"].double())
            z = rewards[:b // 2] - rewards[b // 2:]
            loss = -case["scale"] * (0.95 * torch.nn.functional.logsigmoid(z) + 0.05 * torch.nn.functional.logsigmoid(-z)).mean()
            out = {"loss": loss, "rewards": rewards}
        else:
            ent = None
            if case["op"] == "policy" or case["entropy"]:
                ent = -(logp.exp() * logp.masked_fill(logp == -math.inf, 0.0)).sum(-1) * m
            out = {"logprobs": at, "entropy": ent}
            if case["op"] == "logprobs":
                if case["form"] == "forward":
                    return out
                loss = (at * s["g_logprobs"].double()).sum()
                if ent is not None:
                    loss = loss + (ent * s["g_entropy"].double()).sum()
            else:
                ratio, a = torch.exp(at - s["old"].double()), s["advantages"].double()
                each = -torch.minimum(ratio * a, torch.clamp(ratio, 1 - EPS_CLIP, 1 + EPS_CLIP) * a)
                if case["kl_coef"]:
                    d = s["ref"].double() - at
                    each = each + case["kl_coef"] * (torch.expm1(d) - d)
                loss = (w * (each - case["entropy_coef"] * ent)).sum()
                out["loss"] = loss
    out["grad"] = torch.autograd.grad(loss, x)[0]
    return {k: None if v is None else v.detach() for k, v in out.items()}
