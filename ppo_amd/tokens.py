"""Losses of a policy whose action is a token of a large vocabulary, from the logits of a model of the caller's.

What ``ActorCritic.evaluate`` and the fused update do for a head of a few actions (PPO.py:102-121, 227-244), for
logits ``[sequences, tokens, vocabulary]`` (or ``[tokens, vocabulary]``: one sequence) in float32, bfloat16 or
float16:

``token_logprobs``      log-probability of given tokens and entropy, differentiable
``policy_loss``         clipped surrogate with a KL term against a reference policy and an entropy term
``preference_loss``     paired log ratios: the first half of the sequences preferred to the second half
``distillation_loss``   divergence from a teacher's top logits

The three losses are differentiable with respect to the logits, and each has an ``..._and_grad`` form that returns
``dloss/dlogits`` together with the loss, for ``logits.backward(grad)`` or a model's own backward pass.  That form
reads the logits once where they fit on the chip, and its gradient may take the logits' place (``out=logits``).

Common arguments
  tokens        int64 or int32, the shape of the logits without the vocabulary
  mask          bool or uint8 of that shape, or None: rows that count.  A row that does not count is not read: its
                logits may hold anything (NaN too) and its token may be any number; its outputs and its gradient are 0.
  temperature   probabilities are softmax(logits / temperature)
  reduction     "token_mean" (over all counted rows), "sequence_mean" (mean over a sequence's counted rows, then over
                the sequences that have any) or "sum"; 0 where nothing counts
  scale         factor on loss and gradient: the loss scale of float16 training, or 1 / (tokens of all ranks) with
                reduction="sum" in data-parallel training

Logits may be any view whose last dimension is contiguous (``logits[:, :-1]``, a slice of a padded vocabulary).
Everything runs asynchronously on the current stream of the logits' device; there is no CPU fallback.  A token
outside the vocabulary makes its row's results NaN.
"""
import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_REDUCTIONS = {"sum": 0, "token_mean": 1, "sequence_mean": 2}
MAX_TEACHER_TOP = 512


# ------------------------------------------------------------------------------------------ arguments
def _check_logits(logits):
    if not isinstance(logits, torch.Tensor) or logits.dim() not in (2, 3):
        raise ValueError("logits must be a tensor [sequences, tokens, vocabulary] or [tokens, vocabulary]")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits of type {logits.dtype}: float32, bfloat16 and float16 are supported")
    if logits.shape[-1] < 1:
        raise ValueError("logits over an empty vocabulary")
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        raise ValueError("the vocabulary must be the contiguous dimension of the logits")


def _same_device(logits, t, name):
    if not isinstance(t, torch.Tensor) or t.device != logits.device:
        raise ValueError(f"{name} must be a tensor on {logits.device}, where the logits are")
    if t.requires_grad:
        raise ValueError(f"{name} requires grad, but gradients are computed with respect to the logits only: detach it")


def _integers(logits, t, name, shape):
    _same_device(logits, t, name)
    if t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} of type {t.dtype}: int64 and int32 are supported")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} of shape {tuple(t.shape)}, expected {shape}")
    return t.contiguous()


def _mask(logits, t, shape):
    if t is None:
        return None
    _same_device(logits, t, "mask")
    if t.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"mask of type {t.dtype}: bool and uint8 are supported")
    if tuple(t.shape) != shape:
        raise ValueError(f"mask of shape {tuple(t.shape)}, expected {shape}")
    return t.contiguous()


def _floats(logits, t, name, shape):
    _same_device(logits, t, name)
    if not t.is_floating_point():
        raise ValueError(f"{name} of type {t.dtype}: floating point is expected")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} of shape {tuple(t.shape)}, expected {shape}")
    return t.to(torch.float32)


def _row_strides(t):
    """(sequence stride, token stride) of a per-row tensor."""
    return (t.stride(0), t.stride(1)) if t.dim() == 2 else (0, t.stride(0))


def _temperature(value):
    if not 1e-6 <= value <= 1e6:
        raise ValueError(f"temperature {value}: between 1e-6 and 1e6 is expected")
    return 1.0 / value


def _reduction(name):
    if name not in _REDUCTIONS:
        raise ValueError(f"reduction {name!r}: one of {sorted(_REDUCTIONS)} is expected")
    return _REDUCTIONS[name]


def _span(t):
    """Address range of a tensor's elements."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _check_out(out, logits, others):
    if not isinstance(out, torch.Tensor) or out.shape != logits.shape or out.dtype != logits.dtype \
            or out.device != logits.device:
        raise ValueError("out must have the shape, the type and the device of the logits")
    if out.shape[-1] > 1 and out.stride(-1) != 1:
        raise ValueError("the vocabulary must be the contiguous dimension of out")
    rows = [(out.stride(d), out.shape[d]) for d in range(out.dim() - 1) if out.shape[d] > 1]
    reach = out.shape[-1]
    for stride, n in reversed(rows):
        if stride < reach:
            raise ValueError("rows of out overlap")
        reach = (n - 1) * stride + reach
    lo, hi = _span(out)
    for name, t in others:
        if t is None:
            continue
        a, b = _span(t)
        if a < hi and lo < b and not (t is logits and a == lo and out.stride() == logits.stride()):
            raise ValueError(f"out shares memory with {name}" + (": only the logits themselves can be overwritten"
                                                                 if t is logits else ""))
    return out.detach()


def _grad_like(logits):
    """Storage for the gradient: the logits' own row strides and alignment where that wastes little memory (16-byte
    accesses then fall on the same boundaries in both), dense rows otherwise."""
    if logits.is_contiguous() or not logits.numel():
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    reach = logits.shape[-1]
    for d in range(logits.dim() - 2, -1, -1):
        if logits.shape[d] > 1 and logits.stride(d) < reach:
            return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)   # broadcast or reordered rows
        reach = (logits.shape[d] - 1) * logits.stride(d) + reach
    if reach > 1.25 * logits.numel() + 64:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    lead = logits.data_ptr() % 16 // logits.element_size()
    store = torch.empty(reach + lead, dtype=logits.dtype, device=logits.device)
    return store.as_strided(logits.shape, logits.stride(), lead)


def _rows_of(logits, inv_temperature, grad=None):
    """The C ABI's description of the logits (and of the gradient's rows)."""
    if logits.dim() == 3:
        n_seq, n_tok, vocab = logits.shape
        strides = (logits.stride(0), logits.stride(1))
        gs = (grad.stride(0), grad.stride(1)) if grad is not None else (0, 0)
    else:
        n_seq, (n_tok, vocab) = 1, logits.shape
        strides = (0, logits.stride(0))
        gs = (0, grad.stride(0)) if grad is not None else (0, 0)
    return _lib.TokenLogits(logits.data_ptr(), *strides, *gs, n_seq, n_tok, vocab, _DTYPES[logits.dtype], inv_temperature)


def _call(logits, name, *args):
    """One library call on the current stream of the logits' device."""
    dev = logits.device
    if dev.type != "cuda":
        raise RuntimeError(f"ppo_amd: logits on {dev}; the HIP engine has no CPU fallback")
    fn = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == dev.index:
        code = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            code = fn(*args, torch.cuda.current_stream().cuda_stream)
    _lib.check(code)


def _workspace(logits):
    n_seq, n_tok = logits.shape[:2] if logits.dim() == 3 else (1, logits.shape[0])
    need = _lib.lib().ppo_token_workspace_bytes(n_seq, n_tok)
    return torch.empty(need, dtype=torch.uint8, device=logits.device), need


def _new(logits, *shape):
    return torch.empty(shape, dtype=torch.float32, device=logits.device)


def _wants_grad(logits):
    return torch.is_grad_enabled() and logits.requires_grad


def _written(out, logits):
    """The version counter of overwritten logits moves, so that autograd notices a use of their old values."""
    if out is not None:
        torch.autograd.graph.increment_version(out)
        if out.data_ptr() == logits.data_ptr():
            torch.autograd.graph.increment_version(logits)


# ------------------------------------------------------------------------------------------ log-probabilities
def _logprobs_forward(logits, tokens, mask, inv_t, entropy, stats):
    shape = logits.shape[:-1]
    logp = _new(logits, *shape)
    ent = _new(logits, *shape) if entropy else None
    x = _rows_of(logits, inv_t)
    _call(logits, "ppo_token_logprobs", ctypes.byref(x), tokens.data_ptr(), tokens.dtype == torch.int64,
          _lib.ptr(mask), logp.data_ptr(), _lib.ptr(ent), _lib.ptr(stats))
    return logp, ent


def _logprobs_backward(logits, tokens, mask, inv_t, stats, g_logp, lp_strides, g_ent, ent_strides, factor):
    grad = _grad_like(logits)
    x = _rows_of(logits, inv_t, grad)
    _call(logits, "ppo_token_logprobs_backward", ctypes.byref(x), tokens.data_ptr(), tokens.dtype == torch.int64,
          _lib.ptr(mask), stats.data_ptr(), _lib.ptr(g_logp), *lp_strides, _lib.ptr(g_ent), *ent_strides,
          _lib.ptr(factor), grad.data_ptr())
    return grad


class _LogprobsFn(torch.autograd.Function):
    """token_logprobs() as an autograd node."""

    @staticmethod
    def forward(ctx, logits, tokens, mask, inv_t, entropy):
        stats = _new(logits, *logits.shape[:-1], 4)
        logp, ent = _logprobs_forward(logits, tokens, mask, inv_t, entropy, stats)
        ctx.inv_t = inv_t
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, mask, stats)
        return (logp, ent) if entropy else logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_ent=None):
        if g_logp is None and g_ent is None:
            return (None,) * 5
        logits, tokens, mask, stats = ctx.saved_tensors
        lp_strides = _row_strides(g_logp) if g_logp is not None else (0, 0)
        ent_strides = _row_strides(g_ent) if g_ent is not None else (0, 0)
        return (_logprobs_backward(logits, tokens, mask, ctx.inv_t, stats, g_logp, lp_strides, g_ent, ent_strides, None),
                None, None, None, None)


def token_logprobs(logits, tokens, mask=None, *, temperature=1.0, entropy=True):
    """Log-probability of each token and the entropy of each row's distribution: ``(logprobs, entropy)``, float32 of
    the tokens' shape (entropy is None with ``entropy=False``).  Both carry gradients to the logits; what a rollout
    needs (``[sequences, 1, vocabulary]`` or ``[sequences, vocabulary]`` logits of one step) runs under ``no_grad``."""
    _check_logits(logits)
    shape = tuple(logits.shape[:-1])
    tokens = _integers(logits, tokens, "tokens", shape)
    mask = _mask(logits, mask, shape)
    inv_t = _temperature(temperature)
    if _wants_grad(logits):
        out = _LogprobsFn.apply(logits, tokens, mask, inv_t, bool(entropy))
        return out if entropy else (out, None)
    return _logprobs_forward(logits, tokens, mask, inv_t, entropy, None)


# ------------------------------------------------------------------------------------------ clipped policy loss
def _policy_args(logits, tokens, old_logprobs, advantages, mask, ref_logprobs, eps_clip, eps_clip_high, kl_coef,
                 entropy_coef, temperature, reduction, scale):
    _check_logits(logits)
    shape = tuple(logits.shape[:-1])
    tokens = _integers(logits, tokens, "tokens", shape)
    mask = _mask(logits, mask, shape)
    old = _floats(logits, old_logprobs, "old_logprobs", shape).contiguous()
    _same_device(logits, advantages, "advantages")
    if logits.dim() == 3 and tuple(advantages.shape) in ((shape[0],), (shape[0], 1)):
        adv = _floats(logits, advantages, "advantages", tuple(advantages.shape))
        adv_strides = (adv.stride(0), 0)
    else:
        adv = _floats(logits, advantages, "advantages", shape)
        adv_strides = _row_strides(adv)
    if ref_logprobs is None:
        if kl_coef != 0:
            raise ValueError("kl_coef without ref_logprobs")
        ref = None
    else:
        ref = _floats(logits, ref_logprobs, "ref_logprobs", shape).contiguous()
    high = eps_clip if eps_clip_high is None else eps_clip_high
    if not (0 <= eps_clip <= 1 and high >= 0):
        raise ValueError(f"clip range [1 - {eps_clip}, 1 + {high}]: 0 <= eps_clip <= 1 and eps_clip_high >= 0 are expected")
    terms = _lib.PolicyTerms(eps_clip, high, kl_coef, entropy_coef, scale, _reduction(reduction))
    return tokens, mask, old, adv, adv_strides, ref, terms, _temperature(temperature)


def _policy_call(logits, args, stats, seeds, grad):
    tokens, mask, old, adv, adv_strides, ref, terms, inv_t = args
    shape = logits.shape[:-1]
    loss, logp, ent = _new(logits), _new(logits, *shape), _new(logits, *shape)
    ws, need = _workspace(logits)
    x = _rows_of(logits, inv_t, grad)
    _call(logits, "ppo_policy_loss", ctypes.byref(x), tokens.data_ptr(), tokens.dtype == torch.int64, _lib.ptr(mask),
          old.data_ptr(), adv.data_ptr(), *adv_strides, _lib.ptr(ref), ctypes.byref(terms), loss.data_ptr(),
          logp.data_ptr(), ent.data_ptr(), _lib.ptr(stats), _lib.ptr(seeds), _lib.ptr(grad), ws.data_ptr(), need)
    return loss, logp, ent


class _PolicyLossFn(torch.autograd.Function):
    """policy_loss() as an autograd node: the forward call leaves dloss/dlogprob and dloss/dentropy of each row."""

    @staticmethod
    def forward(ctx, logits, args):
        tokens, mask, *_, terms, ctx.inv_t = args
        stats = _new(logits, *logits.shape[:-1], 4)
        seeds = _new(logits, 2, *logits.shape[:-1])
        loss, logp, ent = _policy_call(logits, args, stats, seeds, None)
        ctx.with_entropy = terms.entropy_coef != 0
        ctx.mark_non_differentiable(logp, ent)
        ctx.save_for_backward(logits, tokens, mask, stats, seeds)
        return loss, logp, ent

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _g_logp, _g_ent):
        logits, tokens, mask, stats, seeds = ctx.saved_tensors
        strides = _row_strides(seeds[0])
        return _logprobs_backward(logits, tokens, mask, ctx.inv_t, stats, seeds[0], strides,
                                  seeds[1] if ctx.with_entropy else None, strides, g_loss), None


def policy_loss(logits, tokens, old_logprobs, advantages, mask=None, *, ref_logprobs=None, eps_clip=0.2,
                eps_clip_high=None, kl_coef=0.0, entropy_coef=0.0, temperature=1.0, reduction="token_mean", scale=1.0):
    """Clipped policy loss (PPO.py:233-240 without the value term) plus ``kl_coef`` times the divergence from a
    reference policy (``exp(d) - d - 1``, ``d = ref - logprob``) minus ``entropy_coef`` times the entropy:
    ``(loss, logprobs, entropy)``.  ``loss`` carries gradients to the logits; the per-token log-probabilities and
    entropies (of ``softmax(logits / temperature)``) are for logging.  ``advantages`` has the tokens' shape, or one
    value for each sequence (``[sequences]`` or ``[sequences, 1]``).  The ratio is clipped to
    ``[1 - eps_clip, 1 + eps_clip_high]`` (``eps_clip_high``: as ``eps_clip``)."""
    args = _policy_args(logits, tokens, old_logprobs, advantages, mask, ref_logprobs, eps_clip, eps_clip_high, kl_coef,
                        entropy_coef, temperature, reduction, scale)
    if _wants_grad(logits):
        return _PolicyLossFn.apply(logits, args)
    return _policy_call(logits, args, None, None, None)


def policy_loss_and_grad(logits, tokens, old_logprobs, advantages, mask=None, *, ref_logprobs=None, eps_clip=0.2,
                         eps_clip_high=None, kl_coef=0.0, entropy_coef=0.0, temperature=1.0, reduction="token_mean",
                         scale=1.0, out=None):
    """``policy_loss`` and its gradient at once: ``(loss, grad, logprobs, entropy)``.  ``out`` (the logits themselves,
    or memory of their shape and type) receives the gradient."""
    logits_ = logits.detach() if isinstance(logits, torch.Tensor) else logits
    args = _policy_args(logits_, tokens, old_logprobs, advantages, mask, ref_logprobs, eps_clip, eps_clip_high, kl_coef,
                        entropy_coef, temperature, reduction, scale)
    grad = _grad_like(logits_) if out is None else _check_out(out, logits_, (
        ("the logits", logits_), ("tokens", args[0]), ("mask", args[1]), ("old_logprobs", args[2]),
        ("advantages", args[3]), ("ref_logprobs", args[5])))
    loss, logp, ent = _policy_call(logits_, args, None, None, grad)
    _written(out, logits)
    return loss, grad, logp, ent


# ------------------------------------------------------------------------------------------ preference loss
def _preference_args(logits, tokens, ref_logprobs, mask, beta, label_smoothing, scale):
    _check_logits(logits)
    if logits.dim() != 3 or logits.shape[0] < 2 or logits.shape[0] % 2:
        raise ValueError("preference losses need logits [2 * pairs, tokens, vocabulary]: the preferred sequences, then "
                         f"the rejected ones in the same order; got {tuple(logits.shape)}")
    shape = tuple(logits.shape[:-1])
    tokens = _integers(logits, tokens, "tokens", shape)
    mask = _mask(logits, mask, shape)
    ref = _floats(logits, ref_logprobs, "ref_logprobs", shape[:1]).contiguous()
    if not 0 <= label_smoothing < 1:
        raise ValueError(f"label_smoothing {label_smoothing}: 0 <= label_smoothing < 1 is expected")
    return tokens, mask, ref, float(beta), float(label_smoothing), float(scale)


def _preference_call(logits, args, stats, seeds, grad):
    tokens, mask, ref, beta, smoothing, scale = args
    loss, rewards = _new(logits), _new(logits, logits.shape[0])
    ws, need = _workspace(logits)
    x = _rows_of(logits, 1.0, grad)
    _call(logits, "ppo_preference_loss", ctypes.byref(x), tokens.data_ptr(), tokens.dtype == torch.int64,
          _lib.ptr(mask), ref.data_ptr(), beta, smoothing, scale, loss.data_ptr(), rewards.data_ptr(), _lib.ptr(stats),
          _lib.ptr(seeds), _lib.ptr(grad), ws.data_ptr(), need)
    return loss, rewards


class _PreferenceLossFn(torch.autograd.Function):
    """preference_loss() as an autograd node: dloss/dlogprob is one number for all tokens of a sequence."""

    @staticmethod
    def forward(ctx, logits, args):
        stats, seeds = _new(logits, *logits.shape[:-1], 4), _new(logits, logits.shape[0])
        loss, rewards = _preference_call(logits, args, stats, seeds, None)
        ctx.mark_non_differentiable(rewards)
        ctx.save_for_backward(logits, args[0], args[1], stats, seeds)
        return loss, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _g_rewards):
        logits, tokens, mask, stats, seeds = ctx.saved_tensors
        return _logprobs_backward(logits, tokens, mask, 1.0, stats, seeds, (1, 0), None, (0, 0), g_loss), None


def preference_loss(logits, tokens, ref_logprobs, mask=None, *, beta=0.1, label_smoothing=0.0, scale=1.0):
    """Preference loss on pairs: ``(loss, rewards)``.  Sequence ``q`` of the first half is preferred to sequence
    ``q + pairs``; ``rewards = beta * (sum of the counted log-probabilities - ref_logprobs)`` per sequence,
    ``ref_logprobs`` being the same sums under the reference policy, and the loss is the mean over the pairs of
    ``-ln sigmoid(difference of rewards)``, with ``label_smoothing`` the probability that a label is wrong.  ``loss``
    carries gradients to the logits, ``rewards`` is for logging."""
    args = _preference_args(logits, tokens, ref_logprobs, mask, beta, label_smoothing, scale)
    if _wants_grad(logits):
        return _PreferenceLossFn.apply(logits, args)
    return _preference_call(logits, args, None, None, None)


def preference_loss_and_grad(logits, tokens, ref_logprobs, mask=None, *, beta=0.1, label_smoothing=0.0, scale=1.0,
                             out=None):
    """``preference_loss`` and its gradient at once: ``(loss, grad, rewards)``; ``out`` as in policy_loss_and_grad."""
    logits_ = logits.detach() if isinstance(logits, torch.Tensor) else logits
    args = _preference_args(logits_, tokens, ref_logprobs, mask, beta, label_smoothing, scale)
    grad = _grad_like(logits_) if out is None else _check_out(out, logits_, (
        ("the logits", logits_), ("tokens", args[0]), ("mask", args[1]), ("ref_logprobs", args[2])))
    loss, rewards = _preference_call(logits_, args, None, None, grad)
    _written(out, logits)
    return loss, grad, rewards


# ------------------------------------------------------------------------------------------ distillation
def _distillation_args(logits, teacher_tokens, teacher_logits, mask, temperature, reduction, scale):
    _check_logits(logits)
    shape = tuple(logits.shape[:-1])
    if not isinstance(teacher_tokens, torch.Tensor) or teacher_tokens.dim() != logits.dim() \
            or not 1 <= teacher_tokens.shape[-1] <= MAX_TEACHER_TOP:
        raise ValueError(f"teacher_tokens must be {shape} by 1 to {MAX_TEACHER_TOP} entries")
    full = shape + (teacher_tokens.shape[-1],)
    index = _integers(logits, teacher_tokens, "teacher_tokens", full)
    _same_device(logits, teacher_logits, "teacher_logits")
    if teacher_logits.dtype not in _DTYPES:
        raise ValueError(f"teacher_logits of type {teacher_logits.dtype}: float32, bfloat16 and float16 are supported")
    if tuple(teacher_logits.shape) != full:
        raise ValueError(f"teacher_logits of shape {tuple(teacher_logits.shape)}, expected {full}")
    return (index, teacher_logits.contiguous(), _mask(logits, mask, shape), _temperature(temperature),
            _reduction(reduction), float(scale))


def _teacher(index, values):
    return index.data_ptr(), index.dtype == torch.int64, values.data_ptr(), _DTYPES[values.dtype], index.shape[-1]


def _distillation_call(logits, args, stats, grad):
    index, values, mask, inv_t, reduction, scale = args
    loss, each = _new(logits), _new(logits, *logits.shape[:-1])
    ws, need = _workspace(logits)
    x = _rows_of(logits, inv_t, grad)
    _call(logits, "ppo_distillation_loss", ctypes.byref(x), *_teacher(index, values), _lib.ptr(mask), reduction, scale,
          loss.data_ptr(), each.data_ptr(), _lib.ptr(stats), _lib.ptr(grad), ws.data_ptr(), need)
    return loss, each


class _DistillationLossFn(torch.autograd.Function):
    """distillation_loss() as an autograd node."""

    @staticmethod
    def forward(ctx, logits, args):
        stats = _new(logits, *logits.shape[:-1], 4)
        loss, each = _distillation_call(logits, args, stats, None)
        ctx.inv_t = args[3]
        ctx.mark_non_differentiable(each)
        ctx.save_for_backward(logits, args[0], args[1], args[2], stats)
        return loss, each

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _g_each):
        logits, index, values, mask, stats = ctx.saved_tensors
        grad = _grad_like(logits)
        x = _rows_of(logits, ctx.inv_t, grad)
        _call(logits, "ppo_distillation_backward", ctypes.byref(x), *_teacher(index, values), _lib.ptr(mask),
              stats.data_ptr(), g_loss.data_ptr(), grad.data_ptr())
        return grad, None


def distillation_loss(logits, teacher_tokens, teacher_logits, mask=None, *, temperature=1.0, reduction="token_mean",
                      scale=1.0):
    """Divergence of the policy from a teacher of which the top logits are known: ``(loss, token_losses)``.
    ``teacher_tokens`` (int64 or int32) and ``teacher_logits`` have one dimension more than the rows, of up to 512
    entries; a negative token is padding.  The teacher's probabilities are the softmax of its logits over the given
    entries, the policy's that over the whole vocabulary, both at ``temperature``; a row's loss is ``temperature**2``
    times the divergence.  ``loss`` carries gradients to the logits, ``token_losses`` is for logging."""
    args = _distillation_args(logits, teacher_tokens, teacher_logits, mask, temperature, reduction, scale)
    if _wants_grad(logits):
        return _DistillationLossFn.apply(logits, args)
    return _distillation_call(logits, args, None, None)


def distillation_loss_and_grad(logits, teacher_tokens, teacher_logits, mask=None, *, temperature=1.0,
                               reduction="token_mean", scale=1.0, out=None):
    """``distillation_loss`` and its gradient at once: ``(loss, grad, token_losses)``; ``out`` as in
    policy_loss_and_grad."""
    logits_ = logits.detach() if isinstance(logits, torch.Tensor) else logits
    args = _distillation_args(logits_, teacher_tokens, teacher_logits, mask, temperature, reduction, scale)
    grad = _grad_like(logits_) if out is None else _check_out(out, logits_, (
        ("the logits", logits_), ("teacher_tokens", args[0]), ("teacher_logits", args[1]), ("mask", args[2])))
    loss, each = _distillation_call(logits_, args, None, grad)
    _written(out, logits)
    return loss, grad, each
