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
# The checks are written for their cost: a call on a few rows is host time and little else.
def _check_logits(logits):
    if not isinstance(logits, torch.Tensor) or logits.dim() not in (2, 3):
        raise ValueError("logits must be a tensor [sequences, tokens, vocabulary] or [tokens, vocabulary]")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits of type {logits.dtype}: float32, bfloat16 and float16 are supported")
    if logits.shape[-1] < 1:
        raise ValueError("logits over an empty vocabulary")
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        raise ValueError("the vocabulary must be the contiguous dimension of the logits")
    return logits.shape[:-1]


def _check(logits, t, name, types, shape):
    """A tensor beside the logits: of these types, of this shape, where the logits are, without a gradient of its own."""
    if not isinstance(t, torch.Tensor) or t.get_device() != logits.get_device():
        raise ValueError(f"{name} must be a tensor on {logits.device}, where the logits are")
    if t.requires_grad:
        raise ValueError(f"{name} requires grad, but gradients are computed with respect to the logits only: detach it")
    if t.dtype not in types:
        raise ValueError(f"{name} of type {t.dtype}: {', '.join(str(d)[6:] for d in types)} are supported")
    if t.shape != shape:
        raise ValueError(f"{name} of shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


_INTEGERS = (torch.int64, torch.int32)
_MASKS = (torch.bool, torch.uint8)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16, torch.float64)


def _integers(logits, t, name, shape):
    return _check(logits, t, name, _INTEGERS, shape).contiguous()


def _mask(logits, t, shape):
    return None if t is None else _check(logits, t, "mask", _MASKS, shape).contiguous()


def _floats(logits, t, name, shape):
    t = _check(logits, t, name, _FLOATS, shape)
    return t if t.dtype is torch.float32 else t.to(torch.float32)


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


def _grad_strides(logits):
    """Strides for a gradient's storage: the logits' own row strides where they waste little memory (16-byte accesses
    then fall on the same boundaries in both), None for dense rows."""
    if logits.is_contiguous():
        return None
    reach = logits.shape[-1]
    for d in range(logits.dim() - 2, -1, -1):
        if logits.shape[d] > 1 and logits.stride(d) < reach:
            return None       # broadcast or reordered rows
        reach = (logits.shape[d] - 1) * logits.stride(d) + reach
    return None if reach > 1.25 * logits.numel() + 64 else logits.stride()


def _grad_like(logits):
    """Storage for the gradient, aligned as the logits are."""
    strides = _grad_strides(logits)
    if strides is None:
        return torch.empty_like(logits, memory_format=torch.contiguous_format)
    lead = logits.data_ptr() % 16 // logits.element_size()
    reach = 1 + sum((n - 1) * s for n, s in zip(logits.shape, strides))
    return logits.new_empty(reach + lead).as_strided(logits.shape, strides, lead)


def _rows_of(logits, inv_temperature, grad=None):
    """The C ABI's description of the logits (and of the gradient's rows)."""
    if logits.dim() == 3:
        n_seq, n_tok, vocab = logits.shape
        s, t, _ = logits.stride()
        gs, gt, _ = (0, 0, 0) if grad is None else grad.stride()
    else:
        n_seq, (n_tok, vocab) = 1, logits.shape
        s, t = 0, logits.stride(0)
        gs, gt = 0, 0 if grad is None else grad.stride(0)
    return _lib.TokenLogits(logits.data_ptr(), s, t, gs, gt, n_seq, n_tok, vocab, _DTYPES[logits.dtype], inv_temperature)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)     # absent from builds of torch without a GPU


def _call(logits, name, *args):
    """One library call on the current stream of the logits' device."""
    index = logits.get_device()
    if index < 0:
        raise RuntimeError(f"ppo_amd: logits on {logits.device}; the HIP engine has no CPU fallback")
    fn = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == index:
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _raw_stream(index))
    if code:
        _lib.check(code)


def _scratch(logits, rows, floats_per_row=0):
    """Scratch of one call and its size in bytes, behind which it has `floats_per_row` floats a row for a backward call."""
    n_seq, n_tok = rows if len(rows) == 2 else (1, rows[0])
    need = _lib.lib().ppo_token_workspace_bytes(n_seq, n_tok)
    ws = torch.empty(need + 4 * floats_per_row * n_seq * n_tok, dtype=torch.uint8, device=logits.device)
    return ws, need


def _new(logits, shape=()):
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
    logp = _new(logits, shape)
    ent = torch.empty_like(logp) if entropy else None
    _call(logits, "ppo_token_logprobs", ctypes.byref(_rows_of(logits, inv_t)), tokens.data_ptr(),
          tokens.dtype is torch.int64, _lib.ptr(mask), logp.data_ptr(), _lib.ptr(ent), _lib.ptr(stats))
    return logp, ent


def _logprobs_backward(logits, tokens, mask, inv_t, stats, g_logp, lp_strides, g_ent, ent_strides, factor):
    """stats, g_logp, g_ent: addresses."""
    grad = _grad_like(logits)
    _call(logits, "ppo_token_logprobs_backward", ctypes.byref(_rows_of(logits, inv_t, grad)), tokens.data_ptr(),
          tokens.dtype is torch.int64, _lib.ptr(mask), stats, g_logp, *lp_strides, g_ent, *ent_strides,
          _lib.ptr(factor), grad.data_ptr())
    return grad


class _LogprobsFn(torch.autograd.Function):
    """token_logprobs() as an autograd node."""

    @staticmethod
    def forward(ctx, logits, tokens, mask, inv_t, entropy):
        stats = _new(logits, (*logits.shape[:-1], 4))
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
        return (_logprobs_backward(logits, tokens, mask, ctx.inv_t, stats.data_ptr(), _lib.ptr(g_logp), lp_strides,
                                   _lib.ptr(g_ent), ent_strides, None), None, None, None, None)


def token_logprobs(logits, tokens, mask=None, *, temperature=1.0, entropy=True):
    """Log-probability of each token and the entropy of each row's distribution: ``(logprobs, entropy)``, float32 of
    the tokens' shape (entropy is None with ``entropy=False``).  Both carry gradients to the logits; what a rollout
    needs (``[sequences, 1, vocabulary]`` or ``[sequences, vocabulary]`` logits of one step) runs under ``no_grad``."""
    shape = _check_logits(logits)
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
    shape = _check_logits(logits)
    tokens = _integers(logits, tokens, "tokens", shape)
    mask = _mask(logits, mask, shape)
    old = _floats(logits, old_logprobs, "old_logprobs", shape).contiguous()
    per = getattr(advantages, "shape", shape)
    if len(shape) == 2 and per != shape and per in ((shape[0],), (shape[0], 1)):
        adv = _floats(logits, advantages, "advantages", per)
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


def _policy_call(logits, args, grad, seeds):
    """-> loss, log-probabilities, entropies, the scratch and where in it (bytes) lies, with `seeds`, what a backward
    call needs: 4 floats a row of statistics, then dloss/dlogprob, then dloss/dentropy."""
    tokens, mask, old, adv, adv_strides, ref, terms, inv_t = args
    loss, logp, ent = _new(logits), torch.empty_like(old), torch.empty_like(old)
    ws, need = _scratch(logits, old.shape, 6 if seeds else 0)
    at = ws.data_ptr()
    stats = at + need if seeds else None
    _call(logits, "ppo_policy_loss", ctypes.byref(_rows_of(logits, inv_t, grad)), tokens.data_ptr(),
          tokens.dtype is torch.int64, _lib.ptr(mask), old.data_ptr(), adv.data_ptr(), *adv_strides, _lib.ptr(ref),
          ctypes.byref(terms), loss.data_ptr(), logp.data_ptr(), ent.data_ptr(), stats,
          stats + 16 * old.numel() if seeds else None, _lib.ptr(grad), at, need)
    return loss, logp, ent, ws, need


class _PolicyLossFn(torch.autograd.Function):
    """policy_loss() as an autograd node: the forward call leaves dloss/dlogprob and dloss/dentropy of each row."""

    @staticmethod
    def forward(ctx, logits, args):
        loss, logp, ent, ws, ctx.offset = _policy_call(logits, args, None, True)
        ctx.with_entropy, ctx.inv_t = args[6].entropy_coef != 0, args[7]
        ctx.strides, ctx.rows = _row_strides(logp), logp.numel()
        ctx.mark_non_differentiable(logp, ent)
        ctx.save_for_backward(logits, args[0], args[1], ws)
        return loss, logp, ent

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _g_logp, _g_ent):
        logits, tokens, mask, ws = ctx.saved_tensors
        stats = ws.data_ptr() + ctx.offset
        g_logp = stats + 16 * ctx.rows
        return _logprobs_backward(logits, tokens, mask, ctx.inv_t, stats, g_logp, ctx.strides,
                                  g_logp + 4 * ctx.rows if ctx.with_entropy else None, ctx.strides, g_loss), None


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
    return _policy_call(logits, args, None, False)[:3]


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
    loss, logp, ent, _, _ = _policy_call(logits_, args, grad, False)
    _written(out, logits)
    return loss, grad, logp, ent


# ------------------------------------------------------------------------------------------ preference loss
def _preference_args(logits, tokens, ref_logprobs, mask, beta, label_smoothing, scale):
    shape = _check_logits(logits)
    if logits.dim() != 3 or logits.shape[0] < 2 or logits.shape[0] % 2:
        raise ValueError("preference losses need logits [2 * pairs, tokens, vocabulary]: the preferred sequences, then "
                         f"the rejected ones in the same order; got {tuple(logits.shape)}")
    tokens = _integers(logits, tokens, "tokens", shape)
    mask = _mask(logits, mask, shape)
    ref = _floats(logits, ref_logprobs, "ref_logprobs", shape[:1]).contiguous()
    if not 0 <= label_smoothing < 1:
        raise ValueError(f"label_smoothing {label_smoothing}: 0 <= label_smoothing < 1 is expected")
    return tokens, mask, ref, float(beta), float(label_smoothing), float(scale)


def _preference_call(logits, args, grad, seeds):
    """-> loss, rewards, the scratch, and with `seeds` what a backward call needs: where in the scratch the rows'
    statistics lie (bytes), and dloss/dlogprob of each sequence's tokens."""
    tokens, mask, ref, beta, smoothing, scale = args
    loss, rewards = _new(logits), torch.empty_like(ref)
    ws, need = _scratch(logits, tokens.shape, 4 if seeds else 0)
    at = torch.empty_like(ref) if seeds else None
    _call(logits, "ppo_preference_loss", ctypes.byref(_rows_of(logits, 1.0, grad)), tokens.data_ptr(),
          tokens.dtype is torch.int64, _lib.ptr(mask), ref.data_ptr(), beta, smoothing, scale, loss.data_ptr(),
          rewards.data_ptr(), ws.data_ptr() + need if seeds else None, _lib.ptr(at), _lib.ptr(grad), ws.data_ptr(), need)
    return loss, rewards, ws, need, at


class _PreferenceLossFn(torch.autograd.Function):
    """preference_loss() as an autograd node: dloss/dlogprob is one number for all tokens of a sequence."""

    @staticmethod
    def forward(ctx, logits, args):
        loss, rewards, ws, ctx.offset, seeds = _preference_call(logits, args, None, True)
        ctx.mark_non_differentiable(rewards)
        ctx.save_for_backward(logits, args[0], args[1], ws, seeds)
        return loss, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _g_rewards):
        logits, tokens, mask, ws, seeds = ctx.saved_tensors
        return _logprobs_backward(logits, tokens, mask, 1.0, ws.data_ptr() + ctx.offset, seeds.data_ptr(), (1, 0), None,
                                  (0, 0), g_loss), None


def preference_loss(logits, tokens, ref_logprobs, mask=None, *, beta=0.1, label_smoothing=0.0, scale=1.0):
    """Preference loss on pairs: ``(loss, rewards)``.  Sequence ``q`` of the first half is preferred to sequence
    ``q + pairs``; ``rewards = beta * (sum of the counted log-probabilities - ref_logprobs)`` per sequence,
    ``ref_logprobs`` being the same sums under the reference policy, and the loss is the mean over the pairs of
    ``-ln sigmoid(difference of rewards)``, with ``label_smoothing`` the probability that a label is wrong.  ``loss``
    carries gradients to the logits, ``rewards`` is for logging."""
    args = _preference_args(logits, tokens, ref_logprobs, mask, beta, label_smoothing, scale)
    if _wants_grad(logits):
        return _PreferenceLossFn.apply(logits, args)
    return _preference_call(logits, args, None, False)[:2]


def preference_loss_and_grad(logits, tokens, ref_logprobs, mask=None, *, beta=0.1, label_smoothing=0.0, scale=1.0,
                             out=None):
    """``preference_loss`` and its gradient at once: ``(loss, grad, rewards)``; ``out`` as in policy_loss_and_grad."""
    logits_ = logits.detach() if isinstance(logits, torch.Tensor) else logits
    args = _preference_args(logits_, tokens, ref_logprobs, mask, beta, label_smoothing, scale)
    grad = _grad_like(logits_) if out is None else _check_out(out, logits_, (
        ("the logits", logits_), ("tokens", args[0]), ("mask", args[1]), ("ref_logprobs", args[2])))
    loss, rewards = _preference_call(logits_, args, grad, False)[:2]
    _written(out, logits)
    return loss, grad, rewards


# ------------------------------------------------------------------------------------------ distillation
def _distillation_args(logits, teacher_tokens, teacher_logits, mask, temperature, reduction, scale):
    shape = _check_logits(logits)
    if not isinstance(teacher_tokens, torch.Tensor) or teacher_tokens.dim() != logits.dim() \
            or not 1 <= teacher_tokens.shape[-1] <= MAX_TEACHER_TOP:
        raise ValueError(f"teacher_tokens must be {tuple(shape)} by 1 to {MAX_TEACHER_TOP} entries")
    full = (*shape, teacher_tokens.shape[-1])
    index = _integers(logits, teacher_tokens, "teacher_tokens", full)
    values = _check(logits, teacher_logits, "teacher_logits", _FLOATS[:3], full).contiguous()
    return (index, values, _mask(logits, mask, shape), _temperature(temperature),
            _reduction(reduction), float(scale))


def _teacher(index, values):
    return index.data_ptr(), index.dtype is torch.int64, values.data_ptr(), _DTYPES[values.dtype], index.shape[-1]


def _distillation_call(logits, args, grad, seeds):
    """-> loss, token losses, the scratch and where in it (bytes) lie, with `seeds`, the statistics for a backward call."""
    index, values, mask, inv_t, reduction, scale = args
    shape = logits.shape[:-1]
    loss, each = _new(logits), _new(logits, shape)
    ws, need = _scratch(logits, shape, 4 if seeds else 0)
    _call(logits, "ppo_distillation_loss", ctypes.byref(_rows_of(logits, inv_t, grad)), *_teacher(index, values),
          _lib.ptr(mask), reduction, scale, loss.data_ptr(), each.data_ptr(), ws.data_ptr() + need if seeds else None,
          _lib.ptr(grad), ws.data_ptr(), need)
    return loss, each, ws, need


class _DistillationLossFn(torch.autograd.Function):
    """distillation_loss() as an autograd node."""

    @staticmethod
    def forward(ctx, logits, args):
        loss, each, ws, ctx.offset = _distillation_call(logits, args, None, True)
        ctx.inv_t = args[3]
        ctx.mark_non_differentiable(each)
        ctx.save_for_backward(logits, args[0], args[1], args[2], ws)
        return loss, each

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _g_each):
        logits, index, values, mask, ws = ctx.saved_tensors
        grad = _grad_like(logits)
        _call(logits, "ppo_distillation_backward", ctypes.byref(_rows_of(logits, ctx.inv_t, grad)),
              *_teacher(index, values), _lib.ptr(mask), ws.data_ptr() + ctx.offset, g_loss.data_ptr(), grad.data_ptr())
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
    return _distillation_call(logits, args, None, False)[:2]


def distillation_loss_and_grad(logits, teacher_tokens, teacher_logits, mask=None, *, temperature=1.0,
                               reduction="token_mean", scale=1.0, out=None):
    """``distillation_loss`` and its gradient at once: ``(loss, grad, token_losses)``; ``out`` as in
    policy_loss_and_grad."""
    logits_ = logits.detach() if isinstance(logits, torch.Tensor) else logits
    args = _distillation_args(logits_, teacher_tokens, teacher_logits, mask, temperature, reduction, scale)
    grad = _grad_like(logits_) if out is None else _check_out(out, logits_, (
        ("the logits", logits_), ("teacher_tokens", args[0]), ("teacher_logits", args[1]), ("mask", args[2])))
    loss, each = _distillation_call(logits_, args, grad, False)[:2]
    _written(out, logits)
    return loss, grad, each
