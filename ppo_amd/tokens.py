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

Logits may be any view whose last dimension is contiguous (``logits[:, :-1]``, a slice of a padded vocabulary).  Positions
that predict nothing may as well be left in and masked off: their rows of the gradient are zeros, and a backward pass has
no slice to undo.
Everything runs asynchronously on the current stream of the logits' device; there is no CPU fallback.  A token
outside the vocabulary makes its row's results NaN, but for the entropy, which does not depend on it.  There are no
second and no forward-mode derivatives: both raise.
"""
import ctypes

import torch  # noqa: F401  (its libraries are what the binding below is linked against)

from . import _lib
try:
    from . import _token_ops as _ops
except ImportError as e:
    raise ImportError("ppo_amd/_token_ops.so is missing or does not fit this torch: build it with "
                      f"`python -m ppo_amd.build` ({e})") from e

_ops.bind({name: ctypes.cast(getattr(_lib.lib(), name), ctypes.c_void_p).value
           for name in _lib.EXPORTS if "token" in name or "_loss" in name or name.startswith(("ppo_distill", "ppo_hip_strerror"))})

MAX_TEACHER_TOP = _ops.MAX_TEACHER_TOP
_REDUCTIONS = _ops.REDUCTIONS


def _reduction(name):
    if name not in _REDUCTIONS:
        raise ValueError(f"reduction {name!r}: one of {sorted(_REDUCTIONS)} is expected")
    return _REDUCTIONS[name]


def token_logprobs(logits, tokens, mask=None, *, temperature=1.0, entropy=True):
    """Log-probability of each token and the entropy of each row's distribution: ``(logprobs, entropy)``, float32 of
    the tokens' shape (entropy is None with ``entropy=False``).  Both carry gradients to the logits; what a rollout
    needs (``[sequences, 1, vocabulary]`` or ``[sequences, vocabulary]`` logits of one step) runs under ``no_grad``."""
    return _ops.token_logprobs(logits, tokens, mask, temperature, entropy)


def policy_loss(logits, tokens, old_logprobs, advantages, mask=None, *, ref_logprobs=None, eps_clip=0.2,
                eps_clip_high=None, kl_coef=0.0, entropy_coef=0.0, temperature=1.0, reduction="token_mean", scale=1.0):
    """Clipped policy loss (PPO.py:233-240 without the value term) plus ``kl_coef`` times the divergence from a
    reference policy (``exp(d) - d - 1``, ``d = ref - logprob``) minus ``entropy_coef`` times the entropy:
    ``(loss, logprobs, entropy)``.  ``loss`` carries gradients to the logits; the per-token log-probabilities and
    entropies (of ``softmax(logits / temperature)``) are for logging.  ``advantages`` has the tokens' shape, or one
    value for each sequence (``[sequences]`` or ``[sequences, 1]``).  The ratio is clipped to
    ``[1 - eps_clip, 1 + eps_clip_high]`` (``eps_clip_high``: as ``eps_clip``)."""
    return _ops.policy_loss(logits, tokens, old_logprobs, advantages, mask, ref_logprobs, eps_clip, eps_clip_high, kl_coef,
                            entropy_coef, temperature, _reduction(reduction), scale)


def policy_loss_and_grad(logits, tokens, old_logprobs, advantages, mask=None, *, ref_logprobs=None, eps_clip=0.2,
                         eps_clip_high=None, kl_coef=0.0, entropy_coef=0.0, temperature=1.0, reduction="token_mean",
                         scale=1.0, out=None):
    """``policy_loss`` and its gradient at once: ``(loss, grad, logprobs, entropy)``.  ``out`` (the logits themselves,
    or memory of their shape and type) receives the gradient."""
    return _ops.policy_loss_and_grad(logits, tokens, old_logprobs, advantages, mask, ref_logprobs, eps_clip, eps_clip_high,
                                     kl_coef, entropy_coef, temperature, _reduction(reduction), scale, out)


def preference_loss(logits, tokens, ref_logprobs, mask=None, *, beta=0.1, label_smoothing=0.0, scale=1.0):
    """Preference loss on pairs: ``(loss, rewards)``.  Sequence ``q`` of the first half is preferred to sequence
    ``q + pairs``; ``rewards = beta * (sum of the counted log-probabilities - ref_logprobs)`` per sequence,
    ``ref_logprobs`` being the same sums under the reference policy, and the loss is the mean over the pairs of
    ``-ln sigmoid(difference of rewards)``, with ``label_smoothing`` the probability that a label is wrong.  ``loss``
    carries gradients to the logits, ``rewards`` is for logging."""
    return _ops.preference_loss(logits, tokens, ref_logprobs, mask, beta, label_smoothing, scale)


def preference_loss_and_grad(logits, tokens, ref_logprobs, mask=None, *, beta=0.1, label_smoothing=0.0, scale=1.0,
                             out=None):
    """``preference_loss`` and its gradient at once: ``(loss, grad, rewards)``; ``out`` as in policy_loss_and_grad."""
    return _ops.preference_loss_and_grad(logits, tokens, ref_logprobs, mask, beta, label_smoothing, scale, out)


def distillation_loss(logits, teacher_tokens, teacher_logits, mask=None, *, temperature=1.0, reduction="token_mean",
                      scale=1.0):
    """Divergence of the policy from a teacher of which the top logits are known: ``(loss, token_losses)``.
    ``teacher_tokens`` (int64 or int32) and ``teacher_logits`` have one dimension more than the rows, of up to 512
    entries; a negative token is padding.  The teacher's probabilities are the softmax of its logits over the given
    entries, the policy's that over the whole vocabulary, both at ``temperature``; a row's loss is ``temperature**2``
    times the divergence.  ``loss`` carries gradients to the logits, ``token_losses`` is for logging."""
    return _ops.distillation_loss(logits, teacher_tokens, teacher_logits, mask, temperature, _reduction(reduction), scale)


def distillation_loss_and_grad(logits, teacher_tokens, teacher_logits, mask=None, *, temperature=1.0,
                               reduction="token_mean", scale=1.0, out=None):
    """``distillation_loss`` and its gradient at once: ``(loss, grad, token_losses)``; ``out`` as in
    policy_loss_and_grad."""
    return _ops.distillation_loss_and_grad(logits, teacher_tokens, teacher_logits, mask, temperature, _reduction(reduction),
                                           scale, out)
