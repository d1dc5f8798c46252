"""Operators for fine-tuning what chooses in a closed-loop rollout: motion modes (``ProSimHip`` / ``Engine.set_mode_choice``), goals, tokens of a motion
vocabulary.  The engine rolls out (``Engine.set_replicas`` gives M rollouts of a scene) and scores on the device (``Engine.pair_metric``,
``Engine.rollout_metric``); these turn the scores into a step of the model that produced the logits:

  choice_logp(logits, choice)                      log-probability of what was drawn (recorded while rolling out), differentiable
  policy_loss(logits, choice, old_logp, advantage) clipped policy loss with a KL term, differentiable
  preference_loss(better, worse, ...)              loss of pairs of rollouts over their log ratios, differentiable
  clip_grads_(grads, max_norm)                     clipping by the global norm, in place

Plain tensors on the GPU in, tensors out (HIP kernels behind the C ABI of include/prosim_hip.h; no CPU fallback).  Everything is enqueued on torch's
current stream of the tensors' device -- ``torch.cuda.ExternalStream(engine.stream_handle)`` orders it behind an engine's rollout -- nothing
synchronises, every call may be captured into a graph (with ``torch.autograd.grad``; as always in torch, no eager graph of the same leaves may be alive
while a backward pass is captured), and equal inputs at equally aligned addresses give equal bits.  Wrong arguments raise TypeError / ValueError before anything is launched.
"""
from __future__ import annotations

from typing import Iterable, NamedTuple, Optional

import torch

try:
    from . import _finetune
except ImportError as e:      # (never a fallback)
    raise RuntimeError(f"prosim_amd/_finetune.so cannot be loaded ({e}): build it with `python -c 'import __graft_entry__ as g; g.build()'`") from e


class PolicyLoss(NamedTuple):
    """Result of :func:`policy_loss`; only ``loss`` carries a gradient."""
    loss: torch.Tensor        # []
    logp: torch.Tensor        # [...] float32, 0 in masked rows
    kl: torch.Tensor          # [] mean of exp(d) - d - 1, d = ref_logp - logp (0 without ref_logp)
    clip_frac: torch.Tensor   # [] share of the valid rows whose ratio the clipping holds


class PreferenceLoss(NamedTuple):
    """Result of :func:`preference_loss`; only ``loss`` carries a gradient."""
    loss: torch.Tensor        # []
    margin: torch.Tensor      # [pairs] beta * (log ratio of the better rollout - log ratio of the worse one)


def choice_logp(logits: torch.Tensor, choice: torch.Tensor, *, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``log_softmax(logits, -1)[choice]``: the log-probability of every drawn choice, float32.

    ``logits`` [..., K] float32 / bfloat16 / float16 (K from 1 up, any strides; rows that do not lie at one stride are copied), ``choice`` [...]
    int32 / int64, ``mask`` [...] bool / uint8 or None.  Rows with mask 0 are not read and give 0 (and a zero gradient) whatever they hold.  A valid
    row with a choice outside [0, K), a NaN, a +inf, or only -inf gives NaN; single -inf logits are choices that cannot be drawn.  Differentiable in
    ``logits`` (once); a row whose incoming gradient is 0 gets zeros."""
    return _finetune.choice_logp(logits, choice, mask)


def policy_loss(logits: torch.Tensor, choice: torch.Tensor, old_logp: torch.Tensor, advantage: torch.Tensor, *, ref_logp: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None, clip_low: float = 0.2, clip_high: Optional[float] = None, kl_coef: float = 0.0,
                reduction: str = "mean", scale: float = 1.0) -> PolicyLoss:
    """The clipped policy loss over drawn choices, with a KL term to a reference policy.

    Per valid row, ``logp = log_softmax(logits)[choice]``, ``ratio = exp(logp - old_logp)``, ``d = ref_logp - logp``::

        -min(ratio * advantage, clip(ratio, 1 - clip_low, 1 + clip_high) * advantage) + kl_coef * (exp(d) - d - 1)

    averaged over the valid rows (``reduction='mean'``) or summed, times ``scale``.  ``logits``, ``choice``, ``mask`` as in :func:`choice_logp`; ``old_logp``,
    ``advantage``, ``ref_logp`` float32 of the rows' shape (``advantage`` may broadcast to it: one score per rollout), constants.  ``clip_high`` defaults to
    ``clip_low``; ``ref_logp`` is needed when ``kl_coef`` > 0 and only reported as ``kl`` otherwise.  Without a valid row the loss is 0.

    Put the factor of an accumulated or scaled step into ``scale`` rather than multiplying the loss: the forward pass has already written the gradient
    (a buffer of the logits' size lives from it to the backward pass), and a backward pass that arrives with 1 costs nothing more; any other factor is
    right too, and costs another pass over the logits."""
    return PolicyLoss._make(_finetune.policy_loss(logits, choice, old_logp, advantage, ref_logp, mask, clip_low, clip_high, kl_coef, reduction, scale))


def preference_loss(better: torch.Tensor, worse: torch.Tensor, better_ref: Optional[torch.Tensor] = None, worse_ref: Optional[torch.Tensor] = None, *,
                    better_mask: Optional[torch.Tensor] = None, worse_mask: Optional[torch.Tensor] = None, beta: float = 0.1,
                    label_smoothing: float = 0.0, reduction: str = "mean", scale: float = 1.0) -> PreferenceLoss:
    """The preference loss of pairs of rollouts: ``better`` / ``worse`` [pairs, steps] (or [pairs]: sums made elsewhere) float32 log-probabilities of the
    choices (:func:`choice_logp`), ``*_ref`` the same under a reference policy (None: 0), ``*_mask`` the valid steps.  With
    ``h = sum(better - better_ref) - sum(worse - worse_ref)``::

        -(1 - label_smoothing) * ln sigmoid(beta * h) - label_smoothing * ln sigmoid(-beta * h)

    averaged over the pairs or summed, times ``scale``.  The two sides may have different lengths (0 included); masked steps may hold anything and get a zero
    gradient.  Differentiable in ``better`` and ``worse`` (once); the sums are held in 64 bits."""
    return PreferenceLoss._make(_finetune.preference_loss(better, worse, better_ref, worse_ref, better_mask, worse_mask, beta, label_smoothing, reduction, scale))


def clip_grads_(grads: Iterable[Optional[torch.Tensor]], max_norm: float, *, eps: float = 1e-6) -> torch.Tensor:
    """Clip a list of gradients by their global norm, in place; returns the norm before clipping (float32, 0-dim, on the GPU).

    ``norm`` = square root of the sum of all squares (held in 64 bits: it neither overflows nor vanishes while the elements do not); every element is
    multiplied by ``max_norm / (norm + eps)`` if that is below 1.  ``max_norm=inf`` only measures.  Gradients: float32 / bfloat16 / float16, mixed
    freely, dense in any order of dimensions, one device; ``None`` (a parameter without a gradient) and empty tensors are passed over.  Tensors that
    share memory are refused (an element must be scaled once).  A NaN or infinite norm follows the formula (NaN gradients, or zeros): look at the
    returned norm before taking the step."""
    return _finetune.clip_grads(list(grads), max_norm, eps)
