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
while a backward pass is captured), and equal inputs give equal bits.  Wrong arguments raise TypeError / ValueError before anything is launched.
"""
from __future__ import annotations

import ctypes as C
from typing import Iterable, NamedTuple, Optional

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from .engine import PsDecisions, PsPolicyTerms, PsPreference, load_library

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


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


# ---- calling the library --------------------------------------------------------------------------------------------

def _call(device: torch.device, fn, *args):
    """Run a C entry on torch's current stream of ``device``."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        msg = load_library().ps_last_error().decode()
        raise (ValueError if rc == -1 else RuntimeError)(f"prosim_hip error {rc}: {msg}")


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _on_gpu(t, name: str, device=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t).__name__}")
    if t.device.type != "cuda" or t.layout != torch.strided:
        raise ValueError(f"{name}: expected a dense tensor on the GPU, got one on {t.device} ({t.layout})")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors are on {device}")
    return t


def _terms(t, name: str, shape, device, broadcast: bool = False) -> torch.Tensor:
    """A float32 tensor of ``shape`` as dense memory."""
    _on_gpu(t, name, device)
    if t.dtype != torch.float32:
        raise TypeError(f"{name}: expected float32, got {t.dtype}")
    if t.shape != shape:
        if not broadcast:
            raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
        try:
            t = t.expand(shape)
        except RuntimeError:
            raise ValueError(f"{name}: shape {tuple(t.shape)} does not broadcast to {tuple(shape)}") from None
    return t.detach().contiguous()


def _mask(mask, name: str, shape, device) -> Optional[torch.Tensor]:
    if mask is None:
        return None
    _on_gpu(mask, name, device)
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"{name}: expected bool or uint8, got {mask.dtype}")
    if mask.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(mask.shape)}")
    return mask.contiguous()


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """``logits`` with rows that lie at one stride (itself where its strides allow that, else a copy: the caller holds on to it until the launch)."""
    k = logits.shape[-1]
    if logits.is_contiguous():
        return logits
    if logits.stride(-1) == 1 or k == 1:
        step = None       # the stride of the flattened rows, from the innermost leading dimension outwards
        for size, stride in zip(reversed(logits.shape[:-1]), reversed(logits.stride()[:-1])):
            if size == 1:
                continue
            if step is None:
                if stride < k:
                    return logits.contiguous()
                step, span = stride, stride * size
            elif stride != span:
                return logits.contiguous()
            else:
                span = stride * size
        return logits
    return logits.contiguous()


def _row_stride(logits: torch.Tensor) -> int:
    for size, stride in zip(reversed(logits.shape[:-1]), reversed(logits.stride()[:-1])):
        if size != 1:
            return stride
    return logits.shape[-1]


def _decisions(logits: torch.Tensor, choice: torch.Tensor, mask: Optional[torch.Tensor]) -> PsDecisions:
    return PsDecisions(logits.data_ptr(), choice.numel(), logits.shape[-1], _row_stride(logits), _DTYPES[logits.dtype],
                       choice.element_size() * 8, choice.data_ptr(), _ptr(mask))


def _check_decisions(logits, choice, mask):
    _on_gpu(logits, "logits")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits: expected float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] < 1 << 31:
        raise ValueError(f"logits: expected [..., choices] with at least one choice, got shape {tuple(logits.shape)}")
    shape = logits.shape[:-1]
    _on_gpu(choice, "choice", logits.device)
    if choice.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"choice: expected int32 or int64, got {choice.dtype}")
    if choice.shape != shape:
        raise ValueError(f"choice: expected shape {tuple(shape)}, got {tuple(choice.shape)}")
    return shape, choice.contiguous(), _mask(mask, "mask", shape, logits.device)


def _reduction(name: str) -> int:
    if name not in ("mean", "sum"):
        raise ValueError(f"reduction: expected 'mean' or 'sum', got {name!r}")
    return int(name == "mean")


# ---- log-probability of a choice -------------------------------------------------------------------------------------

def _logp_forward(logits, choice, mask, stat):
    lib, dev = load_library(), logits.device
    rows = _rows(logits)
    d = _decisions(rows, choice, mask)
    logp = torch.empty(choice.shape, dtype=torch.float32, device=dev)
    space = torch.empty(lib.ps_choice_workspace(d), dtype=torch.uint8, device=dev)
    _call(dev, lib.ps_choice_logp, d, logp.data_ptr(), _ptr(stat), space.data_ptr(), space.numel())
    return logp


class _ChoiceLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, choice, mask):
        stat = torch.empty((choice.numel(), 2), dtype=torch.float32, device=logits.device)
        logp = _logp_forward(logits, choice, mask, stat)
        ctx.save_for_backward(logits, choice, mask, stat)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        logits, choice, mask, stat = ctx.saved_tensors
        return _choice_grad(logits, choice, mask, stat, grad_out.contiguous(), None, None), None, None


def _choice_grad(logits, choice, mask, stat, coef, gain, done):
    """d / d logits from the rows' coefficients; ``done``: a tensor that already holds the result for gain 1."""
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if done is None else done
    rows = _rows(logits)
    _call(logits.device, load_library().ps_choice_grad, _decisions(rows, choice, mask), coef.data_ptr(), stat.data_ptr(), _ptr(gain),
          int(done is not None), grad.data_ptr())
    return grad


def choice_logp(logits: torch.Tensor, choice: torch.Tensor, *, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``log_softmax(logits, -1)[choice]``: the log-probability of every drawn choice, float32.

    ``logits`` [..., K] float32 / bfloat16 / float16 (K from 1 up, any strides; rows that do not lie at one stride are copied), ``choice`` [...]
    int32 / int64, ``mask`` [...] bool / uint8 or None.  Rows with mask 0 are not read and give 0 (and a zero gradient) whatever they hold.  A valid
    row with a choice outside [0, K), a NaN, a +inf, or only -inf gives NaN; single -inf logits are choices that cannot be drawn.  Differentiable in
    ``logits`` (once); a row whose incoming gradient is 0 gets zeros."""
    _, choice, mask = _check_decisions(logits, choice, mask)
    if logits.requires_grad and torch.is_grad_enabled():
        return _ChoiceLogp.apply(logits, choice, mask)
    return _logp_forward(logits, choice, mask, None)


# ---- clipped policy loss ---------------------------------------------------------------------------------------------

def _policy_forward(logits, choice, mask, terms: PsPolicyTerms, grad, stat, coef):
    lib, dev = load_library(), logits.device
    loss, kl, frac = (torch.empty((), dtype=torch.float32, device=dev) for _ in range(3))
    logp = torch.empty(choice.shape, dtype=torch.float32, device=dev)
    rows = _rows(logits)
    d = _decisions(rows, choice, mask)
    space = torch.empty(lib.ps_choice_workspace(d), dtype=torch.uint8, device=dev)
    _call(dev, lib.ps_policy_loss, d, terms, loss.data_ptr(), kl.data_ptr(), frac.data_ptr(), logp.data_ptr(), _ptr(stat), _ptr(coef), _ptr(grad),
          space.data_ptr(), space.numel())
    return loss, logp, kl, frac


class _PolicyLoss(torch.autograd.Function):
    """The gradient is written by the forward pass, which has the row at hand once its sum is known (one read of the logits instead of two); the
    backward pass finds it ready when the incoming gradient is 1 and computes it afresh from the rows' statistics otherwise."""

    @staticmethod
    def forward(ctx, logits, choice, mask, terms):
        n, dev = choice.numel(), logits.device
        stat = torch.empty((n, 2), dtype=torch.float32, device=dev)
        coef = torch.empty((n,), dtype=torch.float32, device=dev)
        ctx.ready = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        out = _policy_forward(logits, choice, mask, terms, ctx.ready, stat, coef)
        ctx.save_for_backward(logits, choice, mask, stat, coef)
        ctx.mark_non_differentiable(*out[1:])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        logits, choice, mask, stat, coef = ctx.saved_tensors
        ready, ctx.ready = ctx.ready, None       # (handed out once: a second backward pass of a retained graph computes its own)
        return _choice_grad(logits, choice, mask, stat, coef, grad_loss.contiguous(), ready), None, None, None


def policy_loss(logits: torch.Tensor, choice: torch.Tensor, old_logp: torch.Tensor, advantage: torch.Tensor, *, ref_logp: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None, clip_low: float = 0.2, clip_high: Optional[float] = None, kl_coef: float = 0.0,
                reduction: str = "mean", scale: float = 1.0) -> PolicyLoss:
    """The clipped policy loss over drawn choices, with a KL term to a reference policy.

    Per valid row, ``logp = log_softmax(logits)[choice]``, ``ratio = exp(logp - old_logp)``, ``d = ref_logp - logp``::

        -min(ratio * advantage, clip(ratio, 1 - clip_low, 1 + clip_high) * advantage) + kl_coef * (exp(d) - d - 1)

    averaged over the valid rows (``reduction='mean'``) or summed, times ``scale``.  ``logits``, ``choice``, ``mask`` as in :func:`choice_logp`; ``old_logp``,
    ``advantage``, ``ref_logp`` float32 of the rows' shape (``advantage`` may broadcast to it: one score per rollout), constants.  ``clip_high`` defaults to
    ``clip_low``; ``ref_logp`` is needed when ``kl_coef`` > 0 and only reported as ``kl`` otherwise.  Without a valid row the loss is 0.

    Put the factor of an accumulated or scaled step into ``scale`` rather than multiplying the loss: the forward pass has already written the gradient,
    and a backward pass that arrives with 1 costs nothing more."""
    shape, choice, mask = _check_decisions(logits, choice, mask)
    dev = logits.device
    old_logp = _terms(old_logp, "old_logp", shape, dev)
    advantage = _terms(advantage, "advantage", shape, dev, broadcast=True)
    ref_logp = None if ref_logp is None else _terms(ref_logp, "ref_logp", shape, dev)
    if kl_coef > 0 and ref_logp is None:
        raise ValueError("kl_coef > 0 needs ref_logp")
    terms = PsPolicyTerms(old_logp.data_ptr(), advantage.data_ptr(), _ptr(ref_logp), clip_low, clip_low if clip_high is None else clip_high, kl_coef, scale,
                          _reduction(reduction))
    if logits.requires_grad and torch.is_grad_enabled():
        return PolicyLoss(*_PolicyLoss.apply(logits, choice, mask, terms))
    return PolicyLoss(*_policy_forward(logits, choice, mask, terms, None, None, None))


# ---- preference loss -------------------------------------------------------------------------------------------------

class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, better, worse, q, masks):
        lib, dev = load_library(), better.device
        loss = torch.empty((), dtype=torch.float32, device=dev)
        margin, coef = (torch.empty((q.pairs,), dtype=torch.float32, device=dev) for _ in range(2))
        space = torch.empty(lib.ps_preference_loss_workspace(q.pairs), dtype=torch.uint8, device=dev)
        _call(dev, lib.ps_preference_loss, q, loss.data_ptr(), margin.data_ptr(), coef.data_ptr(), space.data_ptr(), space.numel())
        ctx.save_for_backward(coef, *masks)
        ctx.q, ctx.shapes = q, (better.shape, worse.shape)
        ctx.mark_non_differentiable(margin)
        return loss, margin

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        coef = ctx.saved_tensors[0]      # (the masks are saved with it: q holds their addresses)
        grads = [torch.empty(s, dtype=torch.float32, device=coef.device) if need else None for s, need in zip(ctx.shapes, ctx.needs_input_grad)]
        _call(coef.device, load_library().ps_preference_grad, ctx.q, coef.data_ptr(), grad_loss.contiguous().data_ptr(), _ptr(grads[0]), _ptr(grads[1]))
        return grads[0], grads[1], None, None


def preference_loss(better: torch.Tensor, worse: torch.Tensor, better_ref: Optional[torch.Tensor] = None, worse_ref: Optional[torch.Tensor] = None, *,
                    better_mask: Optional[torch.Tensor] = None, worse_mask: Optional[torch.Tensor] = None, beta: float = 0.1,
                    label_smoothing: float = 0.0, reduction: str = "mean", scale: float = 1.0) -> PreferenceLoss:
    """The preference loss of pairs of rollouts: ``better`` / ``worse`` [pairs, steps] (or [pairs]: sums made elsewhere) float32 log-probabilities of the
    choices (:func:`choice_logp`), ``*_ref`` the same under a reference policy (None: 0), ``*_mask`` the valid steps.  With
    ``h = sum(better - better_ref) - sum(worse - worse_ref)``::

        -(1 - label_smoothing) * ln sigmoid(beta * h) - label_smoothing * ln sigmoid(-beta * h)

    averaged over the pairs or summed, times ``scale``.  The two sides may have different lengths (0 included); masked steps may hold anything and get a zero
    gradient.  Differentiable in ``better`` and ``worse`` (once); the sums are held in 64 bits."""
    dev = _on_gpu(better, "better").device
    _on_gpu(worse, "worse", dev)
    if better.dim() not in (1, 2) or worse.dim() not in (1, 2) or better.shape[0] != worse.shape[0] or better.shape[0] < 1:
        raise ValueError(f"better / worse: expected [pairs, steps] or [pairs] with the same pairs >= 1, got {tuple(better.shape)} and {tuple(worse.shape)}")
    tensors = []
    for name, t, ref, mask in (("better", better, better_ref, better_mask), ("worse", worse, worse_ref, worse_mask)):
        tensors.append((_terms(t, name, t.shape, dev), None if ref is None else _terms(ref, name + "_ref", t.shape, dev), _mask(mask, name + "_mask", t.shape, dev)))
    (b, b_ref, b_mask), (w, w_ref, w_mask) = tensors
    steps = [t.shape[1] if t.dim() == 2 else 1 for t in (better, worse)]
    q = PsPreference(b.data_ptr(), _ptr(b_ref), w.data_ptr(), _ptr(w_ref), _ptr(b_mask), _ptr(w_mask), better.shape[0], steps[0], steps[1], beta, label_smoothing,
                     scale, _reduction(reduction))
    return PreferenceLoss(*_PreferenceLoss.apply(better, worse, q, (b_mask, w_mask)))


# ---- gradient clipping -----------------------------------------------------------------------------------------------

def _dense(t: torch.Tensor) -> bool:
    """Every element of the tensor's stretch of memory belongs to it exactly once (in whatever order of dimensions)."""
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def clip_grads_(grads: Iterable[Optional[torch.Tensor]], max_norm: float, *, eps: float = 1e-6) -> torch.Tensor:
    """Clip a list of gradients by their global norm, in place; returns the norm before clipping (float32, 0-dim, on the GPU).

    ``norm`` = square root of the sum of all squares (held in 64 bits: it neither overflows nor vanishes while the elements do not); every element is
    multiplied by ``max_norm / (norm + eps)`` if that is below 1.  ``max_norm=inf`` only measures.  Gradients: float32 / bfloat16 / float16, mixed
    freely, dense in any order of dimensions, one device; ``None`` (a parameter without a gradient) and empty tensors are passed over.  Tensors that
    share memory are refused (an element must be scaled once).  A NaN or infinite norm follows the formula (NaN gradients, or zeros): look at the
    returned norm before taking the step."""
    ts = [t for t in grads if t is not None]
    if not ts:
        raise ValueError("clip_grads_: no gradients")
    for t in ts:
        _on_gpu(t, "grads", ts[0].device)
        if t.dtype not in _DTYPES:
            raise TypeError(f"grads: expected float32, bfloat16 or float16, got {t.dtype}")
        if t.requires_grad:
            raise ValueError("grads: a tensor requires a gradient itself (parameters instead of their gradients?)")
        if not t.is_contiguous() and not _dense(t):
            raise ValueError(f"grads: a tensor of shape {tuple(t.shape)} and strides {t.stride()} is not dense")
    dev = ts[0].device
    ptr = np.array([t.data_ptr() for t in ts], np.uint64)
    numel = np.array([t.numel() for t in ts], np.int64)
    dtype = np.array([_DTYPES[t.dtype] for t in ts], np.int32)
    used = np.flatnonzero(numel)
    order = used[np.argsort(ptr[used], kind="stable")]
    ends = ptr[order] + (numel[order] * np.where(dtype[order] == 0, 4, 2)).astype(np.uint64)
    if (ends[:-1] > ptr[order][1:]).any():
        raise ValueError("grads: two tensors share memory")
    lib = load_library()
    norm = torch.empty((), dtype=torch.float32, device=dev)
    space = torch.empty(lib.ps_clip_grads_workspace(len(ts), numel.ctypes.data), dtype=torch.uint8, device=dev)
    _call(dev, lib.ps_clip_grads, len(ts), ptr.ctypes.data, numel.ctypes.data, dtype.ctypes.data, max_norm, eps, norm.data_ptr(), space.data_ptr(), space.numel())
    torch.autograd.graph.increment_version(ts)
    return norm
