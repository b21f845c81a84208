"""Losses that a model is tuned with from the log-probabilities of its tokens: of preferred against rejected answers, and of a policy whose ratio
to an earlier one is clipped, with a penalty for leaving a reference.

Both stand behind ``linear_cross_entropy(..., reduction="none")``, whose negative is a log-probability for every token.  CUDA tensors run
csrc/cuda/tuning_loss.cu (two launches for a loss, one for its gradient), CPU tensors the same formulas in torch.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from ..ops import train_ops
from .counter_dropout import has_tangent, rows_of

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor                  # float32: 0-dim, or of every pair
    chosen_rewards: torch.Tensor        # float32 [pairs]: beta times the chosen answer's log-ratio; no gradient
    rejected_rewards: torch.Tensor


class PolicyLoss(NamedTuple):
    loss: torch.Tensor                  # float32: 0-dim, or of every token
    kl: torch.Tensor                    # float32, 0-dim: mean estimate of the divergence from the reference over the live tokens; no gradient
    clipped: torch.Tensor               # float32, 0-dim: share of the live tokens whose ratio is clipped


def _check(what, logps, others, mask) -> None:
    if logps.dim() != 2:
        raise ValueError(f"{what}: log-probabilities [sequences, tokens] are wanted, got {tuple(logps.shape)}")
    if logps.device.type not in ("cuda", "cpu"):
        raise ValueError(f"{what}: CUDA or CPU tensors are wanted, got {logps.device}")
    if logps.dtype not in _TYPES + (() if logps.is_cuda else (torch.float64,)):
        raise TypeError(f"{what}: float32, float16 or bfloat16 log-probabilities are wanted, got {logps.dtype}")
    for name, t in others.items():
        if t is None:
            continue
        if t.shape != logps.shape or t.dtype != logps.dtype or t.device != logps.device:
            raise ValueError(f"{what}: {name} of the shape, type and device of logps ({tuple(logps.shape)}, {logps.dtype}, {logps.device}) is wanted, got "
                             f"{tuple(t.shape)}, {t.dtype}, {t.device}")
        if (t.requires_grad and torch.is_grad_enabled()) or has_tangent(t):
            raise ValueError(f"{what}: {name} has no gradient: detach it")
    if mask is not None and (mask.shape != logps.shape or mask.dtype != torch.bool or mask.device != logps.device):
        raise ValueError(f"{what}: a bool mask of shape {tuple(logps.shape)} on {logps.device} is wanted, got {mask.dtype} {tuple(mask.shape)} on {mask.device}")
    if logps.numel() >= 2 ** 40 or max(logps.shape) >= 2 ** 30:
        raise ValueError(f"{what}: less than 2^30 sequences and tokens are wanted, got {tuple(logps.shape)}")


def _rows(t):
    return None if t is None else rows_of(t.detach() if t.requires_grad else t)


class _Loss(torch.autograd.Function):
    """A loss that its kernels have made already: what it kept, and the gradient of the log-probabilities from that."""

    @staticmethod
    def forward(ctx, logps, made):
        loss, kept, mask, ctx.tokens, ctx.what = made
        ctx.save_for_backward(kept, mask)
        ctx.shape, ctx.dtype = logps.shape, logps.dtype
        return loss

    @staticmethod
    def backward(ctx, up):
        if torch.is_grad_enabled() or has_tangent(up):
            raise RuntimeError(f"{ctx.what}: its gradients cannot be differentiated again (create_graph=True, or a tangent of the gradient)")
        kept, mask = ctx.saved_tensors
        return train_ops.tune_scale(kept, ctx.tokens, up.contiguous(), mask, ctx.shape, ctx.dtype), None


# ---- preference pairs --------------------------------------------------------------------------------------------------------------------
def _preference_cpu(logps, ref, mask, beta, kind, smoothing, average, reduction):
    wide = logps.double()
    d = wide if ref is None else wide - ref.double()
    live = torch.ones_like(logps, dtype=torch.bool) if mask is None else mask
    s = torch.where(live, d, 0.0).sum(1)
    if average:
        s = s / live.sum(1).clamp(min=1)
    chosen, rejected = s.chunk(2)
    z = chosen - rejected
    if kind == "sigmoid":
        log = torch.nn.functional.logsigmoid
        each = (smoothing - 1) * log(beta * z) - (smoothing * log(-beta * z) if smoothing else 0.0)
    elif kind == "hinge":
        each = torch.where(beta * z >= 1.0, 0.0, 1.0 - beta * z)              # flat from the corner on, NaN of NaN
    else:
        each = (z - 0.5 / beta) ** 2
    loss = each.mean() if reduction == "mean" else each.sum() if reduction == "sum" else each
    out = torch.float64 if logps.dtype == torch.float64 else torch.float32
    return PreferenceLoss(loss.to(out), (beta * chosen).detach().to(out), (beta * rejected).detach().to(out))


def preference_loss(logps: torch.Tensor, ref_logps: torch.Tensor | None, mask: torch.Tensor | None = None, beta: float = 0.1, kind: str = "sigmoid",
                    label_smoothing: float = 0.0, average: bool = False, reduction: str = "mean") -> PreferenceLoss:
    """Loss of preferred answers against rejected ones, differentiable in ``logps``.

    ``logps`` [2 * pairs, tokens]: log-probabilities of the answers' tokens under the model, the chosen answers first, the rejected ones behind them in the same
    order; ``ref_logps``: those of the reference model (None: a loss without one); ``mask`` (bool): the tokens that count, whatever the others hold.  With
    ``s`` the sum of ``logps - ref_logps`` over an answer (``average``: its mean, 0 of an answer without tokens) and ``z = s_chosen - s_rejected``, ``kind`` is

    * "sigmoid": ``(1 - label_smoothing) * -log sigmoid(beta z) + label_smoothing * -log sigmoid(-beta z)``,
    * "hinge": ``max(0, 1 - beta z)``, whose gradient is 0 at ``beta z = 1``,
    * "ipo": ``(z - 1 / (2 beta))^2``,

    and ``reduction`` is "mean" over the pairs, "sum" or "none".  Returns the loss and the rewards ``beta s`` of the chosen and of the rejected answers.  Differences
    and sums are float64, the loss is float32 (float64 of float64, on the CPU), the gradient has the type of ``logps`` and is 0 at masked tokens.  Nothing is read back;
    second and forward-mode derivatives are refused on the GPU."""
    what = "preference_loss"
    _check(what, logps, {"ref_logps": ref_logps}, mask)
    if logps.shape[0] % 2:
        raise ValueError(f"{what}: chosen answers and as many rejected ones are wanted, got {logps.shape[0]} sequences")
    if kind not in train_ops.PREFERENCE_KINDS:
        raise ValueError(f"{what}: kind is one of {', '.join(train_ops.PREFERENCE_KINDS)}, got {kind!r}")
    if reduction not in train_ops.REDUCTIONS:
        raise ValueError(f"{what}: reduction is one of {', '.join(train_ops.REDUCTIONS)}, got {reduction!r}")
    if not (beta > 0.0 and math.isfinite(beta)):
        raise ValueError(f"{what}: beta is above 0, got {beta}")
    if not 0.0 <= label_smoothing <= 1.0 or (label_smoothing and kind != "sigmoid"):
        raise ValueError(f"{what}: label_smoothing is between 0 and 1 and for the sigmoid loss, got {label_smoothing} for {kind}")
    if not logps.is_cuda or logps.numel() == 0:
        return _preference_cpu(logps, ref_logps, mask, float(beta), kind, float(label_smoothing), average, reduction)
    wants_grad = (torch.is_grad_enabled() and logps.requires_grad) or has_tangent(logps)
    rows, mask = rows_of(logps), _rows(mask)
    loss, rewards, kept = train_ops.preference_forward(rows, _rows(ref_logps), mask, float(beta), kind, float(label_smoothing), bool(average), reduction, wants_grad)
    return PreferenceLoss(_Loss.apply(rows, (loss, kept, mask, False, what)) if wants_grad else loss, *rewards.chunk(2))


# ---- clipped policy ratio ----------------------------------------------------------------------------------------------------------------
def _policy_cpu(logps, old, ref, mask, gain, clip, kl_weight, reduction):
    kind = torch.float64 if logps.dtype == torch.float64 else torch.float32
    live = torch.ones_like(logps, dtype=torch.bool) if mask is None else mask
    at = live.nonzero(as_tuple=True)
    l, g = logps[at].to(kind), (gain if gain.dim() == 2 else gain[:, None]).expand_as(logps)[at].to(kind)
    step = l - (l.detach() if old is None else old[at].to(kind))
    far = l.detach().double() - (l.detach().double() if old is None else old[at].double())
    high, low = (g > 0) & (far > math.log1p(clip[1])), (g < 0) & (far < (math.log1p(-clip[0]) if clip[0] < 1 else -math.inf))
    cut = high | low
    gained = torch.where(cut | (g == 0), 0.0, step).exp() * g         # an exponential that overflows enters neither pass
    each = -torch.where(cut, torch.where(high, 1 + clip[1] if math.isfinite(clip[1]) else 1.0, 1 - clip[0]) * g, gained)
    kl = torch.zeros_like(l)
    if ref is not None:
        back = ref[at].to(kind) - l
        kl = torch.expm1(back) - back
        if kl_weight:
            each = each + kl_weight * kl
    per = logps.new_zeros(logps.shape, dtype=kind).index_put(at, each)
    size, total = live.sum(1), per.sum(1, dtype=torch.float64)
    if reduction == "none":
        loss = per
    elif reduction == "sum":
        loss = total.sum()
    elif reduction == "tokens":
        loss = total.sum() / size.sum()
    else:
        loss = (total / size.clamp(min=1)).sum() / (size > 0).sum()
    return PolicyLoss(loss.to(kind), (kl.detach().sum(dtype=torch.float64) / size.sum()).to(kind), (cut.sum(dtype=torch.float64) / size.sum()).to(kind))


def policy_loss(logps: torch.Tensor, old_logps: torch.Tensor | None, advantages: torch.Tensor, mask: torch.Tensor | None = None,
                ref_logps: torch.Tensor | None = None, clip: tuple[float, float] = (0.2, 0.2), kl_weight: float = 0.0, reduction: str = "tokens") -> PolicyLoss:
    """Policy loss over clipped probability ratios with a penalty for leaving a reference, differentiable in ``logps``.

    ``logps`` [sequences, tokens]: log-probabilities of the sampled tokens under the model, ``old_logps`` under the policy that sampled them (None: the model
    itself, a ratio of 1), ``ref_logps`` under the reference (None: no penalty), ``advantages`` [sequences] or [sequences, tokens] (no gradient), ``mask`` (bool) the
    tokens that count, whatever the others hold.  With ``ratio = exp(logps - old_logps)`` and ``gap = ref_logps - logps`` a token's loss is

        ``-min(ratio * advantage, clamp(ratio, 1 - clip[0], 1 + clip[1]) * advantage) + kl_weight * (exp(gap) - gap - 1)``

    ``reduction``: "tokens" is the mean over all live tokens, "sequences" the mean over the sequences that have live tokens of each one's mean, "sum", or "none"
    (a loss of the shape of ``logps``, 0 at masked tokens); means of nothing are NaN, with a gradient of 0.  A clipped token has no gradient but the penalty's;
    whether it is clipped is decided on ``logps - old_logps`` in float64.  An advantage of 0 leaves the penalty alone, also where the ratio is infinite.  Returns
    the loss, the mean of ``exp(gap) - gap - 1`` and the share of clipped tokens.  Sums are float64 (on the GPU over fours that are added in
    float32), losses float32 (float64 of float64, on the CPU), the gradient has the type of ``logps``.  Between the passes four bytes for every token are kept.  Nothing is read back; second and forward-mode derivatives are refused on the GPU."""
    what = "policy_loss"
    _check(what, logps, {"old_logps": old_logps, "ref_logps": ref_logps}, mask)
    if advantages.shape not in (logps.shape[:1], logps.shape) or advantages.device != logps.device or not advantages.is_floating_point():
        raise ValueError(f"{what}: floating advantages of shape {tuple(logps.shape[:1])} or {tuple(logps.shape)} on {logps.device} are wanted, got "
                         f"{advantages.dtype} {tuple(advantages.shape)} on {advantages.device}")
    if (advantages.requires_grad and torch.is_grad_enabled()) or has_tangent(advantages):
        raise ValueError(f"{what}: advantages have no gradient: detach them")
    if len(clip) != 2 or not 0.0 <= clip[0] <= 1.0 or not clip[1] >= 0.0:
        raise ValueError(f"{what}: clip is (low, high) with low from 0 to 1 and high from 0 on, got {clip}")
    if reduction not in train_ops.POLICY_REDUCTIONS:
        raise ValueError(f"{what}: reduction is one of {', '.join(train_ops.POLICY_REDUCTIONS)}, got {reduction!r}")
    if not math.isfinite(kl_weight) or (kl_weight and ref_logps is None):
        raise ValueError(f"{what}: a finite kl_weight, and ref_logps with it, are wanted, got {kl_weight}")
    clip = float(clip[0]), float(clip[1])
    if not logps.is_cuda or logps.numel() == 0:
        return _policy_cpu(logps, old_logps, ref_logps, mask, advantages, clip, float(kl_weight), reduction)
    gain = _rows(advantages.float()) if advantages.dim() == 2 else advantages.detach().float()
    wants_grad = (torch.is_grad_enabled() and logps.requires_grad) or has_tangent(logps)
    rows = rows_of(logps)
    loss, stats, kept = train_ops.policy_forward(rows, _rows(old_logps), _rows(ref_logps), _rows(mask), gain, clip, float(kl_weight), reduction, wants_grad)
    return PolicyLoss(_Loss.apply(rows, (loss, kept, None, True, what)) if wants_grad else loss, *stats.unbind())
