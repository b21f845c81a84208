"""Cross entropy of a language-model head straight from the hidden states, without its logits.

``cross_entropy`` takes logits: at 8192 tokens and 151 936 entries they are 5 GB in float32, and their softmax and gradient as much
again.  Here the head's product, the softmax and the gradients go through the vocabulary in pieces: the forward pass keeps one
log-sum-exp per token, the backward pass makes each piece of the logits again.  CUDA tensors run csrc/cuda/linear_ce.cu, CPU tensors
the same steps in torch.

Reference: crates/oxibonsai-model/src/losses.rs (cross-entropy, label smoothing, next-token loss over logits).
"""
from __future__ import annotations

import torch

from ..ops import train_ops

_PIECE = 8192         # vocabulary rows of a piece on the CPU


def _cpu_forward(hidden, weight, targets, ignore_index, reduction, smoothing):
    live = targets != ignore_index
    if bool(((targets < 0) | (targets >= weight.shape[0]))[live].any()):
        raise IndexError(f"linear_cross_entropy: a target is outside the vocabulary of {weight.shape[0]}")
    kind = torch.float64 if hidden.dtype == torch.float64 else torch.float32
    h, top = hidden[live].to(kind), None
    total = torch.zeros(len(h), dtype=kind)
    sums, at = torch.zeros(len(h), dtype=kind), (h * weight[targets[live]].to(kind)).sum(1)
    for w in weight.split(_PIECE):
        z = h @ w.to(kind).T
        new = z.max(1).values if top is None else torch.maximum(top, z.max(1).values)
        total = (0.0 if top is None else total * (top - new).exp()) + (z - new[:, None]).exp().sum(1)
        sums, top = sums + z.sum(1), new
    lse = top + total.log()
    loss = torch.zeros(len(targets), dtype=kind).masked_scatter(live, lse - (1 - smoothing) * at - smoothing / len(weight) * sums)
    if reduction == "mean":
        loss = loss.sum() / live.sum()
    elif reduction == "sum":
        loss = loss.sum()
    return loss, live, lse


def _cpu_backward(hidden, weight, targets, live, lse, up, reduction, smoothing, want_hidden, want_weight):
    kind = lse.dtype
    h, t = hidden[live].to(kind), targets[live]
    each = up[live] if reduction == "none" else (up / live.sum() if reduction == "mean" else up).expand(len(h))
    dh = torch.zeros_like(h) if want_hidden else None
    dw = torch.empty_like(weight) if want_weight else None
    for c in range(0, len(weight), _PIECE):
        w = weight[c:c + _PIECE].to(kind)
        dz = (h @ w.T - lse[:, None]).exp() - smoothing / len(weight)
        inside = ((t >= c) & (t < c + len(w))).nonzero().flatten()
        dz[inside, t[inside] - c] -= 1 - smoothing
        dz *= each[:, None]
        if want_hidden:
            dh += dz @ w
        if want_weight:
            dw[c:c + _PIECE] = (dz.T @ h).to(dw.dtype)
    if want_hidden:
        dh = torch.zeros_like(hidden).masked_scatter(live[:, None].expand_as(hidden), dh.to(hidden.dtype))
    return dh, dw


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction, smoothing):
        if hidden.is_cuda:
            loss, kept = train_ops.linear_ce_forward(hidden, weight, targets, ignore_index, reduction, smoothing)
            ctx.save_for_backward(weight, kept)
        else:
            loss, live, lse = _cpu_forward(hidden, weight, targets, ignore_index, reduction, smoothing)
            ctx.save_for_backward(weight, hidden, live, targets, lse)
        ctx.rows = len(hidden)
        ctx.reduction, ctx.smoothing = reduction, smoothing
        return loss

    @staticmethod
    def backward(ctx, up):
        if torch.is_grad_enabled():
            raise RuntimeError("linear_cross_entropy: its gradients cannot be differentiated again (create_graph=True)")
        weight, *rest = ctx.saved_tensors
        want = ctx.needs_input_grad[:2]
        if weight.is_cuda:
            dh, dw = train_ops.linear_ce_backward(weight, rest[0], ctx.rows, up.contiguous(), ctx.reduction, ctx.smoothing, *want)
        else:
            hidden, live, targets, lse = rest
            dh, dw = _cpu_backward(hidden, weight, targets, live, lse, up, ctx.reduction, ctx.smoothing, *want)
        return dh, dw, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100, reduction: str = "mean",
                         label_smoothing: float = 0.0) -> torch.Tensor:
    """Cross entropy of the logits ``hidden @ weight.T`` against ``targets``, differentiable in ``hidden`` and ``weight``.

    ``hidden`` [..., d] and ``weight`` [vocab, d] have one type (float32, float16 or bfloat16; on the CPU float64 too), ``targets`` [...]
    are int64 or int32; there are less than 2^30 tokens and vocabulary rows, of at most 2^24 values.  Tokens with ``ignore_index`` have
    loss 0 and no gradient, whatever their hidden row holds; ``reduction`` is "mean" over the others (NaN where there are none), "sum" or
    "none" (a loss of the shape of ``targets``).  The target distribution is ``(1 - label_smoothing)`` at the target plus
    ``label_smoothing / vocab`` everywhere.  The loss is float32 (float64 of float64), gradients have the inputs' type; logits, sums and products are float32 whatever the inputs, and on the GPU the gradient of the logits is rounded to the
    inputs' type before it is multiplied, as a product of that type does.  A target outside the vocabulary raises on the CPU; on the GPU,
    where nothing waits for the result, its loss and the gradients that it enters are NaN.  float16 gradients underflow as everywhere:
    scale the loss; with "none" the GPU holds the gradient of the logits in steps of 2^-39 of the largest finite upstream gradient of the
    call.  A token whose upstream gradient is not finite has no finite gradient, and neither has the head; other tokens' are as without it.

    On the GPU nothing is read back and all memory comes from torch's allocator, so that a pass and its gradients can be captured into a
    CUDA graph; as with every operator of torch, no eager graph of the same leaves may be alive while a backward pass is captured.
    Second derivatives are refused.  Between the passes the live rows of ``hidden`` are kept (a copy) with 16 bytes per token; changing
    ``weight`` in between is an error that autograd reports."""
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: hidden [..., d] and weight [vocab, d] are wanted, got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: targets of shape {tuple(hidden.shape[:-1])} are wanted, got {tuple(targets.shape)}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"linear_cross_entropy: targets are int64 or int32, got {targets.dtype}")
    if reduction not in train_ops.REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction is one of {', '.join(train_ops.REDUCTIONS)}, got {reduction!r}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"linear_cross_entropy: label_smoothing is between 0 and 1, got {label_smoothing}")
    if not hidden.device == weight.device == targets.device:
        raise ValueError(f"linear_cross_entropy: tensors of one device are wanted, got {hidden.device}, {weight.device} and {targets.device}")
    if hidden.device.type not in ("cuda", "cpu"):
        raise ValueError(f"linear_cross_entropy: CUDA or CPU tensors are wanted, got {hidden.device}")
    types = (torch.float32, torch.float16, torch.bfloat16) + (() if hidden.is_cuda else (torch.float64,))
    if hidden.dtype != weight.dtype or hidden.dtype not in types:
        raise TypeError(f"linear_cross_entropy: hidden and weight of one type (float32, float16, bfloat16) are wanted, got {hidden.dtype} and {weight.dtype}")
    if min(weight.shape) < 1 or max(*weight.shape, targets.numel()) >= 2 ** 30:
        raise ValueError(f"linear_cross_entropy: a vocabulary and a width of at least 1 and less than 2^30 are wanted, got {tuple(weight.shape)} and "
                         f"{targets.numel()} targets")
    if weight.shape[1] > 2 ** 24:
        raise ValueError(f"linear_cross_entropy: rows of at most 2^24 values are wanted, got {weight.shape[1]}")
    flat = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    if targets.numel() == 0:
        kind = torch.float64 if flat.dtype == torch.float64 else torch.float32
        loss = flat.to(kind).sum(1) + weight[:0].to(kind).sum()                # zero gradients of both
        return loss.sum() * float("nan") if reduction == "mean" else loss.sum() if reduction == "sum" else loss.reshape(targets.shape)
    if flat.is_cuda:
        flat = flat if flat.is_contiguous() or (flat.stride(1) == 1 and flat.stride(0) >= flat.shape[1]) else flat.contiguous()
        weight = weight if weight.is_contiguous() or (weight.stride(1) == 1 and weight.stride(0) >= weight.shape[1]) else weight.contiguous()
    loss = _LinearCrossEntropy.apply(flat, weight, targets.reshape(-1).long().contiguous(), ignore_index, reduction, float(label_smoothing))
    return loss.reshape(targets.shape) if reduction == "none" and targets.dim() != 1 else loss


def linear_ntp_loss(hidden: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
    """``ntp_loss`` from hidden states: position t predicts token t + 1."""
    return linear_cross_entropy(hidden[:-1], weight, tokens[1:])


@torch.no_grad()
def linear_sequence_perplexity(hidden: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor) -> float:
    """``sequence_perplexity`` from hidden states."""
    return float(torch.exp(linear_ntp_loss(hidden, weight, tokens)))
