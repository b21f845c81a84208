"""Torch-facing wrappers of the training kernels in ``libbonsai_cuda.so`` (csrc/cuda/multi_tensor.cu, linear_ce.cu, dropout.cu,
low_rank.cu, tuning_loss.cu).

Every function launches on torch's current stream of the tensors' device.  As in :mod:`cuda_ops` there is no PyTorch fallback:
CUDA tensors go through the kernels, and a missing library raises.
"""
from __future__ import annotations

import array
import contextlib
import ctypes as C
from typing import Sequence

import torch

from . import cuda_ops as K

_vp, _i, _d, _ll, _u64, _f = C.c_void_p, C.c_int, C.c_double, C.c_longlong, C.c_uint64, C.c_float
_SIG = {
    "bonsai_mt_partials": [_i],
    "bonsai_mt_norm": [_i, _vp, _vp, _vp, _vp, _vp, _vp],
    "bonsai_mt_clip": [_i, _vp, _vp, _vp, _vp, _vp, _d, _vp, _vp, _vp],
    "bonsai_ce_bytes": [_vp, _ll, _i, _i, _i, _i, C.c_float, _i],
    "bonsai_ce_forward": [_vp, _ll, _vp, _ll, _vp, _i, _i, _i, _i, _ll, _i, C.c_float, _vp, _ll, _vp, _vp, _ll, _vp],
    "bonsai_ce_backward": [_vp, _ll, _i, _i, _i, _i, _i, C.c_float, _vp, _ll, _vp, _vp, _vp, _vp, _ll, _vp],
    "bonsai_mt_adam": [_i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _d, _vp, _d, _d, _d, _d, _i, _vp, _d, _vp, _vp, _vp],
    "bonsai_dropout": [_vp, _ll, _vp, _ll, _ll, _i, _u64, _vp, _i, _vp],
    "bonsai_lr_self_rows": [],
    "bonsai_lr_bytes": [_i, _i, _i, _i, _i, _i, _i, _i, _i],
    "bonsai_lr_forward": [_vp, _ll, _vp, _vp, _vp, _ll, _vp, _ll, _vp, _f, _i, _i, _i, _i, _i, _i, _vp, _i, _vp, _ll, _i, _u64, _vp, _i, _vp],
    "bonsai_lr_backward": [_vp, _ll, _vp, _ll, _vp, _vp, _vp, _vp, _vp, _vp, _f, _i, _i, _i, _i, _i, _i, _i, _vp, _ll, _i, _vp, _ll, _u64, _vp, _i, _vp],
    "bonsai_tune_bytes": [_ll, _ll, _i],
    "bonsai_policy_loss": [_vp, _ll, _vp, _ll, _vp, _ll, _vp, _ll, _vp, _ll, _i, _ll, _ll, _i, _d, _d, _d, _i, _vp, _vp, _vp, _ll, _i, _vp],
    "bonsai_preference_loss": [_vp, _ll, _vp, _ll, _vp, _ll, _ll, _ll, _i, _i, _i, _i, _d, _d, _vp, _vp, _vp, _ll, _i, _vp],
    "bonsai_tune_scale": [_vp, _ll, _i, _vp, _i, _ll, _vp, _ll, _ll, _ll, _i, _vp, _vp],
}
_declared = False
_HERE = contextlib.nullcontext()
TYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _lib():
    global _declared
    l = K.lib()
    if not _declared:
        K.declare(_SIG, {"bonsai_mt_partials": _ll, "bonsai_ce_bytes": _ll, "bonsai_tune_bytes": _ll, "bonsai_lr_bytes": _ll})
        _declared = True
    return l


def _on(device: torch.device):
    """A context in which ``device`` is the current one."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    """The current stream's handle, without a stream object around it."""
    return torch._C._cuda_getCurrentRawStream(device.index)


# ---- many tensors ---------------------------------------------------------------------------------------------------------------
class TensorTable:
    """Addresses, sizes and types of dense CUDA tensors of one device, packed for the kernels.  Tensors without values are left out.
    ``like``: the table of as many tensors of the same sizes (others are refused).  ``keep``: the memory stays allocated as long as the
    table is there, whatever becomes of the tensors."""

    def __init__(self, tensors: Sequence[torch.Tensor], like: "TensorTable | None" = None, keep: bool = False):
        self.memory = [t.untyped_storage() for t in tensors] if keep else None
        self.sizes = [t.numel() for t in tensors]
        if like is not None and self.sizes != like.sizes:
            raise ValueError("TensorTable: tensors of the sizes of the other table are wanted")
        if 0 in self.sizes:
            tensors = [t for t, n in zip(tensors, self.sizes) if n]
        self.n = len(tensors)
        # an optimizer makes a table for each of its steps: arrays from buffers, not element by element
        self.ptrs = (C.c_void_p * max(1, self.n)).from_buffer(array.array("Q", [t.data_ptr() for t in tensors] or [0]))
        self.types = (C.c_ubyte * max(1, self.n)).from_buffer_copy(bytes([TYPE_CODES[t.dtype] for t in tensors] or [0]))
        if like is not None:
            self.numel, self.partials = like.numel, like.partials
        else:
            self.numel = (C.c_longlong * max(1, self.n))(*[n for n in self.sizes if n])
            self.partials = int(_lib().bonsai_mt_partials(self.n))


def _norm_room(grads: TensorTable, device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
    return torch.empty((), dtype=torch.float32, device=device), torch.empty(grads.partials, dtype=torch.float64, device=device)


def mt_norm(grads: TensorTable, device: torch.device) -> torch.Tensor:
    """The 2-norm over all values of a table's tensors: a 0-dim f32 tensor."""
    if grads.n == 0:
        return torch.zeros((), dtype=torch.float32, device=device)
    with _on(device):
        norm, partial = _norm_room(grads, device)
        K.check(_lib().bonsai_mt_norm(grads.n, grads.ptrs, grads.numel, grads.types, partial.data_ptr(), norm.data_ptr(), _stream(device)), "mt_norm")
    return norm


def mt_clip(grads: TensorTable, out: TensorTable, max_norm: float, device: torch.device) -> torch.Tensor:
    """``out`` = ``grads`` scaled to a global norm of at most ``max_norm``; returns the norm before.  ``out`` may be ``grads``."""
    if grads.n == 0:
        return torch.zeros((), dtype=torch.float32, device=device)
    with _on(device):
        norm, partial = _norm_room(grads, device)
        K.check(_lib().bonsai_mt_clip(grads.n, grads.ptrs, out.ptrs, grads.numel, grads.types, out.types, max_norm, partial.data_ptr(),
                                      norm.data_ptr(), _stream(device)), "mt_clip")
    return norm


def mt_adam(params: TensorTable, grads: TensorTable, m: TensorTable, v: TensorTable, step: torch.Tensor, lr: float | torch.Tensor,
            betas: tuple[float, float], eps: float, weight_decay: float, decoupled: bool, max_norm: float | None = None) -> torch.Tensor | None:
    """One Adam step; ``step`` (int64 on the device) is raised by one.  With ``max_norm`` the gradients enter scaled to that global norm,
    and the norm before comes back."""
    device = step.device
    with _on(device):
        norm = partial = None
        if max_norm is not None:
            norm, partial = _norm_room(grads, device)
        lr_dev = lr if isinstance(lr, torch.Tensor) else None
        K.check(_lib().bonsai_mt_adam(params.n, params.ptrs, grads.ptrs, m.ptrs, v.ptrs, params.numel, params.types, grads.types,
                                      0.0 if lr_dev is not None else lr, K.ptr(lr_dev), betas[0], betas[1], eps, weight_decay, int(decoupled),
                                      step.data_ptr(), 0.0 if max_norm is None else max_norm, K.ptr(partial), K.ptr(norm), _stream(device)), "mt_adam")
    return norm


# ---- cross entropy of a linear head ------------------------------------------------------------------------------------------------
REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


def _ld(t: torch.Tensor) -> int:
    """Row stride; that of a single row may be anything."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _ce_bytes(weight: torch.Tensor, n: int, label_smoothing: float, what: int) -> int:
    size = int(_lib().bonsai_ce_bytes(weight.data_ptr(), _ld(weight), n, *weight.shape, TYPE_CODES[weight.dtype], label_smoothing, what))
    K.check(min(0, size), "linear_ce_bytes")
    return size


def linear_ce_forward(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int, reduction: str,
                      label_smoothing: float) -> tuple[torch.Tensor, torch.Tensor]:
    """hidden [n, d], weight [v, d] (one type, unit stride along d), targets int64 [n] -> the loss (f32, 0-dim or [n]) and what the
    backward pass takes: the live rows side by side, their list and their log-sum-exp."""
    (n, d), v, device = hidden.shape, weight.shape[0], hidden.device
    with _on(device):
        loss = torch.empty(n if reduction == "none" else (), dtype=torch.float32, device=device)
        kept = torch.empty(_ce_bytes(weight, n, label_smoothing, 0), dtype=torch.uint8, device=device)
        ws = torch.empty(_ce_bytes(weight, n, label_smoothing, 1), dtype=torch.uint8, device=device)
        K.check(_lib().bonsai_ce_forward(hidden.data_ptr(), _ld(hidden), weight.data_ptr(), _ld(weight), targets.data_ptr(), n, v, d,
                                         TYPE_CODES[hidden.dtype], ignore_index, REDUCTIONS[reduction], label_smoothing, kept.data_ptr(), kept.numel(),
                                         loss.data_ptr(), ws.data_ptr(), ws.numel(), _stream(device)), "linear_ce_forward")
    return loss, kept


def linear_ce_backward(weight: torch.Tensor, kept: torch.Tensor, n: int, up: torch.Tensor, reduction: str, label_smoothing: float, want_hidden: bool,
                       want_weight: bool) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """Gradients of :func:`linear_ce_forward` over n rows; ``up`` is the loss's gradient (f32, contiguous)."""
    (v, d), device = weight.shape, weight.device
    with _on(device):
        dh = torch.empty((n, d), dtype=weight.dtype, device=device) if want_hidden else None
        dw = torch.empty((v, d), dtype=weight.dtype, device=device) if want_weight else None
        ws = torch.empty(_ce_bytes(weight, n, label_smoothing, 3 if want_hidden else 2), dtype=torch.uint8, device=device)
        K.check(_lib().bonsai_ce_backward(weight.data_ptr(), _ld(weight), n, v, d, TYPE_CODES[weight.dtype], REDUCTIONS[reduction], label_smoothing,
                                          kept.data_ptr(), kept.numel(), up.data_ptr(), K.ptr(dh), K.ptr(dw), ws.data_ptr(), ws.numel(),
                                          _stream(device)), "linear_ce_backward")
    return dh, dw


# ---- dropout ---------------------------------------------------------------------------------------------------------------------------
Seed = int | torch.Tensor          # a tensor (int64, on the device) is read when the kernel runs


def _seed(seed: Seed) -> tuple[int, int | None]:
    return (0, seed.data_ptr()) if isinstance(seed, torch.Tensor) else (seed, None)


def dropout(x: torch.Tensor, steps: int, seed: Seed) -> torch.Tensor:
    """Rows x [n, d] (unit stride along d): each value stays, over steps / 65536, where its 16 random bits are below ``steps`` (< 65536)."""
    device = x.device
    with _on(device):
        y = x.new_empty(x.shape)
        K.check(_lib().bonsai_dropout(x.data_ptr(), _ld(x), y.data_ptr(), *x.shape, TYPE_CODES[x.dtype], *_seed(seed), steps, _stream(device)), "dropout")
    return y


_LR_SELF_ROWS = 256          # rows that the kernels group by themselves; a test compares it with the library's


# ---- low-rank updates --------------------------------------------------------------------------------------------------------------------
def _scale(scale: float | torch.Tensor) -> tuple[int | None, float]:
    return (scale.data_ptr(), 0.0) if isinstance(scale, torch.Tensor) else (None, scale)


def _lr_room(n: int, d: int, out: int, rank: int, adapters: int, grouped: bool, values: bool, back: bool, like: torch.Tensor) -> torch.Tensor | None:
    size = int(_lib().bonsai_lr_bytes(n, d, out, rank, adapters, TYPE_CODES[like.dtype], grouped, values, back))
    K.check(min(0, size), "low_rank_bytes")
    return like.new_empty(size, dtype=torch.uint8) if size else None


def low_rank_forward(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, base: torch.Tensor | None, ids: torch.Tensor | None, scale: float | torch.Tensor,
                     steps: int, seed: Seed, out: torch.Tensor | None = None, train: bool = False,
                     values: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """x [n, d], a [e, r, d], b [e, out, r] (dense, or of one adapter without e), base [n, out] or None (unit strides along rows), ids [n] or None -> the result [n, out] and what a
    backward pass takes (``train``; ``values``: that of ``b`` too)."""
    (n, d), (cols, r), e, device = x.shape, b.shape[-2:], 1 if b.dim() == 2 else b.shape[0], x.device
    with _on(device):
        y = x.new_empty((n, cols)) if out is None else out
        grouped = ids is not None
        kept = None if not train and n <= _LR_SELF_ROWS else _lr_room(n, d, cols, r, e, grouped, values, False, x)
        K.check(_lib().bonsai_lr_forward(x.data_ptr(), _ld(x), a.data_ptr(), b.data_ptr(), K.ptr(base), 0 if base is None else _ld(base), y.data_ptr(), _ld(y),
                                         *_scale(scale), n, d, cols, r, e, TYPE_CODES[x.dtype], K.ptr(ids), grouped and ids.dtype == torch.int64,
                                         K.ptr(kept), 0 if kept is None else kept.numel(), values, *_seed(seed), steps, _stream(device)), "low_rank_forward")
    return y, kept


def low_rank_backward(x: torch.Tensor | None, dy: torch.Tensor, a: torch.Tensor | None, b: torch.Tensor, d: int, kept: torch.Tensor | None, grouped: bool,
                      scale: float | torch.Tensor, steps: int, seed: Seed, want_x: bool, want_a: bool, want_b: bool) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Gradients of :func:`low_rank_forward` by x (needs ``a``), a (needs ``x``) and b (needs a pass with ``values``, and only that)."""
    (n, cols), r, e, one, device, dtype = dy.shape, b.shape[-1], 1 if b.dim() == 2 else b.shape[0], b.dim() == 2, dy.device, dy.dtype
    with _on(device):
        dx = dy.new_empty((n, d)) if want_x else None
        da = dy.new_empty((r, d) if one else (e, r, d)) if want_a else None
        db = dy.new_empty(b.shape) if want_b else None
        ws = _lr_room(n, d, cols, r, e, grouped, want_b, True, dy) if want_x or want_a else None
        K.check(_lib().bonsai_lr_backward(K.ptr(x), 0 if x is None else _ld(x), dy.data_ptr(), _ld(dy), K.ptr(a), b.data_ptr(), K.ptr(dx), K.ptr(da), K.ptr(db),
                                          *_scale(scale), n, d, cols, r, e, TYPE_CODES[dtype], grouped, K.ptr(kept), 0 if kept is None else kept.numel(), want_b,
                                          K.ptr(ws), 0 if ws is None else ws.numel(), *_seed(seed), steps, _stream(device)), "low_rank_backward")
    return dx, da, db


# ---- losses over log-probabilities ---------------------------------------------------------------------------------------------------------
POLICY_REDUCTIONS = {"tokens": 0, "sequences": 1, "sum": 2, "none": 3}
PREFERENCE_KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}


def _tune_room(rows: int, length: int, slopes: int, like: torch.Tensor) -> torch.Tensor:
    size = int(_lib().bonsai_tune_bytes(rows, length, slopes))
    K.check(min(0, size), "tune_bytes")
    return like.new_empty(size, dtype=torch.uint8)


def _rows(t: torch.Tensor | None) -> tuple[int | None, int]:
    return (None, 0) if t is None else (t.data_ptr(), _ld(t))


def policy_forward(logps, old, ref, mask, gain, clip: tuple[float, float], kl_weight: float, reduction: str, keep: bool) -> tuple:
    """Rows [n, t] (unit stride along t), gain f32 [n] or [n, t] -> (loss, [mean divergence, clipped share], what :func:`tune_scale` takes)."""
    n, t = logps.shape
    device = logps.device
    with _on(device):
        loss = logps.new_empty((n, t) if reduction == "none" else (), dtype=torch.float32)
        stats, kept = logps.new_empty(2, dtype=torch.float32), _tune_room(n, t, 2 * keep, logps)
        K.check(_lib().bonsai_policy_loss(*_rows(logps), *_rows(old), *_rows(ref), *_rows(mask), gain.data_ptr(), _ld(gain) if gain.dim() == 2 else gain.stride(0),
                                          gain.dim() == 2, n, t, TYPE_CODES[logps.dtype], *clip, kl_weight, POLICY_REDUCTIONS[reduction], loss.data_ptr(),
                                          stats.data_ptr(), kept.data_ptr(), kept.numel(), keep, _stream(device)), "policy_loss")
    return loss, stats, kept


def preference_forward(logps, ref, mask, beta: float, kind: str, smoothing: float, average: bool, reduction: str, keep: bool) -> tuple:
    """Rows [2 pairs, t] -> (loss, rewards [2 pairs], what :func:`tune_scale` takes)."""
    n, t = logps.shape
    device = logps.device
    with _on(device):
        loss = logps.new_empty(n // 2 if reduction == "none" else (), dtype=torch.float32)
        rewards, kept = logps.new_empty(n, dtype=torch.float32), _tune_room(n, t, keep, logps)
        K.check(_lib().bonsai_preference_loss(*_rows(logps), *_rows(ref), *_rows(mask), n // 2, t, TYPE_CODES[logps.dtype], PREFERENCE_KINDS[kind], average,
                                              REDUCTIONS[reduction], beta, smoothing, loss.data_ptr(), rewards.data_ptr(), kept.data_ptr(), kept.numel(), keep,
                                              _stream(device)), "preference_loss")
    return loss, rewards, kept


def tune_scale(kept: torch.Tensor, tokens: bool, up: torch.Tensor, mask: torch.Tensor | None, shape: tuple[int, int], dtype: torch.dtype) -> torch.Tensor:
    """Gradient [n, t] from what a loss kept (``tokens``: a slope for each) and the loss's own gradient (0-dim, [n, t], or one for every row modulo its
    length)."""
    n, t = shape
    device = kept.device
    with _on(device):
        out = kept.new_empty((n, t), dtype=dtype)
        kind = 0 if up.dim() == 0 else 2 if up.dim() == 2 else 1
        K.check(_lib().bonsai_tune_scale(kept.data_ptr(), kept.numel(), 1 + tokens, up.data_ptr(), kind, up.numel() if kind == 1 else 1, *_rows(mask), n, t,
                                         TYPE_CODES[dtype], out.data_ptr(), _stream(device)), "tune_scale")
    return out
