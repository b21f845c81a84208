"""Torch-facing wrappers of the training kernels in ``libbonsai_cuda.so`` (csrc/cuda/multi_tensor.cu, linear_ce.cu).

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

_vp, _i, _d, _ll = C.c_void_p, C.c_int, C.c_double, C.c_longlong
_SIG = {
    "bonsai_mt_partials": [_i],
    "bonsai_mt_norm": [_i, _vp, _vp, _vp, _vp, _vp, _vp],
    "bonsai_mt_clip": [_i, _vp, _vp, _vp, _vp, _vp, _d, _vp, _vp, _vp],
    "bonsai_ce_bytes": [_vp, _ll, _i, _i, _i, _i, C.c_float, _i],
    "bonsai_ce_forward": [_vp, _ll, _vp, _ll, _vp, _i, _i, _i, _i, _ll, _i, C.c_float, _vp, _ll, _vp, _vp, _ll, _vp],
    "bonsai_ce_backward": [_vp, _ll, _i, _i, _i, _i, _i, C.c_float, _vp, _ll, _vp, _vp, _vp, _vp, _ll, _vp],
    "bonsai_mt_adam": [_i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _d, _vp, _d, _d, _d, _d, _i, _vp, _d, _vp, _vp, _vp],
}
_declared = False
_HERE = contextlib.nullcontext()
TYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _lib():
    global _declared
    l = K.lib()
    if not _declared:
        K.declare(_SIG, {"bonsai_mt_partials": _ll, "bonsai_ce_bytes": _ll})
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
