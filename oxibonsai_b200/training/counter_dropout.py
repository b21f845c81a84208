"""Dropout whose mask is a function of a seed and of each value's place, made again in the backward pass instead of stored.

``torch.nn.functional.dropout`` keeps one byte for every value between the passes.  Here 16 random bits of a value come from Philox4x32-10
(J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): eight neighbouring values of a row share
the counter (column // 8, 0, row, row >> 32) under the seed as key.  CUDA tensors run csrc/cuda/dropout.cu, CPU tensors the same bits in
torch, so that a mask does not depend on where it is made.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from ..ops import train_ops

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_LOW = 0xFFFFFFFF


def keep_steps(p: float) -> int:
    """Of the 65536 values of 16 bits, how many keep: the probability in steps of 2^-16."""
    return round((1.0 - p) * 65536)


def check_seed(seed, device: torch.device, what: str) -> train_ops.Seed:
    """``None`` draws one from torch's CPU generator; a tensor is read when the kernel runs."""
    if seed is None:
        return int(torch.randint(0, 2 ** 63 - 1, (), dtype=torch.int64, device="cpu"))
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"{what}: a seed tensor holds one int64 on {device}, got {seed.dtype} of shape {tuple(seed.shape)} on {seed.device}")
        return seed
    if isinstance(seed, bool) or not isinstance(seed, int) or not 0 <= seed < 2 ** 64:
        raise ValueError(f"{what}: a seed is an integer from 0 to 2^64 - 1 or an int64 tensor, got {seed!r}")
    return seed


def check_p(p: float, what: str) -> float:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: the probability is between 0 and 1, got {p}")
    return float(p)


def kept(rows: int, d: int, steps: int, seed: train_ops.Seed) -> torch.Tensor:
    """The mask [rows, d] on the CPU: what stays."""
    seed = int(seed) & (2 ** 64 - 1)
    groups = -(-d // 8)
    c0 = torch.arange(groups, dtype=torch.int64, device="cpu").expand(rows, groups)
    c1, r = torch.zeros_like(c0), torch.arange(rows, dtype=torch.int64, device="cpu")[:, None].expand(rows, groups)
    c2, c3 = r & _LOW, r >> 32
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(10):
        x, y = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # the low 64 bits, which is all of an unsigned product
        c0, c1, c2, c3 = (y >> 32 & _LOW) ^ c1 ^ k0, y & _LOW, (x >> 32 & _LOW) ^ c3 ^ k1, x & _LOW
        k0, k1 = k0 + 0x9E3779B9 & _LOW, k1 + 0xBB67AE85 & _LOW
    words = torch.stack([c0, c1, c2, c3], 2)
    return torch.stack([words & 0xFFFF, words >> 16], 3).reshape(rows, groups * 8)[:, :d] < steps


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """x as rows of its last dimension, with unit stride along them and no negative place."""
    flat = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return flat if flat.is_contiguous() or flat.stride(1) == 1 or flat.shape[1] == 1 and flat.stride(0) >= 1 else flat.contiguous()


def has_tangent(*tensors) -> bool:
    """Whether forward-mode differentiation goes through one of these (None is none): a kernel sees their values alone."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _cuda(x, steps, seed):
    y = train_ops.dropout(rows_of(x), steps, seed)
    return y if x.dim() == 2 else y.view(x.shape)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, steps, seed):
        ctx.steps, ctx.seed = steps, None if isinstance(seed, torch.Tensor) else seed
        if ctx.seed is None:
            ctx.save_for_backward(seed)
        if x.is_cuda:
            return _cuda(x, steps, seed)
        kind = torch.float64 if x.dtype == torch.float64 else torch.float32
        share = 65536.0 / steps if steps else 0.0
        mask = kept(x.numel() // x.shape[-1], x.shape[-1], steps, seed).view(x.shape)
        return torch.where(mask, x.to(kind) * share, 0.0).to(x.dtype)

    @staticmethod
    def backward(ctx, up):
        seed = ctx.saved_tensors[0] if ctx.seed is None else ctx.seed
        if up.is_cuda and not torch.is_grad_enabled() and not has_tangent(up):
            return _cuda(up, ctx.steps, seed), None, None
        return _Dropout.apply(up, ctx.steps, seed), None, None


def dropout(x: torch.Tensor, p: float = 0.5, seed: int | torch.Tensor | None = None, training: bool = True) -> torch.Tensor:
    """``x`` [..., d] with each value set to 0 with probability ``p`` and the others scaled by ``1 / (1 - p)``.  ``p`` is taken in steps of
    2^-16, and so is the scale that goes with it; where it is 0 then, ``x`` itself comes back.  A value that is dropped is 0 whatever it holds, and so is its gradient.

    ``seed``: an integer, or an int64 tensor on the device of ``x``, which is read when the kernel runs: a captured graph takes a new mask
    in each replay if the program changes the tensor in between (not between a pass and its backward pass, where autograd reports the change).
    Without a seed one is drawn from torch's CPU generator; a graph captured that way drops the same values every time.  A segment
    under :func:`checkpoint`, which is run again, draws the same one again.  The same seed, shape and ``p`` give the same mask on any device, and in :func:`low_rank_update`.  Nothing is kept between the passes but the seed.  Types are
    float32, float16 and bfloat16 (float64 on the CPU); the result is dense, rounded once.  Forward-mode derivatives are refused."""
    check_p(p, "dropout")
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("dropout: a tensor of at least one dimension is wanted")
    if x.device.type not in ("cuda", "cpu"):
        raise ValueError(f"dropout: CUDA or CPU tensors are wanted, got {x.device}")
    if x.dtype not in _TYPES + (() if x.is_cuda else (torch.float64,)):
        raise TypeError(f"dropout: float32, float16 or bfloat16 values are wanted, got {x.dtype}")
    if x.shape[-1] >= 2 ** 31:
        raise ValueError(f"dropout: rows of less than 2^31 values are wanted, got {x.shape[-1]}")
    seed = check_seed(seed, x.device, "dropout") if seed is not None or (training and p > 0.0) else 0
    steps = keep_steps(p)
    if not training or steps == 65536 or x.numel() == 0:
        return x
    if x.is_cuda and not (x.requires_grad and torch.is_grad_enabled()) and not has_tangent(x):
        return _cuda(x, steps, seed)
    return _Dropout.apply(x, steps, seed)
