"""Low-rank updates of one or many adapters beside a shared projection, with their gradients.

``LoraAdapter`` applies one adapter to all rows in two matrix products, which write the rank values to memory and the update once more than it
is needed.  Here the rows of a batch name their adapters, and one kernel makes the whole update: for serving many requests whose
adapters differ beside one packed projection, and for training one or several adapters, with dropout on the way in.  CUDA tensors
run csrc/cuda/low_rank.cu, CPU tensors the same steps in torch.

Reference: crates/oxibonsai-model/src/lora.rs (``LoraAdapter::apply`` = ``(alpha / r) * B(A x)``, one adapter for all rows).
"""
from __future__ import annotations

import math

import torch
from torch.autograd.graph import increment_version

from ..ops import train_ops
from .counter_dropout import check_p, check_seed, has_tangent, keep_steps, kept, rows_of

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_CPU_TYPES = _TYPES + (torch.float64,)
MAX_RANK, MAX_ADAPTERS = 128, 4096


def _cpu_parts(x, a, ids, scale, steps, seed):
    """What both passes on the CPU need: the type of the sums, the mask and its scale, the adapters' scales and rows."""
    kind = torch.float64 if x.dtype == torch.float64 else torch.float32
    keep = kept(*x.shape, steps, seed) if steps < 65536 else None
    share = 1.0 if keep is None else 65536.0 / steps if steps else 0.0
    count = 1 if a.dim() == 2 else len(a)
    scales = scale.to(kind) if isinstance(scale, torch.Tensor) else torch.full((count,), scale, dtype=kind, device=x.device)
    rows = [torch.arange(len(x), device=x.device)] if ids is None else [(ids.reshape(-1) == e).nonzero().flatten() for e in range(count)]
    return kind, keep, share, scales.reshape(-1), rows


def _cpu_forward(x, a, b, base, ids, scale, steps, seed):
    kind, keep, share, scales, rows = _cpu_parts(x, a, ids, scale, steps, seed)
    xs = x.to(kind) if keep is None else torch.where(keep, x.to(kind) * share, 0.0)
    y = x.new_zeros(len(x), b.shape[-2], dtype=kind) if base is None else base.to(kind).clone()
    a, b = a.view(-1, *a.shape[-2:]), b.view(-1, *b.shape[-2:])
    for e, at in enumerate(rows):
        if len(at):
            y[at] += (xs[at] @ a[e].to(kind).T) @ b[e].to(kind).T * scales[e]
    return y.to(x.dtype)


def _cpu_backward(x, a, b, ids, scale, steps, seed, up):
    kind, keep, share, scales, rows = _cpu_parts(x, a, ids, scale, steps, seed)
    xs = x.to(kind) if keep is None else torch.where(keep, x.to(kind) * share, 0.0)
    shapes, a, b = (a.shape, b.shape), a.view(-1, *a.shape[-2:]), b.view(-1, *b.shape[-2:])
    dx, da, db = torch.zeros_like(xs), a.new_zeros(a.shape, dtype=kind), b.new_zeros(b.shape, dtype=kind)
    for e, at in enumerate(rows):
        if len(at):
            u, ae, be = up[at].to(kind) * scales[e], a[e].to(kind), b[e].to(kind)
            g = u @ be
            dx[at], da[e], db[e] = g @ ae, g.T @ xs[at], u.T @ (xs[at] @ ae.T)
    if keep is not None:
        dx = torch.where(keep, dx * share, 0.0)
    return dx.to(x.dtype), da.to(a.dtype).view(shapes[0]), db.to(b.dtype).view(shapes[1])


class _LowRankUpdate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, base, how):
        ids, scale, steps, seed = how
        held = [v for v in (scale, seed) if isinstance(v, torch.Tensor)]
        ctx.how = ids is not None, None if isinstance(scale, torch.Tensor) else scale, steps, None if isinstance(seed, torch.Tensor) else seed, a.dim()
        if not x.is_cuda:
            ctx.save_for_backward(x, a, b, ids, *held)
            return _cpu_forward(x, a, b, base, ids, scale, steps, seed)
        want_x, want_a, want_b = ctx.needs_input_grad[:3]
        y, kept = train_ops.low_rank_forward(x, a, b, base, ids, scale, steps, seed, train=True, values=want_b)
        # x is for the gradient of a, a for that of x
        ctx.save_for_backward(x if want_a else None, a if want_x else None, b, kept, *held)
        ctx.width = x.shape[1]
        return y

    @staticmethod
    def backward(ctx, up):
        if torch.is_grad_enabled() or (up.is_cuda and has_tangent(up)):
            raise RuntimeError("low_rank_update: its gradients cannot be differentiated again (create_graph=True, or a tangent of the gradient)")
        x, a, b, more, *held = ctx.saved_tensors
        grouped, scale, steps, seed, _ = ctx.how
        if scale is None:
            scale = held.pop(0)
        if seed is None:
            seed = held.pop(0)
        want_x, want_a, want_b, want_base = ctx.needs_input_grad[:4]
        dx = da = db = None
        if not up.is_cuda:
            dx, da, db = _cpu_backward(x, a, b, more, scale, steps, seed, up)
            dx, da, db = dx if want_x else None, da if want_a else None, db if want_b else None
        elif want_x or want_a or want_b:
            dx, da, db = train_ops.low_rank_backward(x, rows_of(up), a, b, ctx.width, more, grouped, scale, steps, seed, want_x, want_a, want_b)
        return dx, da, db, up if want_base else None, None


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First byte of a tensor's values and the one behind the last."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _check_out(out, shape, x, others, base, wants_grad) -> None:
    if wants_grad or has_tangent(out):
        raise ValueError("low_rank_update: out is for calls without gradients")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("low_rank_update: out has a gradient or a history of its own, which a result written into it would not change: detach it")
    if out.shape != shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"low_rank_update: out is {tuple(shape)} of {x.dtype} on {x.device}, got {tuple(out.shape)} of {out.dtype} on {out.device}")
    if out.numel() == 0:
        return
    rows = out.view(-1, shape[-1]) if out.is_contiguous() else out if out.dim() == 2 else None
    if rows is None or (rows.stride(1) != 1 and shape[-1] > 1) or (len(rows) > 1 and rows.stride(0) < shape[-1]):
        raise ValueError(f"low_rank_update: out is dense, or a matrix of rows that do not overlap, got strides {out.stride()}")
    same = base is not None and base.data_ptr() == out.data_ptr() and base.stride() == out.stride()
    begin, end = _span(out)
    for t in others + ([] if base is None or same else [base]):
        lo, hi = _span(t) if t.numel() else (0, 0)
        if lo < end and begin < hi:
            raise ValueError("low_rank_update: out shares memory with an input that it is not itself")


def low_rank_update(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, base: torch.Tensor | None = None, ids: torch.Tensor | None = None,
                    scale: float | torch.Tensor = 1.0, dropout: float = 0.0, seed: int | torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """``base + scale * b[e] (a[e] x)`` for every row of ``x``, where ``e`` is the row's adapter; differentiable in ``x``, ``a``, ``b`` and ``base``.

    ``x`` [..., in], ``base`` [..., out] (what the shared projection gave; None: 0).  One adapter: ``a`` [rank, in] and ``b`` [out, rank]; many:
    ``a`` [count, rank, in], ``b`` [count, out, rank] and ``ids`` [...] (int32 or int64) with each row's adapter, in any order.  A negative id
    is a row without one, whose result is ``base`` as it is.  An id of ``count`` or more raises IndexError on the CPU; on the GPU, where nothing waits,
    the results of that row and the gradient of its ``x`` are NaN, and no adapter's gradient has it.  ``scale``: a number, or float32 [count].  All
    tensors have one type (float32, float16 or bfloat16; float64 on the CPU); ranks go up to 128, adapters to 4096, all sizes stay below 2^30.  ``dropout``
    zeroes values of ``x`` on their way in, as :func:`dropout` of ``x`` (as rows) with the same ``seed`` does.

    Sums are float32 whatever the inputs, the rank values keep 22 bits (24 of bfloat16), results and gradients are rounded once.  How sums are split goes by the
    sizes of the call: a row's last bits may differ between batches of different sizes, within a batch they do not depend on its place or the other rows.  A
    row with an infinity has results that are not finite; other rows are as without it.  ``out`` takes the result of a call
    without gradients and has none itself; it may be ``base``.  Between the passes the rank values are kept (4 bytes each, 6 of bfloat16, the rank rounded up to 16, 32, 64 or 128), and
    ``x``, ``a`` and ``b`` as every product keeps them.  On the GPU nothing is read back and all memory comes from torch's allocator; a pass and its
    gradients can be captured into a CUDA graph as those of :func:`linear_cross_entropy` can.  Second derivatives and, on the GPU, forward-mode ones are refused."""
    what = "low_rank_update"
    xs, sa, sb, device, dtype = x.shape, a.shape, b.shape, x.device, x.dtype
    single = len(sa) == 2
    if len(xs) < 1 or len(sa) not in (2, 3) or len(sb) != len(sa) or xs[-1] != sa[-1] or sa[-2] != sb[-1] or sa[:-2] != sb[:-2]:
        raise ValueError(f"{what}: x [..., in], a [count, rank, in] and b [count, out, rank] (or one adapter without count) are wanted, got "
                         f"{tuple(xs)}, {tuple(sa)} and {tuple(sb)}")
    rows, d, rank, cols, count = xs[:-1], sa[-1], sa[-2], sb[-2], 1 if single else sa[0]
    n = math.prod(rows)
    if not 1 <= rank <= MAX_RANK or not 1 <= count <= MAX_ADAPTERS or d < 1 or cols < 1 or max(d, cols, n) >= 2 ** 30:
        raise ValueError(f"{what}: 1 to {MAX_ADAPTERS} adapters of rank 1 to {MAX_RANK}, widths of at least 1 and sizes below 2^30 are wanted, got {count} of rank {rank}, "
                         f"widths {d} and {cols}, {n} rows")
    if base is not None:
        if base.shape[:-1] != rows or base.shape[-1] != cols or base.dim() != len(xs):
            raise ValueError(f"{what}: base of shape {(*rows, cols)} is wanted, got {tuple(base.shape)}")
        if base.dtype != dtype:
            raise TypeError(f"{what}: base has the type of x, {dtype}, got {base.dtype}")
    if ids is None:
        if count != 1:
            raise ValueError(f"{what}: with {count} adapters ids of shape {tuple(rows)} are wanted")
    elif ids.shape != rows:
        raise ValueError(f"{what}: ids of shape {tuple(rows)} are wanted, got {tuple(ids.shape)}")
    elif ids.dtype != torch.int32 and ids.dtype != torch.int64:
        raise TypeError(f"{what}: ids are int32 or int64, got {ids.dtype}")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.numel() != count or scale.dim() > 1:
            raise ValueError(f"{what}: a scale for each adapter is float32 [{count}], got {scale.dtype} of shape {tuple(scale.shape)}")
        if (scale.requires_grad and torch.is_grad_enabled()) or has_tangent(scale):
            raise ValueError(f"{what}: the scale has no gradient")
        if scale.device != device:
            raise ValueError(f"{what}: tensors of one device are wanted, got a scale on {scale.device} and x on {device}")
        if scale.requires_grad or not scale.is_contiguous():
            scale = scale.detach().contiguous()
    else:
        scale = float(scale)
    if a.device != device or b.device != device or (base is not None and base.device != device) or (ids is not None and ids.device != device):
        raise ValueError(f"{what}: tensors of one device are wanted, got {', '.join(str(t.device) for t in (x, a, b, base, ids) if t is not None)}")
    if device.type not in ("cuda", "cpu"):
        raise ValueError(f"{what}: CUDA or CPU tensors are wanted, got {device}")
    if a.dtype != dtype or b.dtype != dtype or dtype not in (_TYPES if device.type == "cuda" else _CPU_TYPES):
        raise TypeError(f"{what}: x, a and b of one type (float32, float16, bfloat16) are wanted, got {dtype}, {a.dtype} and {b.dtype}")
    steps = 65536 if dropout == 0.0 else keep_steps(check_p(dropout, what))
    seed = 0 if seed is None and steps == 65536 else check_seed(seed, device, what)
    wants_grad = torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad or (base is not None and base.requires_grad))
    wants_grad = wants_grad or (x.is_cuda and has_tangent(x, a, b, base))                # which autograd refuses
    if out is not None:
        _check_out(out, (*rows, cols), x, [t for t in (x, a, b, ids, scale, seed) if isinstance(t, torch.Tensor)], base, wants_grad)
    if n == 0:
        y = (x @ a.T @ b.T) if single else x @ a[0].T @ b[0].T                     # zero gradients
        return out if out is not None else y if base is None else base + y
    flat, base2 = rows_of(x), None if base is None else rows_of(base)
    a, b = a.contiguous(), b.contiguous()
    if ids is not None:
        ids = ids.contiguous()
        if not x.is_cuda and bool((ids >= count).any()):
            raise IndexError(f"{what}: an id names none of {count} adapters")
    if wants_grad:
        y = _LowRankUpdate.apply(flat, a, b, base2, (ids, scale, steps, seed))
        return y if len(xs) == 2 else y.reshape((*rows, cols))
    if not x.is_cuda:
        y = _cpu_forward(flat, a, b, base2, ids, scale, steps, seed).reshape((*rows, cols))
        return y if out is None else out.copy_(y)
    y, _ = train_ops.low_rank_forward(flat, a, b, base2, ids, scale, steps, seed, out=None if out is None else out if out.dim() == 2 else out.view(-1, cols))
    if out is None:
        return y if len(xs) == 2 else y.reshape((*rows, cols))
    if not out.is_inference():
        increment_version(out)
    return out


class AdapterBank:
    """The adapters of one projection that requests may name: factors side by side, as :func:`low_rank_update` takes them.  Adapters of a lower rank
    than the bank's are filled up with zeros, which costs their bytes and changes no result.

    >>> bank = AdapterBank(4096, 4096, rank=16, count=64, dtype=torch.bfloat16, device="cuda")
    >>> bank.set(3, adapter)                        # a LoraAdapter
    >>> y = bank(x, base, ids)                      # ids: each row's adapter, -1 without one
    """

    def __init__(self, in_features: int, out_features: int, rank: int, count: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if not 1 <= rank <= MAX_RANK or not 1 <= count <= MAX_ADAPTERS or min(in_features, out_features) < 1:
            raise ValueError(f"AdapterBank: 1 to {MAX_ADAPTERS} adapters of rank 1 to {MAX_RANK} are wanted, got {count} of rank {rank}, {in_features} to {out_features}")
        self.a = torch.zeros(count, rank, in_features, dtype=dtype, device=device)
        self.b = torch.zeros(count, out_features, rank, dtype=dtype, device=device)
        self.scales = torch.zeros(count, dtype=torch.float32, device=device)

    @property
    def count(self) -> int:
        return len(self.a)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.a, self.b, self.scales))

    @torch.no_grad()
    def set(self, index: int, adapter) -> None:
        """Copies a ``LoraAdapter`` into place ``index``."""
        if not 0 <= index < self.count:
            raise IndexError(f"AdapterBank: place {index} of {self.count}")
        r, d = adapter.A.shape
        if r > self.a.shape[1] or d != self.a.shape[2] or adapter.B.shape != (self.b.shape[1], r):
            raise ValueError(f"AdapterBank: an adapter of rank up to {self.a.shape[1]} from {self.a.shape[2]} to {self.b.shape[1]} is wanted, got "
                             f"{tuple(adapter.A.shape)} and {tuple(adapter.B.shape)}")
        self.clear(index)
        self.a[index, :r] = adapter.A
        self.b[index, :, :r] = adapter.B
        self.scales[index] = adapter.config.scale

    @torch.no_grad()
    def clear(self, index: int) -> None:
        """Leaves place ``index`` without effect."""
        if not 0 <= index < self.count:
            raise IndexError(f"AdapterBank: place {index} of {self.count}")
        for t in (self.a, self.b, self.scales):
            t[index] = 0

    @torch.no_grad()
    def __call__(self, x: torch.Tensor, base: torch.Tensor | None, ids: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        return low_rank_update(x, self.a, self.b, base=base, ids=ids, scale=self.scales, out=out)
