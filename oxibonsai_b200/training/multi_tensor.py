"""Global gradient norm, clipping and Adam steps over many tensors, without a launch or a host synchronisation per tensor.

``grad_norm`` / ``clip_grad_norm`` / ``Adam`` of this package work tensor by tensor (a clip of the 288 adapter matrices of a 36-layer
model waits for the GPU 288 times).  The forms here take the whole set at once, keep the norm on the device and can be captured
into a CUDA graph; on CPU tensors they compute the same with torch.

Reference: crates/oxibonsai-model/src/optimizer.rs (``clip_grad_norm``, Adam, AdamW).
"""
from __future__ import annotations

from typing import Iterable, Sequence

import torch
from torch.autograd.graph import increment_version

from ..ops import train_ops

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _dense(t: torch.Tensor) -> bool:
    """Whether the values fill one stretch of memory, in whatever order of the axes."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.shape == b.shape and (a.stride() == b.stride() or all(x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n != 1))


def _layout(tensors: Sequence[torch.Tensor]) -> tuple[list, list, list]:
    return [t.shape for t in tensors], [t.stride() for t in tensors], [t.dtype for t in tensors]


def _check(tensors: Sequence[torch.Tensor], what: str) -> torch.device:
    device = None
    for t in tensors:
        if not isinstance(t, torch.Tensor) or t.dtype not in _TYPES or t.layout != torch.strided:
            raise TypeError(f"{what}: dense float32, float16 or bfloat16 tensors are wanted, got "
                            f"{t.dtype if isinstance(t, torch.Tensor) else type(t).__name__}")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"{what}: tensors of one device are wanted, got {device} and {t.device}")
        if not _dense(t) and t.numel():
            raise ValueError(f"{what}: a tensor of shape {tuple(t.shape)} has gaps or repeats in memory (strides {t.stride()})")
    if device is not None and device.type not in ("cuda", "cpu"):
        raise ValueError(f"{what}: CUDA or CPU tensors are wanted, got {device}")
    return device or torch.device("cpu")


def _check_apart(tensors: Iterable[torch.Tensor], what: str, read: Iterable[torch.Tensor] = ()) -> None:
    """Tensors that are written must not share memory, with one another or with those that are only ``read``: two blocks would scale or
    step the same values, or one would read what another has written."""
    last = last_written = 0
    for begin, size, written in sorted([(t.data_ptr(), t.nbytes, True) for t in tensors] + [(t.data_ptr(), t.nbytes, False) for t in read]):
        if size and begin < (last if written else last_written):
            raise ValueError(f"{what}: two of the tensors share memory")
        last = max(last, begin + size)
        last_written = max(last_written, begin + size if written else 0)


def _counters(tensors: Sequence[torch.Tensor]) -> list[torch.Tensor]:
    """Tensors that have the version counters of all of these: views of one tensor share its counter."""
    tensors = [t for t in tensors if not t.is_inference()]          # those have none
    owners = [t if t._base is None else t._base for t in tensors]
    return list({id(o): t for o, t in zip(owners, tensors)}.values())


class GradientSet:
    """A fixed list of gradient tensors (any mix of float32, float16 and bfloat16, on one device) and the table of their places that
    the kernels take.  The set keeps its tensors alive; their values may change between calls, their memory may not.  ``out``: tensors
    that take the clipped gradients (the same shapes and order in memory, any of the types) in place of the gradients themselves.

    >>> grads = GradientSet([p.grad for p in params])
    >>> norm = grads.clip(1.0)          # a 0-dim tensor: nothing waits for the GPU
    """

    def __init__(self, tensors: Iterable[torch.Tensor], out: Iterable[torch.Tensor] | None = None):
        self.tensors = list(tensors)
        self.out = self.tensors if out is None else list(out)
        self.device = _check(self.tensors, "GradientSet")
        if out is not None:
            if len(self.out) != len(self.tensors) or not all(_same_order(a, b) for a, b in zip(self.tensors, self.out)):
                raise ValueError("GradientSet: out needs tensors of the gradients' shapes and strides")
            if self.out and _check(self.out, "GradientSet: out") != self.device:
                raise ValueError(f"GradientSet: out is on {self.out[0].device}, the gradients on {self.device}")
        # a tensor may be clipped onto itself and onto nothing else that the set holds
        _check_apart([g for g, o in zip(self.tensors, self.out) if g.data_ptr() != o.data_ptr() or g.dtype != o.dtype] + self.out, "GradientSet")
        self._written = _counters(self.out)
        self._table = self._out_table = None
        if self.device.type == "cuda":
            self._table = train_ops.TensorTable(self.tensors, keep=True)
            self._out_table = self._table if out is None else train_ops.TensorTable(self.out, keep=True)

    def __len__(self) -> int:
        return len(self.tensors)

    def norm(self) -> torch.Tensor:
        """sqrt(sum of all squares) as a 0-dim float32 tensor."""
        if self._table is not None:
            return train_ops.mt_norm(self._table, self.device)
        return _norm(self.tensors).float()

    def clip(self, max_norm: float) -> torch.Tensor:
        """Scales by ``max_norm / (norm + 1e-6)`` where the norm is above ``max_norm > 0`` (by 1 otherwise, as ``clip_grad_norm`` does)
        and returns the norm before.  A norm that is NaN scales nothing; an infinite one scales by 0."""
        if self._table is not None:
            norm = train_ops.mt_clip(self._table, self._out_table, float(max_norm), self.device)
        else:
            n = _norm(self.tensors)
            share, norm = _share(float(n), max_norm), n.float()
            with torch.no_grad():
                for g, o in zip(self.tensors, self.out):
                    if share != 1.0 or g is not o:
                        o.copy_(g.float() * share)
        increment_version(self._written)
        return norm


@torch.no_grad()
def _norm(tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    return sum((t.double().square().sum() for t in tensors), torch.zeros((), dtype=torch.float64)).sqrt()


def _share(norm: float, max_norm: float) -> float:
    return max_norm / (norm + 1e-6) if norm > max_norm > 0 else 1.0


def global_grad_norm(params: Iterable[torch.Tensor]) -> torch.Tensor:
    """``grad_norm`` as a 0-dim tensor on the gradients' device, in two launches.  Nothing is written: a parameter may be listed twice, and
    counts twice."""
    grads = [g for g in [p.grad for p in params] if g is not None]
    device = _check(grads, "global_grad_norm")
    return train_ops.mt_norm(train_ops.TensorTable(grads), device) if device.type == "cuda" else _norm(grads).float()


def clip_global_norm(params: Iterable[torch.Tensor], max_norm: float) -> torch.Tensor:
    """``clip_grad_norm`` as a 0-dim tensor on the gradients' device, in two launches.  Gradients that share memory are refused."""
    return GradientSet([g for g in [p.grad for p in params] if g is not None]).clip(max_norm)


class FusedAdam:
    """``Adam`` as one pass over all parameters, with clipping folded in: ``step(max_norm=1.0)`` scales the gradients while it reads them
    (``p.grad`` itself stays as it is) and returns their norm as a 0-dim tensor.

    Parameters are float32, float16 or bfloat16, the moments float32.  ``grads``: fixed gradient tensors, one for each parameter, whose
    table is made once (neither they nor the parameters may change their memory then); without them every step looks up ``p.grad``
    (parameters without one are skipped) and where the parameters are.  ``state``: lists of first and
    second moments to go on from, updated in place.  The step count is on the device: with ``grads`` a step can be captured into a
    CUDA graph, ``lr`` then as a 0-dim float32 CUDA tensor where it changes."""

    decoupled = False

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, grads: Sequence[torch.Tensor] | None = None,
                 state: tuple[Sequence[torch.Tensor], Sequence[torch.Tensor]] | None = None, steps: int = 0):
        self.params, self.lr, self.betas, self.eps, self.wd = list(params), lr, betas, eps, weight_decay
        name = type(self).__name__
        if not self.params:
            raise ValueError(f"{name}: no parameters")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"{name}: betas in [0, 1) are wanted, got {betas}")
        self.device = _check(self.params, name)
        if state is None:
            self.m = [torch.zeros_like(p, dtype=torch.float32, requires_grad=False) for p in self.params]
            self.v = [torch.zeros_like(p, dtype=torch.float32, requires_grad=False) for p in self.params]
        else:
            self.m, self.v = list(state[0]), list(state[1])
        for part in (self.m, self.v):
            if len(part) != len(self.params) or any(t.dtype != torch.float32 or t.device != self.device or not _same_order(t, p)
                                                    for t, p in zip(part, self.params)):
                raise ValueError(f"{name}: state needs a float32 tensor of each parameter's shape and strides, on its device")
        _check_apart(self.params + self.m + self.v, name)
        self.steps = torch.full((), steps, dtype=torch.int64, device=self.device)
        self.grads = None if grads is None else list(grads)
        self._tables = None
        self._place()
        if self.grads is not None:
            if len(self.grads) != len(self.params):
                raise ValueError(f"{name}: {len(self.grads)} gradients for {len(self.params)} parameters")
            self._check_grads(self.params, self.grads)
            if any(not _same_order(p, g) for p, g in zip(self.params, self.grads)):
                raise ValueError(f"{name}: fixed gradients need their parameters' shapes and strides")
            _check_apart(self.params + self.m + self.v, name, read=self.grads)
            if self.device.type == "cuda":
                self._tables = self._with(self.grads, keep=True)

    def _place(self) -> None:
        """Notes where the parameters and moments are."""
        self._written = _counters(self.params)
        self._at, self._layout = [p.data_ptr() for p in self.params], _layout(self.params)
        if self.device.type == "cuda":
            self._fixed = [train_ops.TensorTable(x, keep=True) for x in (self.params, self.m, self.v)]

    def _follow(self) -> None:
        """Parameters whose memory was replaced since (``p.data = ...``) are found at their new places.  ``p.data[:n]`` has the old address: the
        tables hold for the noted sizes, orders and types only."""
        if [p.data_ptr() for p in self.params] == self._at and _layout(self.params) == self._layout:
            return
        name = type(self).__name__
        if _check(self.params, name) != self.device or not all(_same_order(p, m) for p, m in zip(self.params, self.m)):
            raise ValueError(f"{name}: a parameter has moved to another device or changed its shape since the optimizer was made")
        _check_apart(self.params + self.m + self.v, name)
        self._place()

    def _lie_like_params(self, grads: Sequence[torch.Tensor | None]) -> bool:
        """Whether every parameter has a gradient that the kernel can walk as it is (list by list: some 0.1 us for each tensor and property)."""
        if type(None) in set(map(type, grads)) or set([g.get_device() for g in grads]) != {self.device.index} or not set([g.dtype for g in grads]) <= set(_TYPES):
            return False
        try:
            return [g.shape for g in grads] == self._layout[0] and [g.stride() for g in grads] == self._layout[1]
        except RuntimeError:          # a sparse tensor has no strides
            return False

    def _with(self, grads: Sequence[torch.Tensor], keep: bool = False) -> list[train_ops.TensorTable]:
        return [self._fixed[0], train_ops.TensorTable(grads, like=self._fixed[0], keep=keep), *self._fixed[1:]]

    def _check_grads(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor]) -> None:
        name = type(self).__name__
        for p, g in zip(params, grads):
            if not isinstance(g, torch.Tensor) or g.dtype not in _TYPES or g.layout != torch.strided:
                raise TypeError(f"{name}: dense float32, float16 or bfloat16 gradients are wanted, got {getattr(g, 'dtype', type(g).__name__)}")
            if g.shape != p.shape or g.device != self.device:
                raise ValueError(f"{name}: a gradient of shape {tuple(g.shape)} on {g.device} for a parameter of shape {tuple(p.shape)} on {p.device}")

    @property
    def t(self) -> int:
        """Steps done (waits for the GPU)."""
        return int(self.steps)

    def step(self, lr: float | torch.Tensor | None = None, max_norm: float | None = None) -> torch.Tensor | None:
        lr = self.lr if lr is None else lr
        if isinstance(lr, torch.Tensor) and (lr.numel() != 1 or lr.dtype != torch.float32 or lr.device != self.device):
            raise ValueError(f"{type(self).__name__}: lr as a tensor is one float32 on {self.device}")
        if self._tables is not None:
            tables = self._tables
        else:
            self._follow()
            grads = self.grads if self.grads is not None else [p.grad for p in self.params]
            params, m, v, every = self.params, self.m, self.v, True
            if self.device.type == "cuda" and self._lie_like_params(grads):
                return self._run(self._with(grads), lr, max_norm)
            if any(g is None for g in grads):
                live = [i for i, g in enumerate(grads) if g is not None]
                params, grads, m, v = ([part[i] for i in live] for part in (params, grads, m, v))
                every = False
            self._check_grads(params, grads)
            if self.device.type == "cpu":
                return self._step_cpu(params, grads, m, v, float(lr), max_norm)
            # the kernel walks memory: a gradient that autograd laid out in another order than its parameter is copied into it
            with torch.no_grad():
                grads = [g if _same_order(p, g) else torch.empty_like(p, dtype=g.dtype).copy_(g) for p, g in zip(params, grads)]
            if not every:
                return self._run([train_ops.TensorTable(x) for x in (params, grads, m, v)], lr, max_norm, _counters(params))
            tables = self._with(grads)
        return self._run(tables, lr, max_norm)

    def _run(self, tables: list[train_ops.TensorTable], lr: float | torch.Tensor, max_norm: float | None,
             written: list[torch.Tensor] | None = None) -> torch.Tensor | None:
        """``written``: tensors with the version counters of the parameters that are stepped, where those are not all."""
        if tables[0].n == 0:
            self.steps += 1
            return None if max_norm is None else torch.zeros((), dtype=torch.float32, device=self.device)
        norm = train_ops.mt_adam(*tables, self.steps, lr if isinstance(lr, torch.Tensor) else float(lr), self.betas, self.eps, self.wd, self.decoupled,
                                 None if max_norm is None else float(max_norm))
        increment_version(self._written if written is None else written)
        return norm

    @torch.no_grad()
    def _step_cpu(self, params, grads, m, v, lr: float, max_norm: float | None) -> torch.Tensor | None:
        self.steps += 1
        t, (b1, b2), norm, share = int(self.steps), self.betas, None, 1.0
        if max_norm is not None:
            n = _norm(grads)
            norm, share = n.float(), _share(float(n), max_norm)
        for p, g, mi, vi in zip(params, grads, m, v):
            x, g = p.float(), g.float() * share
            if self.wd and not self.decoupled:
                g = g + self.wd * x
            mi.mul_(b1).add_(g, alpha=1 - b1)
            vi.mul_(b2).addcmul_(g, g, value=1 - b2)
            if self.decoupled:
                x = x * (1 - lr * self.wd)
            p.copy_(x - (lr / (1 - b1 ** t)) * mi / (vi.sqrt() / (1 - b2 ** t) ** 0.5 + self.eps))
        return norm

    @torch.no_grad()
    def reset(self) -> None:
        for part in (*self.m, *self.v, self.steps):
            part.zero_()

    def zero_grad(self) -> None:
        """Drops ``p.grad``; with fixed gradients fills those with zeros."""
        if self.grads is not None:
            for g in self.grads:
                g.zero_()
        else:
            for p in self.params:
                p.grad = None


class FusedAdamW(FusedAdam):
    """:class:`FusedAdam` with decoupled weight decay."""

    decoupled = True

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, grads: Sequence[torch.Tensor] | None = None,
                 state: tuple[Sequence[torch.Tensor], Sequence[torch.Tensor]] | None = None, steps: int = 0):
        super().__init__(params, lr, betas, eps, weight_decay, grads, state, steps)
