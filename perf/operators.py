"""The operators of a fine-tuning step, as a training program calls them: the loss of a language-model head that keeps no logits
(``training.linear_cross_entropy``, alone and with its gradients), the global gradient norm with clipping over many tensors
(``training.GradientSet``) and the Adam step that takes the clipped gradients (``training.FusedAdamW``).

Sizes are those of the 1.7B, 4B and 8B decoders of ``bench.py`` (hidden 2048 / 2560 / 4096, vocabulary 151 936) and generic ones.
Hidden rows lean towards the head's row of their target by a different amount for each token, so that the loss runs from tokens that
the model is sure of to ones that it did not expect.  Tensors of the norm and of Adam are views of one flat buffer, as a program
lays out its gradients for an all-reduce; the flat buffers come back.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
IGNORE = -100
BETA1, BETA2, EPS, DECAY, LR = 0.9, 0.95, 1e-8, 0.1, 3e-4
MODELS = {
    "1.7b": dict(hidden=2048, inter=6144, heads=16, kv_heads=8),
    "4b": dict(hidden=2560, inter=9728, heads=32, kv_heads=8),
    "8b": dict(hidden=4096, inter=12288, heads=32, kv_heads=8),
}


def _loss(name, rows, vocab, hidden, dtype, grads="", reduction="mean", masked=0.0, smoothing=0.0):
    """``grads``: which of the hidden rows ("h") and the head ("w") get a gradient; "" is the loss alone."""
    c = dict(do="loss", rows=rows, vocab=vocab, hidden=hidden, dtype=dtype, grads=grads, reduction=reduction, masked=masked, smoothing=smoothing)
    return dict(c, name=name) if name else c


def _tensors(name, do, of, dtype, model="", layers=0, rank=0, count=0, largest=0, align=64, max_norm=1.0, norm=4.0):
    """``of``: "adapters" (LoRA pairs of every layer), "layers" (all matrices and norms) or "mixed" (``count`` tensors of 1 to ``largest``
    values).  Gradients have about the global norm ``norm``; views start at multiples of ``align`` values."""
    c = dict(do=do, of=of, dtype=dtype, model=model, layers=layers, rank=rank, count=count, largest=largest, align=align, max_norm=max_norm, norm=norm)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the log-probability of one proposed token (speculative checks, beam scores): latency, and the head read once
        _loss("score 1 token 8B f16", 1, 151936, 4096, "f16", reduction="none"),
        # perplexity of a window of text
        _loss("score 1024 tokens 4B bf16", 1024, 151936, 2560, "bf16"),
        # a whole fine-tuning batch, the head trained too: the largest
        _loss("train 8192 tokens 8B bf16", 8192, 151936, 4096, "bf16", grads="hw"),
        # adapters on a frozen head, prompts masked out
        _loss("adapters 4096 tokens 8B masked", 4096, 151936, 4096, "bf16", grads="h", masked=0.6),
        # distilling into the small model in f16 with smoothed labels
        _loss("train 2048 tokens 1.7B f16", 2048, 151936, 2048, "f16", grads="hw", smoothing=0.1),
        # one short ragged batch, a weight for every token, a vocabulary and a width that no tile divides
        _loss("train 777 tokens ragged", 777, 32003, 1001, "bf16", grads="hw", reduction="none", masked=0.1),
        # 32-bit training of a small model
        _loss("train 512 tokens f32", 512, 32000, 1024, "f32", grads="hw"),
        # clipping the adapters of every layer of the 8B model
        _tensors("clip adapters 8B f32", "clip", "adapters", "f32", model="8b", layers=36, rank=8),
        # clipping full gradients of the small model, views at odd places, into 32-bit gradients
        _tensors("clip layers 1.7B bf16", "clip", "layers", "bf16", model="1.7b", layers=14, align=1),
        # a small adapter set: launches and latency
        _tensors("adam adapters 1.7B f32", "adam", "adapters", "f32", model="1.7b", layers=28, rank=4),
        # the 8B adapters
        _tensors("adam adapters 8B f32", "adam", "adapters", "f32", model="8b", layers=36, rank=16),
        # full fine-tuning of bf16 parameters with 32-bit moments
        _tensors("adam layers 1.7B bf16", "adam", "layers", "bf16", model="1.7b", layers=14),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "f16", "f32"])
    do = rng.choice(["loss", "loss", "clip", "adam"])
    if do == "loss":
        hidden, vocab, rows = _spread(rng, 64, 4096), _spread(rng, 1000, 151936), _spread(rng, 1, 8192)
        if rng.random() < 0.6:
            hidden = max(64, hidden // 64 * 64)
        grads = rng.choice(["", "h", "hw", "hw"])
        return _loss("", rows, vocab, hidden, dtype, grads, rng.choice(["mean", "sum", "none"]), rng.choice([0.0, 0.25, 0.6]), rng.choice([0.0, 0.0, 0.1]))
    of, align, norm = rng.choice(["adapters", "layers", "mixed"]), rng.choice([64, 64, 1]), rng.choice([0.25, 4.0, 30.0])
    if of == "adapters":
        return _tensors("", do, of, dtype, model=rng.choice(sorted(MODELS)), layers=rng.randint(1, 36), rank=_spread(rng, 1, 64), align=align, norm=norm)
    if of == "layers":
        return _tensors("", do, of, dtype, model=rng.choice(sorted(MODELS)), layers=rng.randint(1, 3), align=align, norm=norm)
    return _tensors("", do, of, dtype, count=_spread(rng, 1, 600), largest=_spread(rng, 10, 1000000), align=align, norm=norm)


# ---- the loss -----------------------------------------------------------------------------------------------------------------------
def _loss_inputs(case, seed):
    n, v, d = case["rows"], case["vocab"], case["hidden"]
    g = torch.Generator(device=DEV).manual_seed(seed)
    weight = (torch.randn(v, d, device=DEV, generator=g) * (1.28 / math.sqrt(d))).to(TYPES[case["dtype"]])
    targets = torch.randint(0, v, (n,), device=DEV, generator=g)
    lean = torch.rand(n, 1, device=DEV, generator=g) * 10.0
    hidden = torch.randn(n, d, device=DEV, generator=g)
    hidden = (hidden + lean * weight[targets].float() / 1.28).to(TYPES[case["dtype"]])
    turn = min(512, n)          # conversations of 512 tokens that begin with a masked prompt
    if n > 1:
        targets = torch.where(torch.arange(n, device=DEV) % turn < int(case["masked"] * turn), IGNORE, targets)
    each = case["reduction"] == "none"
    scale = 4096.0 if case["dtype"] == "f16" and case["reduction"] != "sum" else 1.0          # f16 gradients need a loss scale
    up = torch.rand(n, device=DEV, generator=g) * (0.5 * scale / n) if each else torch.full((), 0.25 * scale, device=DEV)
    return hidden, weight, targets, up


def _loss_plain(s):
    h, w, t, c = s["hidden"].detach().float(), s["weight"].detach().float(), s["targets"], s["case"]
    keep = t != IGNORE
    at = torch.where(keep, t, 0)[:, None]
    z = h @ w.T
    top = z.max(1, keepdim=True).values
    lse = top + (z - top).exp().sum(1, keepdim=True).log()
    a = c["smoothing"]
    nll = (lse - (1 - a) * z.gather(1, at)).squeeze(1)
    if a:
        nll = nll - a * z.mean(1)
    nll = torch.where(keep, nll, 0.0)
    loss = nll if c["reduction"] == "none" else nll.sum() if c["reduction"] == "sum" else nll.sum() / keep.sum()
    if not c["grads"]:
        return [loss]
    each = s["up"] / keep.sum() if c["reduction"] == "mean" else s["up"]
    each = torch.where(keep, each, 0.0)[:, None]
    dz = (z - lse).exp_()
    if a:
        dz -= a / c["vocab"]
    dz.scatter_add_(1, at, torch.full_like(at, -(1 - a), dtype=torch.float32))
    dz *= each
    grads = [dz @ w] if "h" in c["grads"] else []
    if "w" in c["grads"]:
        grads.append(dz.T @ h)
    return [loss] + [g.to(s["hidden"].dtype) for g in grads]


def _loss_own(s):
    from oxibonsai_b200 import training

    c = s["case"]
    loss = training.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], ignore_index=IGNORE, reduction=c["reduction"], label_smoothing=c["smoothing"])
    if not c["grads"]:
        return [loss]
    wanted = [s["hidden"]] if c["grads"] == "h" else [s["hidden"], s["weight"]]
    return [loss.detach()] + list(torch.autograd.grad(loss, wanted, s["up"]))


def _loss_exact(case, seed):
    hidden, weight, targets, up = _loss_inputs(case, seed)
    w, a, v, n = weight.double(), case["smoothing"], case["vocab"], case["rows"]
    live = (targets != IGNORE).nonzero().flatten()
    loss = torch.zeros(n, dtype=torch.float64, device=DEV)
    dh = torch.zeros(n, case["hidden"], dtype=torch.float64, device=DEV)
    dw = torch.zeros_like(w) if "w" in case["grads"] else None
    for rows in live.split(1024):
        x, t = hidden[rows].double(), targets[rows]
        logp = torch.log_softmax(x @ w.T, 1)
        q = torch.full_like(logp, a / v)
        q[torch.arange(len(rows), device=DEV), t] += 1 - a
        loss[rows] = -(q * logp).sum(1)
        if case["grads"]:
            scale = up[rows].double()[:, None] if up.dim() else up.double() / (len(live) if case["reduction"] == "mean" else 1)
            q = (logp.exp() - q) * scale
            dh[rows] = q @ w
            if dw is not None:
                dw += q.T @ x
    total = loss if case["reduction"] == "none" else loss.sum() / (len(live) if case["reduction"] == "mean" else 1)
    return [total] + ([dh] if "h" in case["grads"] else []) + ([dw] if dw is not None else [])


# ---- many tensors -------------------------------------------------------------------------------------------------------------------
def _shapes(case):
    if case["of"] == "mixed":
        rng = random.Random(case["count"] * 1000003 + case["largest"])
        return [(_spread(rng, 1, case["largest"]),) for _ in range(case["count"])]
    m = MODELS[case["model"]]
    h, i, q, kv = m["hidden"], m["inter"], m["heads"] * 128, m["kv_heads"] * 128
    if case["of"] == "adapters":
        r = case["rank"]
        one = [(r, h), (q, r), (r, h), (kv, r), (r, h), (i, r), (r, i), (h, r)]
    else:
        one = [(h,), (q, h), (kv, h), (kv, h), (128,), (128,), (h, q), (h,), (i, h), (i, h), (h, i)]
    return one * case["layers"]


def _places(case):
    shapes, at, places = _shapes(case), 0, []
    for s in shapes:
        places.append((at, math.prod(s), s))
        at = -(-(at + math.prod(s)) // case["align"]) * case["align"]
    return places, at


def _views(flat, places):
    return [flat[at:at + n].view(s) for at, n, s in places]


def _gradients(case, seed, places, total):
    """Flat gradients, zero between the views; some tensors get larger ones than others."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    flat = torch.randn(total, device=DEV, generator=g)
    live = torch.zeros(total, device=DEV)
    sizes = torch.rand(len(places), generator=torch.Generator().manual_seed(seed)).mul(2).exp().tolist()
    for (at, n, _), size in zip(places, sizes):
        live[at:at + n] = size
    flat *= live
    flat *= case["norm"] / flat.double().square().sum().sqrt()
    return flat.to(TYPES[case["dtype"]]), live > 0


def _adam_inputs(case, seed):
    places, total = _places(case)
    grads, live = _gradients(case, seed, places, total)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    draws = lambda size: torch.randn(total, device=DEV, generator=g) * size * live  # noqa: E731
    per = case["norm"] / math.sqrt(max(1, total))
    params, m, v = draws(0.02).to(TYPES[case["dtype"]]), draws(0.3 * per), draws(per).square_()
    return places, grads, params, m, v


def _clipped(flat, max_norm):
    norm = flat.double().square().sum().sqrt().float()
    return norm, torch.where(norm > max_norm, max_norm / (norm + 1e-6), 1.0)


def _clip_plain(s):
    norm, share = _clipped(s["grads"], s["case"]["max_norm"])
    torch.mul(s["grads"].float(), share, out=s["out"])
    return [norm, s["out"]]


def _clip_own(s):
    return [s["set"].clip(s["case"]["max_norm"]), s["out"]]


def _adam_plain(s):
    norm, share = _clipped(s["grads"], s["case"]["max_norm"])
    s["step"] += 1
    g = s["grads"].float() * share
    s["m"].mul_(BETA1).add_(g * (1 - BETA1))
    s["v"].mul_(BETA2).add_(g * g * (1 - BETA2))
    mean, root = s["m"] / (1 - BETA1 ** s["step"]), (s["v"] / (1 - BETA2 ** s["step"])).sqrt()
    p = s["params"].float()
    p = p * (1 - LR * DECAY) - LR * mean / (root + EPS)
    s["params"].copy_(p)
    return [norm, s["params"], s["m"], s["v"]]


def _adam_own(s):
    return [s["adam"].step(max_norm=s["case"]["max_norm"]), s["params"], s["m"], s["v"]]


def _tensors_exact(case, seed):
    places, total = _places(case)
    if case["do"] == "clip":
        grads = _gradients(case, seed, places, total)[0].double()
    else:
        grads, params, m, v = (x.double() for x in _adam_inputs(case, seed)[1:])
    norm = grads.norm()
    if norm > case["max_norm"]:
        grads = grads * (case["max_norm"] / (norm + 1e-6))
    if case["do"] == "clip":
        return [norm, grads]
    m, v = torch.lerp(grads, m, BETA1), torch.lerp(grads ** 2, v, BETA2)
    params = params - LR * (DECAY * params + (m / (1 - BETA1)) / ((v / (1 - BETA2)) ** 0.5 + EPS))
    return [norm, params, m, v]


# ---- the module's interface -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    if case["do"] == "loss":
        hidden, weight, targets, up = _loss_inputs(case, seed)
        hidden.requires_grad_("h" in case["grads"])
        weight.requires_grad_("w" in case["grads"])
        return dict(case=case, hidden=hidden, weight=weight, targets=targets, up=up)
    if case["do"] == "clip":
        places, total = _places(case)
        grads, _ = _gradients(case, seed, places, total)
        out = torch.zeros(total, device=DEV)
        s = dict(case=case, grads=grads, out=out)
        if own:
            from oxibonsai_b200 import training

            s["set"] = training.GradientSet(_views(grads, places), out=_views(out, places))
        return s
    places, grads, params, m, v = _adam_inputs(case, seed)
    s = dict(case=case, grads=grads, params=params, m=m, v=v, step=0)
    if own:
        from oxibonsai_b200 import training

        s["adam"] = training.FusedAdamW(_views(params, places), lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                        grads=_views(grads, places), state=(_views(m, places), _views(v, places)))
    return s


def run(state):
    do = state["case"]["do"]
    if do == "loss":
        return _loss_own(state) if own else _loss_plain(state)
    if do == "clip":
        return _clip_own(state) if own else _clip_plain(state)
    return _adam_own(state) if own else _adam_plain(state)


def work(case):
    if case["do"] == "loss":
        n, v, d, size = case["rows"], case["vocab"], case["hidden"], BYTES[case["dtype"]]
        turn = min(512, n)
        live = sum(1 for i in range(n) if n == 1 or i % turn >= int(case["masked"] * turn))
        moved = live * d * size + v * d * size + 8 * n + 4 * (n if case["reduction"] == "none" else 1)
        moved += n * d * size * ("h" in case["grads"]) + v * d * size * ("w" in case["grads"])
        return {"bytes": moved, "flops": 2.0 * live * v * d * (1 + len(case["grads"]))}
    count, size = sum(math.prod(s) for s in _shapes(case)), BYTES[case["dtype"]]
    if case["do"] == "clip":
        return {"bytes": count * (size + 4) + 4, "flops": 3.0 * count}
    return {"bytes": count * (size + 2 * size + 16) + 4, "flops": 16.0 * count}


def exact(case, seed):
    return _loss_exact(case, seed) if case["do"] == "loss" else _tensors_exact(case, seed)
