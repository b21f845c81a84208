"""What adapters need beside the operators of ``operators.py``: the low-rank update of many adapters at once, for serving and with its
gradients (``training.low_rank_update``), dropout whose mask is made again instead of stored (``training.dropout``, and within the
update), and the losses that adapters are tuned with from log-probabilities (``training.preference_loss``, ``training.policy_loss``).

Projections are those of the 1.7B, 4B and 8B decoders of ``bench.py`` (hidden 2048 / 2560 / 4096, feed-forward 6144 / 9728 / 12288)
and generic ones.  Adapters are drawn as a program has them after some steps of training: neither factor is zero.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _update(name, rows, d, out, rank, dtype, adapters=0, spread="runs", bare=0.0, train=False, p=0.0):
    """``adapters``: 0 is one adapter for every row.  ``spread``: rows of one adapter lie side by side ("runs") or anywhere ("mixed");
    a share ``bare`` of the rows (or runs) has no adapter."""
    c = dict(do="update", rows=rows, d=d, out=out, rank=rank, dtype=dtype, adapters=adapters, spread=spread, bare=bare, train=train, p=p)
    return dict(c, name=name) if name else c


def _dropout(name, rows, d, dtype, p):
    c = dict(do="dropout", rows=rows, d=d, dtype=dtype, p=p)
    return dict(c, name=name) if name else c


def _preference(name, pairs, length, dtype, kind="sigmoid", beta=0.1, smoothing=0.0, average=False):
    c = dict(do="preference", pairs=pairs, length=length, dtype=dtype, kind=kind, beta=beta, smoothing=smoothing, average=average)
    return dict(c, name=name) if name else c


def _policy(name, rows, length, dtype, per_token=False, kl=0.0, reduction="tokens"):
    c = dict(do="policy", rows=rows, length=length, dtype=dtype, per_token=per_token, kl=kl, reduction=reduction)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one request that decodes with its adapter beside the 8B query projection: latency
        _update("serve 1 token 8B q", 1, 4096, 4096, 16, "bf16", adapters=8),
        # a decode batch of requests over 48 adapters beside the 8B feed-forward projection, some requests without one
        _update("serve 64 requests 8B up", 64, 4096, 12288, 16, "f16", adapters=48, spread="mixed", bare=0.1),
        # prompts of several requests in one ragged chunk, 4B feed-forward
        _update("serve 2999 prompt rows 4B up", 2999, 2560, 9728, 8, "bf16", adapters=6, bare=0.15),
        # one fine-tuning step of the 8B feed-forward adapter with dropout: the largest
        _update("train 8192 rows 8B up", 8192, 4096, 12288, 16, "bf16", train=True, p=0.05),
        # 32-bit adapters of the small model, as LoraAdapter makes them
        _update("train 2048 rows 1.7B q f32", 2048, 2048, 2048, 8, "f32", train=True),
        # several adapters trained side by side on a short batch, sizes and a rank that no tile divides
        _update("train 777 rows ragged f16", 777, 1001, 515, 5, "f16", adapters=3, spread="mixed", train=True, p=0.1),
        # dropout of a batch of 8B hidden rows, there and back
        _dropout("dropout 8192 x 4096 bf16", 8192, 4096, "bf16", 0.1),
        # of a short 32-bit batch of odd width
        _dropout("dropout 333 x 2049 f32", 333, 2049, "f32", 0.25),
        # a small batch of preference pairs
        _preference("preference 8 pairs x 511", 8, 511, "f32"),
        # a large one of long answers, scored by the mean of their tokens against a margin
        _preference("preference 256 pairs x 4096", 256, 4096, "f32", kind="ipo", average=True),
        # one group of short answers to a prompt
        _policy("policy 16 x 300", 16, 300, "f32", kl=0.05),
        # a rollout batch of long answers, an advantage for each token
        _policy("policy 1024 x 8192", 1024, 8192, "f32", per_token=True, kl=0.02, reduction="sequences"),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "f16", "f32"])
    do = rng.choice(["update", "update", "update", "dropout", "preference", "policy"])
    if do == "update":
        d, out = _spread(rng, 16, 12288), _spread(rng, 16, 12288)
        if rng.random() < 0.6:
            d, out = max(16, d // 64 * 64), max(16, out // 64 * 64)
        rank = _spread(rng, 1, 64)
        rows = _spread(rng, 1, max(1, min(8192, (1 << 27) // BYTES[dtype] // (d + out), (1 << 31) // rank // (d + out))))
        train = rng.random() < 0.5
        adapters = rng.choice([0, 1, _spread(rng, 2, 64)])
        return _update("", rows, d, out, rank, dtype, adapters, rng.choice(["runs", "mixed"]), rng.choice([0.0, 0.2]) if adapters else 0.0,
                       train, rng.choice([0.0, 0.1, 0.5]) if train else 0.0)
    if do == "dropout":
        return _dropout("", _spread(rng, 1, 8192), _spread(rng, 1, 4096 * 2 // BYTES[dtype]), dtype, rng.choice([0.05, 0.1, 0.5, 0.9]))
    if do == "preference":
        kind = rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"])
        return _preference("", _spread(rng, 1, 256), _spread(rng, 1, 8192), rng.choice([dtype, "f32"]), kind, rng.choice([0.05, 0.1, 0.5]),
                           rng.choice([0.0, 0.1]) if kind == "sigmoid" else 0.0, rng.random() < 0.3)
    return _policy("", _spread(rng, 1, 1024), _spread(rng, 1, 8192), rng.choice([dtype, "f32"]), rng.random() < 0.5, rng.choice([0.0, 0.05]),
                   rng.choice(["tokens", "sequences", "sum", "none"]))


# ---- random numbers: Philox4x32-10 of the counter (group of 8 columns, 0, row, 0), 16 bits for each value -----------------------------
# (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011)
M0, M1, W0, W1, LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _steps(p):
    """Of the 65536 values of 16 bits, how many keep."""
    return round((1.0 - p) * 65536)


def _keep_plain(rows, d, p, seed):
    groups = -(-d // 8)
    c0 = torch.arange(groups, device=DEV).expand(rows, groups)
    c1 = c3 = torch.zeros_like(c0)
    c2 = torch.arange(rows, device=DEV)[:, None].expand(rows, groups)
    k0, k1 = seed & LOW, seed >> 32 & LOW
    for _ in range(10):
        x, y = c0 * M0, c2 * M1
        c0, c1, c2, c3 = (y >> 32 & LOW) ^ c1 ^ k0, y & LOW, (x >> 32 & LOW) ^ c3 ^ k1, x & LOW
        k0, k1 = k0 + W0 & LOW, k1 + W1 & LOW
    words = torch.stack([c0, c1, c2, c3], 2)
    halves = torch.stack([words & 0xFFFF, words >> 16], 3)
    return halves.reshape(rows, groups * 8)[:, :d] < _steps(p)


def _keep_exact(rows, d, p, seed):
    """The same bits, one state [4, rows, groups] in 32-bit halves that never pass 2^63."""
    groups = (d + 7) // 8
    s = torch.zeros(4, rows, groups, dtype=torch.int64, device=DEV)
    s[0] += torch.arange(groups, device=DEV)
    s[2] += torch.arange(rows, device=DEV)[:, None]

    def times(a, m):
        low, high = a * (m & 0xFFFF), a * (m >> 16)
        low = low + ((high & 0xFFFF) << 16)
        return (high >> 16) + (low >> 32), low & LOW

    for i in range(10):
        key = (seed + i * W0) & LOW, ((seed >> 32) + i * W1) & LOW
        (h0, l0), (h1, l1) = times(s[0], M0), times(s[2], M1)
        s = torch.stack([h1 ^ s[1] ^ key[0], l1, h0 ^ s[3] ^ key[1], l0])
    bits = torch.empty(rows, groups, 8, dtype=torch.int64, device=DEV)
    for j in range(8):
        bits[:, :, j] = s[j // 2] >> (16 * (j % 2)) & 0xFFFF
    return bits.flatten(1)[:, :d] < _steps(p)


# ---- the low-rank update ---------------------------------------------------------------------------------------------------------------
def _update_inputs(case, seed):
    n, d, out, r, kind = case["rows"], case["d"], case["out"], case["rank"], TYPES[case["dtype"]]
    count = max(1, case["adapters"])
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    x, base, dy = rand(n, d), rand(n, out), rand(n, out) * (1024.0 if case["dtype"] == "f16" else 1.0) / n
    a, b = rand(count, r, d) / math.sqrt(d), rand(count, out, r) * (0.3 / math.sqrt(r))
    scales = torch.rand(count, device=DEV, generator=g) * 2 + 0.5
    ids = None
    if case["adapters"]:
        of = torch.randint(0, count, (n,), device=DEV, generator=g)
        bare = torch.rand(n, device=DEV, generator=g) < case["bare"]
        of = torch.where(bare, -1, of)
        if case["spread"] == "runs":                 # prompts of different lengths, one behind another
            starts = torch.rand(n, device=DEV, generator=g) < 8.0 / n
            of = of[torch.cumsum(starts, 0).clamp(max=n - 1)]
        ids = of.to(torch.int32)
    x, base, dy, a, b = (t.to(kind) for t in (x, base, dy, a, b))
    return x, base, dy, a, b, scales, ids


def _update_plain(s):
    c = s["case"]
    x, base, a, b = (s[k].detach().float() for k in ("x", "base", "a", "b"))
    (n, d), (e, r), out = x.shape, a.shape[:2], b.shape[1]
    if c["p"]:
        keep, share = _keep_plain(n, d, c["p"], s["seed"]), 65536.0 / _steps(c["p"])
        x = torch.where(keep, x * share, 0.0)
    ids = torch.zeros(n, dtype=torch.int32, device=DEV) if s["ids"] is None else s["ids"]
    of = torch.where(ids[:, None] == torch.arange(e, device=DEV), s["scales"], 0.0)[:, :, None].expand(n, e, r).reshape(n, e * r)
    a_all, b_all = a.reshape(e * r, d), b.permute(1, 0, 2).reshape(out, e * r)
    h = (x @ a_all.T) * of
    y = (base + h @ b_all.T).to(s["base"].dtype)
    if not c["train"]:
        return [y]
    dy = s["dy"].float()
    dh = (dy @ b_all) * of
    dx = dh @ a_all
    if c["p"]:
        dx = torch.where(keep, dx * share, 0.0)
    da, db = (dh.T @ x).reshape(e, r, d), (dy.T @ h).reshape(out, e, r).permute(1, 0, 2)
    return [y] + [t.to(y.dtype) for t in (dx, da, db)]


def _update_own(s):
    from oxibonsai_b200 import training

    c = s["case"]
    y = training.low_rank_update(s["x"], s["a"], s["b"], base=s["base"], ids=s["ids"], scale=s["scales"], dropout=c["p"], seed=s["seed"])
    if not c["train"]:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, [s["x"], s["a"], s["b"]], s["dy"]))


def _update_exact(case, seed):
    x, base, dy, a, b, scales, ids = (t if t is None else t.double() for t in _update_inputs(case, seed))
    n, d = x.shape
    y, dx, da, db = base.clone(), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    factor = torch.ones((), dtype=torch.float64, device=DEV)
    if case["p"]:
        factor = _keep_exact(n, d, case["p"], _key(seed)) / (_steps(case["p"]) / 65536.0)
        x = x * factor
    for e in range(a.shape[0]):
        rows = torch.arange(n, device=DEV) if ids is None else (ids == e).nonzero().flatten()
        f = factor[rows] if factor.dim() else factor
        w = scales[e] * b[e] @ a[e]
        y[rows] += x[rows] @ w.T
        if case["train"]:
            dx[rows] = (dy[rows] @ w) * f
            dw = scales[e] * dy[rows].T @ x[rows]
            da[e], db[e] = b[e].T @ dw, dw @ a[e].T
    return [y, dx, da, db] if case["train"] else [y]


def _key(seed):
    return seed * 0x9E3779B97F4A7C15 + 12345 & (1 << 63) - 1


# ---- dropout -----------------------------------------------------------------------------------------------------------------------------
def _dropout_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(case["rows"], case["d"], device=DEV, generator=g).to(TYPES[case["dtype"]]) for _ in range(2)]


def _dropout_plain(s):
    x, c = s["x"].detach(), s["case"]
    keep, share = _keep_plain(*x.shape, c["p"], s["seed"]), 65536.0 / _steps(c["p"])
    return [torch.where(keep, t.float() * share, 0.0).to(t.dtype) for t in (x, s["dy"])]


def _dropout_own(s):
    from oxibonsai_b200 import training

    y = training.dropout(s["x"], s["case"]["p"], seed=s["seed"])
    return [y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]]


def _dropout_exact(case, seed):
    factor = _keep_exact(case["rows"], case["d"], case["p"], _key(seed)).double() * 65536.0 / _steps(case["p"])
    return [t.double() * factor for t in _dropout_inputs(case, seed)]


# ---- preference pairs ----------------------------------------------------------------------------------------------------------------------
def _answers(rows, length, g):
    """Which places of padded sequences are an answer: behind a prompt, up to an end."""
    at = torch.arange(length, device=DEV)
    begin = (torch.rand(rows, 1, device=DEV, generator=g) * 0.3 * length).long()
    size = 1 + (torch.rand(rows, 1, device=DEV, generator=g) * 0.7 * (length - 1)).long()
    return (at >= begin) & (at < begin + size)


def _token_logps(rows, length, g):
    return torch.log(torch.rand(rows, length, device=DEV, generator=g) * 0.98 + 0.01) * 0.8


def _preference_inputs(case, seed):
    pairs, length, kind = case["pairs"], case["length"], TYPES[case["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed)
    mask = _answers(2 * pairs, length, g)
    ref = _token_logps(2 * pairs, length, g)
    # answers that the model has moved towards or away from, each by its own amount
    moved = torch.randn(2 * pairs, 1, device=DEV, generator=g) * (3.0 / math.sqrt(length))
    logps = ref + (moved + torch.randn(2 * pairs, length, device=DEV, generator=g)) * 0.2
    return logps.to(kind), ref.to(kind), mask


def _preference_plain(s):
    c = s["case"]
    mask, beta = s["mask"], c["beta"]
    d = torch.where(mask, s["logps"].detach().float() - s["ref"].float(), 0.0).sum(1, dtype=torch.float64)
    count = mask.sum(1)
    if c["average"]:
        d = d / count.clamp(min=1)
    chosen, rejected = d.chunk(2)
    z = chosen - rejected
    m = beta * z
    soft = lambda v: v.clamp(min=0.0) + (1.0 + (-v.abs()).exp()).log()  # noqa: E731
    e = c["smoothing"]
    if c["kind"] == "sigmoid":
        each, up = (1 - e) * soft(-m) + e * soft(m), beta * (1.0 / (1.0 + (-m).exp()) - (1 - e))
    elif c["kind"] == "hinge":
        each, up = (1.0 - m).clamp(min=0.0), torch.where(m < 1.0, -beta, 0.0)
    else:
        each, up = (z - 0.5 / beta) ** 2, 2.0 * (z - 0.5 / beta)
    up = torch.cat([up, -up]) / c["pairs"]
    if c["average"]:
        up = up / count.clamp(min=1)
    grad = torch.where(mask, up[:, None], 0.0).to(s["logps"].dtype)
    return [t.float() for t in (each.mean(), beta * chosen, beta * rejected)] + [grad]


def _preference_own(s):
    from oxibonsai_b200 import training

    c = s["case"]
    r = training.preference_loss(s["logps"], s["ref"], s["mask"], beta=c["beta"], kind=c["kind"], label_smoothing=c["smoothing"], average=c["average"])
    return [r.loss.detach(), r.chosen_rewards, r.rejected_rewards, torch.autograd.grad(r.loss, s["logps"])[0]]


def _preference_exact(case, seed):
    logps, ref, mask = _preference_inputs(case, seed)
    logps = logps.double().requires_grad_()
    beta, e = case["beta"], case["smoothing"]
    weight = mask.double()
    if case["average"]:
        weight = weight / weight.sum(1, keepdim=True)
    score = ((logps - ref.double()) * weight).sum(1).view(2, -1)
    m = beta * (score[0] - score[1])
    if case["kind"] == "sigmoid":
        each = -(1 - e) * torch.nn.functional.logsigmoid(m) - e * torch.nn.functional.logsigmoid(-m)
    elif case["kind"] == "hinge":
        each = torch.relu(1 - m)
    else:
        each = (m / beta - 1 / (2 * beta)).square()
    loss = each.sum() / case["pairs"]
    return [loss.detach(), *(beta * score.detach()), torch.autograd.grad(loss, logps)[0]]


# ---- clipped policy ratio ----------------------------------------------------------------------------------------------------------------
CLIP = (0.2, 0.28)


def _policy_inputs(case, seed):
    n, length, kind = case["rows"], case["length"], TYPES[case["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed)
    mask = _answers(n, length, g)
    old = _token_logps(n, length, g)
    logps = old + torch.randn(n, length, device=DEV, generator=g) * 0.2
    ref = old + torch.randn(n, length, device=DEV, generator=g) * 0.3
    gain = torch.randn(n, length if case["per_token"] else 1, device=DEV, generator=g)
    up = torch.rand(n, length, device=DEV, generator=g) / n if case["reduction"] == "none" else torch.ones((), device=DEV)
    return logps.to(kind), old.to(kind), ref.to(kind), gain if case["per_token"] else gain[:, 0], mask, up


def _policy_plain(s):
    c, mask, up = s["case"], s["mask"], s["up"]
    logps, old, ref = (s[k].detach().float() for k in ("logps", "old", "ref"))
    gain = s["gain"] if c["per_token"] else s["gain"][:, None]
    step = logps.double() - old.double()                  # next to a border every bit counts
    clipped = ((gain > 0) & (step > math.log1p(CLIP[1])) | (gain < 0) & (step < math.log1p(-CLIP[0]))) & mask
    ratio, back = step.float().exp(), ref - logps
    grown = torch.expm1(back)
    kl = torch.where(mask, grown - back, 0.0)
    surrogate = torch.minimum(ratio * gain, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * gain)
    each = torch.where(mask, c["kl"] * kl - surrogate, 0.0)
    grad = torch.where(clipped, 0.0, -ratio * gain) - c["kl"] * grown
    count, live = mask.sum(), mask.sum(1, keepdim=True)
    if c["reduction"] == "sequences":
        w = 1.0 / (live.clamp(min=1) * (live > 0).sum())
    else:
        w = 1.0 / count if c["reduction"] == "tokens" else torch.ones((), device=DEV)
    loss = each if c["reduction"] == "none" else (each * w).sum()
    grad = torch.where(mask, grad * (w * up), 0.0).to(s["logps"].dtype)
    return [loss, kl.sum() / count, clipped.sum() / count, grad]


def _policy_own(s):
    from oxibonsai_b200 import training

    c = s["case"]
    r = training.policy_loss(s["logps"], s["old"], s["gain"], mask=s["mask"], ref_logps=s["ref"], clip=CLIP, kl_weight=c["kl"], reduction=c["reduction"])
    return [r.loss.detach(), r.kl, r.clipped, torch.autograd.grad(r.loss, s["logps"], s["up"])[0]]


def _policy_exact(case, seed):
    logps, old, ref, gain, mask, up = _policy_inputs(case, seed)
    logps, old, ref = logps.double().requires_grad_(), old.double(), ref.double()
    gain = gain.double().view(case["rows"], -1).expand_as(old)
    live = mask.nonzero(as_tuple=True)
    lp, a = logps[live], gain[live]
    ratio = torch.exp(lp - old[live])
    inside = torch.clip(ratio, 1 - CLIP[0], 1 + CLIP[1])
    gap = ref[live] - lp
    kl = torch.expm1(gap) - gap
    each = torch.max(-a * ratio, -a * inside) + case["kl"] * kl
    per = torch.zeros_like(old).index_put(live, each)
    size = mask.sum(1)
    loss = {"none": lambda: per, "sum": lambda: per.sum(), "tokens": lambda: each.mean(),
            "sequences": lambda: (per.sum(1)[size > 0] / size[size > 0]).mean()}[case["reduction"]]()
    share = (-a * inside > -a * ratio).double().mean()
    return [loss.detach(), kl.detach().mean(), share, torch.autograd.grad(loss, logps, up.double())[0]]


# ---- the module's interface -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    s = dict(case=case, seed=_key(seed))
    if case["do"] == "update":
        s["x"], s["base"], s["dy"], s["a"], s["b"], s["scales"], s["ids"] = _update_inputs(case, seed)
        for k in "xab":
            s[k].requires_grad_(case["train"])
    elif case["do"] == "dropout":
        s["x"], s["dy"] = _dropout_inputs(case, seed)
        s["x"].requires_grad_()
    elif case["do"] == "preference":
        s["logps"], s["ref"], s["mask"] = _preference_inputs(case, seed)
        s["logps"].requires_grad_()
    else:
        s["logps"], s["old"], s["ref"], s["gain"], s["mask"], s["up"] = _policy_inputs(case, seed)
        s["logps"].requires_grad_()
    return s


_RUNS = {"update": (_update_plain, _update_own), "dropout": (_dropout_plain, _dropout_own), "preference": (_preference_plain, _preference_own),
         "policy": (_policy_plain, _policy_own)}
_EXACT = {"update": _update_exact, "dropout": _dropout_exact, "preference": _preference_exact, "policy": _policy_exact}


def run(state):
    return _RUNS[state["case"]["do"]][own](state)


def work(case):
    size = BYTES[case["dtype"]]
    if case["do"] == "update":
        n, d, out, r = case["rows"], case["d"], case["out"], case["rank"]
        weights = max(1, min(n, case["adapters"])) * r * (d + out) * size
        moved, flops = n * (d + 2 * out) * size + weights + 4 * n * (case["adapters"] > 0), 2.0 * n * r * (d + out)
        if case["train"]:          # the gradient of the output comes in, those of the rows and of both factors go out
            moved, flops = moved + n * (d + out) * size + weights, 3 * flops
        return {"bytes": moved, "flops": flops}
    if case["do"] == "dropout":
        n = case["rows"] * case["d"]
        return {"bytes": 4 * n * size, "flops": 2.0 * n}
    if case["do"] == "preference":         # two log-probabilities and a mask; the gradient
        n = 2 * case["pairs"] * case["length"]
        return {"bytes": n * (3 * size + 1) + 8 * case["pairs"], "flops": 3.0 * n}
    n = case["rows"] * case["length"]      # three log-probabilities, gains and a mask; the gradient
    gains = n if case["per_token"] else case["rows"]
    return {"bytes": n * (4 * size + 1) + 4 * gains + 8 * n * (case["reduction"] == "none"), "flops": 30.0 * n}


def exact(case, seed):
    return _EXACT[case["do"]](case, seed)
