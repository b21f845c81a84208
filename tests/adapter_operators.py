"""Plain 64-bit forms of the adapter operators (low-rank updates, dropout, preference and policy losses), and the bounds that kernels keep."""
import torch
from training_operators import HALF_STEP

S = 2.0 ** -23          # of a sum of magnitudes, for each addition of a float32 sum that may truncate
TINY = {torch.float32: 2.0 ** -120, torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -25, torch.float64: 0.0}


def philox(counter, key):
    """Philox4x32-10 of four counter words and two key words, in Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        x, y = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [y >> 32 ^ c[1] ^ k[0], y & 0xFFFFFFFF, x >> 32 ^ c[3] ^ k[1], x & 0xFFFFFFFF]
        k = [k[0] + 0x9E3779B9 & 0xFFFFFFFF, k[1] + 0xBB67AE85 & 0xFFFFFFFF]
    return c


def mask_by_formula(places, p, seed):
    """What dropout keeps at (row, column) places."""
    steps, got = round((1 - p) * 65536), []
    for row, col in places:
        word = philox([col // 8, 0, row & 0xFFFFFFFF, row >> 32], [seed & 0xFFFFFFFF, seed >> 32])[col % 8 // 2]
        got.append((word >> 16 * (col % 2) & 0xFFFF) < steps)
    return torch.tensor(got)


def update_inputs(n, d, out, rank, adapters, dtype, device, seed=0, bare=0.0, spread="mixed"):
    g = torch.Generator().manual_seed(seed)
    e = max(1, adapters)
    x, base, dy = torch.randn(n, d, generator=g), torch.randn(n, out, generator=g), torch.randn(n, out, generator=g)
    a, b = torch.randn(e, rank, d, generator=g) / d ** 0.5, torch.randn(e, out, rank, generator=g) / rank ** 0.5
    scales = torch.rand(e, generator=g) * 2 - 0.5
    ids = None
    if adapters:
        ids = torch.randint(0, adapters, (n,), generator=g)
        ids = torch.where(torch.rand(n, generator=g) < bare, -1, ids)
        if spread == "runs":
            ids = ids.sort().values
    return [t.to(device, dtype) for t in (x, base, dy, a, b)] + [scales.to(device), None if ids is None else ids.to(device)]


def update_by_formula(x, base, dy, a, b, scales, ids, keep=None, share=1.0):
    """(y, dx, da, db) and a bound for each, in float64.

    With u the half step of the type: rank values are off by (d + 20) S of sum |a x| (the products of 16-bit values are exact in float32, those of float32
    parts are off by 2^-21); they enter what follows to 2^-21, whose sums over rank (or rows) add their own S each; a result is rounded by u, its addition to base by
    2 S of the magnitudes."""
    kind = x.dtype
    u, tiny = HALF_STEP[kind], TINY[kind]
    x, dy, a, b, scales = x.double(), dy.double(), a.double(), b.double(), scales.double()
    base = torch.zeros(len(x), b.shape[1], dtype=torch.float64, device=x.device) if base is None else base.double()
    if keep is not None:
        x = torch.where(keep, x * share, 0.0)
    n, d, out, r = len(x), x.shape[1], b.shape[1], a.shape[1]
    y, dx, da, db = base.clone(), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    by, bx, ba, bb = (torch.zeros_like(t) for t in (y, dx, da, db))
    for e in range(len(a)):
        rows = torch.arange(n, device=x.device) if ids is None else (ids == e).nonzero().flatten()
        if not len(rows):
            continue
        xe, ue, s, k = x[rows], dy[rows], scales[e], len(rows)
        h, g, hm, gm = xe @ a[e].T, ue @ b[e], xe.abs() @ a[e].abs().T, ue.abs() @ b[e].abs()
        y[rows] += s * (h @ b[e].T)
        dx[rows], da[e], db[e] = s * (g @ a[e]), s * (g.T @ xe), s * (ue.T @ h)
        s = s.abs()
        by[rows] = (d + r + 60) * S * s * (hm @ b[e].abs().T)
        bx[rows] = (out + r + 60) * S * s * (gm @ a[e].abs())
        ba[e] = (out + k + 60) * S * s * (gm.T @ xe.abs())
        bb[e] = (d + k + 60) * S * s * (ue.abs().T @ hm)
    if keep is not None:
        dx, bx = torch.where(keep, dx * share, 0.0), torch.where(keep, bx * share, 0.0)
    return (y, dx, da, db), (by * (1 + u) + 2 * S * (base.abs() + y.abs()) + u * y.abs() + tiny, *(t * (1 + u) + 2 * S * v.abs() + u * v.abs() + tiny
                                                                                   for t, v in ((bx, dx), (ba, da), (bb, db))))


def preference_by_formula(logps, ref, mask, beta, kind, smoothing=0.0, average=False, reduction="mean", up=None):
    """(loss, chosen, rejected, gradient) and bounds: a difference of two log-probabilities is rounded once, everything behind it is float64 until the
    end; the loss bends by at most beta^2 / 4 (ipo: 2)."""
    u, tiny = HALF_STEP[logps.dtype], TINY[logps.dtype]
    d = logps.double() - (0.0 if ref is None else ref.double())
    live = torch.ones_like(d, dtype=torch.bool) if mask is None else mask
    d = torch.where(live, d, 0.0)
    w = (1.0 / live.sum(1).clamp(min=1) if average else torch.ones(len(d), dtype=torch.float64, device=d.device))
    s, off = d.sum(1) * w, 2.0 ** -23 * d.abs().sum(1) * w
    (c, r), p = s.chunk(2), len(d) // 2
    z, offz = c - r, off[:p] + off[p:]
    m = beta * z
    if kind == "sigmoid":
        minus, plus = -torch.nn.functional.logsigmoid(m), -torch.nn.functional.logsigmoid(-m)
        each, slope, bend = (1 - smoothing) * minus + smoothing * plus, beta * (smoothing * torch.sigmoid(m) - (1 - smoothing) * torch.sigmoid(-m)), beta * beta / 4
    elif kind == "hinge":
        assert float((m - 1).abs().min()) > beta * float(offz.max())
        each, slope, bend = (1 - m).clamp(min=0.0), torch.where(m < 1, -beta, 0.0).double(), 0.0
    else:
        each, slope, bend = (z - 0.5 / beta) ** 2, 2 * (z - 0.5 / beta), 2.0
    off_each = slope.abs() * offz + bend * offz ** 2
    loss, b_loss = (each, off_each) if reduction == "none" else (t.sum() / (p if reduction == "mean" else 1) for t in (each, off_each))
    up = torch.ones_like(loss) if up is None else up.double()
    by = (up / (p if reduction == "mean" else 1)).expand(p)
    grad = torch.cat([slope * by, -slope * by]) * w
    b_grad = torch.cat([bend * offz * by.abs()] * 2) * w
    grad, b_grad = (torch.where(live, t[:, None], 0.0) for t in (grad, b_grad))
    out = (loss, beta * c, beta * r, grad)
    return out, (b_loss + 2 * S * loss.abs(), *(beta * o + S * v.abs() for o, v in ((off[:p], out[1]), (off[p:], out[2]))),
                 b_grad * (1 + u) + (u + 4 * S) * grad.abs() + tiny)


def policy_by_formula(logps, old, gain, mask, ref, clip, weight, reduction="tokens", up=None):
    """(loss, kl, clipped, gradient) and bounds: step = l - old is exact in float64 and rounded once, exp and expm1 are within 2 steps of float32."""
    u, tiny = HALF_STEP[logps.dtype], TINY[logps.dtype]
    l = logps.double()
    live = torch.ones_like(l, dtype=torch.bool) if mask is None else mask
    zero = lambda t: torch.where(live, t, 0.0)  # noqa: E731
    step = zero(l - (l if old is None else old.double()))
    g = zero((gain.double() if gain.dim() == 2 else gain.double()[:, None]).expand_as(l))
    ratio = step.exp()
    each = -torch.minimum(ratio * g, ratio.clamp(1 - clip[0], 1 + clip[1]) * g)
    cut = ((g > 0) & (ratio > 1 + clip[1]) | (g < 0) & (ratio < 1 - clip[0])) & live
    slope = torch.where(cut, 0.0, -ratio * g)
    b_each, b_slope = ((4 + step.abs()) * S * t for t in (ratio * g.abs(), slope.abs()))
    kl = torch.zeros_like(l)
    if ref is not None:
        back = zero(ref.double() - l)
        grown = torch.expm1(back)
        kl, b_kl = grown - back, 4 * S * (grown.abs() * (1 + back.abs()) + back.abs())
        if weight:
            each, slope = each + weight * kl, slope - weight * grown
            b_each, b_slope = b_each + weight * b_kl, b_slope + weight * 4 * S * (grown.abs() + (1 + grown.abs()) * back.abs())
    else:
        b_kl = torch.zeros_like(l)
    each, slope, kl, b_each, b_slope, b_kl = (zero(t) for t in (each, slope, kl, b_each, b_slope, b_kl))
    b_each, b_slope = b_each + S * each.abs(), b_slope + S * slope.abs()
    n, size = live.sum(), live.sum(1, keepdim=True)
    w = 1.0 / n if reduction == "tokens" else 1.0 / (size.clamp(min=1) * (size > 0).sum()) if reduction == "sequences" else torch.ones((), device=l.device)
    loss = each if reduction == "none" else (each * w).sum() if int(n) or reduction == "sum" else each.sum() * float("nan")
    b_loss = b_each if reduction == "none" else torch.nan_to_num((b_each * w).sum())
    up = torch.ones_like(loss) if up is None else up.double()
    grad, b_grad = zero(slope * w * up), zero(b_slope * w * up.abs())
    mean, b_mean = kl.sum() / n, torch.nan_to_num(b_kl.sum() / n)
    return ((loss, mean, cut.sum() / n.double(), grad),
            (b_loss + 2 * S * loss.abs().nan_to_num(), b_mean + S * mean.abs().nan_to_num(), torch.tensor(2.0 ** -23, device=l.device), b_grad * (1 + u) + (u + 4 * S) * grad.abs() + tiny))


def loss_inputs(rows, length, dtype, device, seed=0, masked=0.4):
    g = torch.Generator().manual_seed(seed)
    ref = torch.log(torch.rand(rows, length, generator=g) * 0.98 + 0.01)
    logps, old = ref + 0.3 * torch.randn(rows, length, generator=g), ref + 0.2 * torch.randn(rows, length, generator=g)
    mask = torch.rand(rows, length, generator=g) >= masked
    return logps.to(device, dtype), old.to(device, dtype), ref.to(device, dtype), mask.to(device), torch.randn(rows, length, generator=g).to(device)
