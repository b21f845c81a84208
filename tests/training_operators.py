"""Plain 64-bit forms of the training operators, and the bounds that their GPU kernels have to keep."""
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float64: 2.0 ** -53}


def loss_by_formula(hidden, weight, targets, up=None, ignore_index=-100, reduction="mean", smoothing=0.0):
    """(loss, dhidden, dweight) and a dict of bounds for each, in float64.

    Bounds, with u the half step of the inputs' type (2^-24 for float32) and s = 2^-23 per addition of a float32 sum that may truncate:
    a logit is off by at most d_i = D s sum_k |h_ik w_vk|; log-sum-exp by that and by 64 steps of float32; the loss of a row by twice that.
    exp(z - lse) is off by a factor 2 d_i + 64 s; dz is rounded to the inputs' type (u); each gradient sums dz times the other operand
    (s per addition, on the sum of magnitudes) and is rounded once (u), float16 also by 2^-25 absolute.  A float32 exp below 2^-126 may be
    taken for 0: less than 2^18 terms with operands below 2^8 leave 2^-100."""
    h, w = hidden.double(), weight.double()
    n, v, d = len(h), len(w), h.shape[1]
    u, s = HALF_STEP[hidden.dtype], 2.0 ** -23
    live = targets != ignore_index
    t = torch.where(live, targets, 0)
    hl = torch.where(live[:, None], h, 0.0)
    z = hl @ w.T
    lse = torch.logsumexp(z, 1)
    q = torch.full_like(z, smoothing / v)
    q[torch.arange(n, device=h.device), t] += 1 - smoothing
    each = torch.where(live, lse - (q * z).sum(1), 0.0)
    count = int(live.sum())
    loss = each if reduction == "none" else each.sum() if reduction == "sum" else each.sum() / count if count else each.sum() * float("nan")
    off = d * s * (hl.abs() @ w.abs().T).max(1).values
    row = 2 * (off + 64 * s * (1 + lse.abs() + z.abs().max(1).values))
    b_loss = row if reduction == "none" else row.sum() if reduction == "sum" else row.sum() / max(1, count)
    b_loss = b_loss + 2.0 ** -23 * loss.abs()
    up = torch.ones_like(loss) if up is None else up.double()
    g = up if reduction == "none" else up / max(1, count) if reduction == "mean" else up
    g = torch.where(live, g.expand(n), 0.0)[:, None]
    p = (z - lse[:, None]).exp()
    dz = (p - q) * g
    mag = (p * (1 + 2 * off[:, None] + 64 * s) + q) * g.abs()
    rel = (u + 2 * off + 64 * s)[:, None]
    tiny = 2.0 ** -25 if hidden.dtype == torch.float16 else 2.0 ** -100
    dh, dw = dz @ w, dz.T @ hl
    b_h = (mag * (rel + v * s)) @ w.abs() + u * dh.abs() + tiny
    b_w = (mag * (rel + n * s)).T @ hl.abs() + u * dw.abs() + tiny
    return (loss, dh, dw), (b_loss, b_h, b_w)


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(want.shape)}"
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    off = torch.where(want.isnan(), 0.0, (got - want).abs() - bound)
    assert float(off.max() if off.numel() else 0.0) <= 0.0, f"{what}: {float((got - want).abs().max()):.3g} off, {float(off.max()):.3g} over the bound"


def loss_inputs(n, v, d, dtype, device, seed=0, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    weight = torch.randn(v, d, generator=g) * 1.28 / d ** 0.5
    targets = torch.randint(0, v, (n,), generator=g)
    hidden = torch.randn(n, d, generator=g) + torch.rand(n, 1, generator=g) * 8 * weight[targets]
    targets[torch.rand(n, generator=g) < masked] = -100
    return hidden.to(device, dtype), weight.to(device, dtype), targets.to(device)


def adam_by_formula(params, grads, m, v, t, lr, betas, eps, decay, decoupled, max_norm):
    """One step in float64: (params, m, v, norm)."""
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    share = max_norm / (float(norm) + 1e-6) if max_norm is not None and float(norm) > max_norm > 0 else 1.0
    out = ([], [], [])
    for p, g, mi, vi in zip(params, grads, m, v):
        p, g = p.double(), g.double() * share
        if not decoupled:
            g = g + decay * p
        mi, vi = betas[0] * mi.double() + (1 - betas[0]) * g, betas[1] * vi.double() + (1 - betas[1]) * g * g
        if decoupled:
            p = p * (1 - lr * decay)
        p = p - lr * (mi / (1 - betas[0] ** t)) / ((vi / (1 - betas[1] ** t)).sqrt() + eps)
        for part, x in zip(out, (p, mi, vi)):
            part.append(x)
    return (*out, norm)
