"""Inputs on which the loss of a head has few or exact sums, so that its bounds are the arithmetic's own and not a sum's length, and these bounds.

float32 operands of the tensor cores are three bfloat16 parts, x = x0 + x1 + x2 with |x1| <= 2^-8 |x|, |x2| <= 2^-16 |x| and nothing left; of
the nine products of parts the three smallest are left out: 2^-24 + 2^-24 + 2^-32 of the product, below OUT = 2^-23 (1 + 2^-7).  An addition on the
tensor cores may truncate, 2^-23 of the sum so far: for k products that is 2^-23 k of the sum of magnitudes for the large parts' product, and a 2^-7th
and a 2^-15th of that for the two and three products below, in all SUM(k)."""
import torch

OUT = 2.0 ** -23 * (1 + 2.0 ** -7)


def SUM(k):
    return 2.0 ** -23 * k * (1 + 2 * 2.0 ** -7 + 3 * 2.0 ** -15)


def parts(x, count):
    """The first ``count`` bfloat16 parts of x, in float64."""
    out, rest = [], x.double()
    for _ in range(count):
        out.append(rest.float().bfloat16().double())
        rest = rest - out[-1]
    return out


def product(a, b, count):
    """a @ b of ``count`` parts each: products of parts i, j with i + j < 3, of two parts all four."""
    return sum(x @ y for i, x in enumerate(parts(a, count)) for j, y in enumerate(parts(b, count)) if i + j < 3)


def loss_and_gradients(h, w, t, up, mul):
    """The definition with ``mul`` as its product; each token's loss, the gradients for upstream gradients ``up``.  Results in float64."""
    live = t >= 0
    z = mul(h, w.T)
    lse = torch.logsumexp(z, 1)
    at = t.clamp_min(0)[:, None]
    loss = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    q = torch.zeros_like(z).scatter_(1, at, 1.0)
    dz = ((z - lse[:, None]).exp() - q) * torch.where(live, up.double(), 0.0)[:, None]
    return loss, mul(dz.float(), w), mul(dz.float().T, h)


def plain(a, b):
    return a.double() @ b.double()


def logits_case(n, v, d, device, seed):
    """Hidden rows of one value each: every logit is one product, and the largest is tens.  Returns inputs and the bound of each token's loss.

    |dz| <= (OUT + SUM(1)) |z|; log-sum-exp is off by the largest of those and by 2^-26 max|z| for log2(e) in float32, its sum of
    exponentials by 64 roundings and one approximate exponential (2^-22); the loss is rounded once."""
    g = torch.Generator().manual_seed(seed)
    h, w = torch.zeros(n, d), torch.randn(v, d, generator=g)
    h[torch.arange(n), torch.randint(0, d, (n,), generator=g)] = torch.randn(n, generator=g).sign() * (20 + 20 * torch.rand(n, generator=g))
    t = torch.randint(0, v, (n,), generator=g)
    z = plain(h, w.T)
    loss = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    top = z.abs().max(1).values
    bound = (OUT + SUM(1)) * (top + z.gather(1, t[:, None])[:, 0].abs()) + 2.0 ** -26 * top + 64 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -24 * loss.abs()
    return h.to(device), w.to(device), t.to(device), bound.to(device)


def gradient_case(which, n, v, d, live, device, seed):
    """Logits of 0, so that every probability is 1 / v, a power of two.  which "h": hidden rows of 0 and any head, for dh; "w": a head of 0 and any
    hidden rows, ``live`` of them with a target, for dw.  Returns inputs, upstream gradients and the bound of that gradient.

    dz is p - q in float32: a quotient, a product and a difference, 4 * 2^-24 of p + q, and the exponential's 2^-22 of p; then a product of
    v (of ``live``) terms, its factor and the rounding of the result, 3 * 2^-24."""
    g = torch.Generator().manual_seed(seed)
    h = torch.zeros(n, d) if which == "h" else torch.randn(n, d, generator=g)
    w = torch.randn(v, d, generator=g) if which == "h" else torch.zeros(v, d)
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.randperm(n, generator=g)[live:]] = -100
    up = 0.1 + torch.rand(n, generator=g)
    u = torch.where(t >= 0, up, 0.0).double()[:, None]
    q = torch.zeros(n, v, dtype=torch.float64).scatter_(1, t.clamp_min(0)[:, None], 1.0)
    dz, off = (1 / v - q).abs() * u, (4 * 2.0 ** -24 * (1 / v + q) + 2.0 ** -22 / v) * u
    a, b, k = (dz, w.double().abs(), v) if which == "h" else (dz.T, h.double().abs(), live)
    bound = (off if which == "h" else off.T) @ b + (OUT + SUM(k) + 3 * 2.0 ** -24) * (a @ b)
    return h.to(device), w.to(device), t.to(device), up.to(device), bound.to(device)


def pieces_case(n, v, d, dtype, device, seed):
    """Hidden rows of 0 and v = 2^17 head rows of 32nds between 1 and 1.75: dh = mean(w) - w_t, a small difference of large sums over the whole
    vocabulary.  Returns inputs, dh and its bound for the "sum" of the losses.

    In 16 bits p = 2^-17 is exact and p - 1 is taken for -1, off by 1 / v.  Products are multiples of 2^-22 and their sums stay below 2 in size:
    nothing is lost in float32, whatever the order, and only the result is rounded.  In float32 p is off by 2^-22 of itself, p - q by 4 * 2^-24 (p + q),
    and sums may truncate in 128 additions between two to registers and are rounded some 2^11 times behind them."""
    assert v == 2 ** 17
    g = torch.Generator(device=device).manual_seed(seed)
    w = (1 + torch.randint(0, 25, (v, d), generator=g, device=device) / 32).to(dtype)
    t = torch.randint(0, v, (n,), generator=g, device=device)
    mean, at = w.double().mean(0), w[t].double()
    size, want = mean + at.abs(), mean - at
    if dtype == torch.float32:
        bound = (OUT + SUM(128) + 2.0 ** -13) * size + 4 * 2.0 ** -24 * size + 2.0 ** -22 * mean + 2.0 ** -24 * want.abs()
    else:
        step = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
        bound = at.abs() / v + 2.0 ** -23 * size + step * want.abs()
    return torch.zeros(n, d, dtype=dtype, device=device), w, t, want, bound
