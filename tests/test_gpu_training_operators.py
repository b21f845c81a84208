"""The training operators' kernels against their formulas in 64 bits: ragged sizes, masks, strides, streams, graphs, wrong targets."""
import pytest
import torch
from training_operators import adam_by_formula, loss_by_formula, loss_inputs, within

from oxibonsai_b200 import training as TR

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
UP = {torch.float16: 1024.0}


def run_loss(h, w, t, up=None, reduction="mean", smoothing=0.0, want="hw", ignore_index=-100):
    h, w = h.detach().requires_grad_("h" in want), w.detach().requires_grad_("w" in want)
    loss = TR.linear_cross_entropy(h, w, t, ignore_index=ignore_index, reduction=reduction, label_smoothing=smoothing)
    grads = torch.autograd.grad(loss, [x for x in (h, w) if x.requires_grad], up if up is not None else torch.ones_like(loss)) if want else ()
    return (loss.detach(), *grads)


def compare(h, w, t, up=None, reduction="mean", smoothing=0.0, ignore_index=-100):
    got = run_loss(h, w, t, up, reduction, smoothing, ignore_index=ignore_index)
    want, bound = loss_by_formula(h, w, t, up, ignore_index, reduction, smoothing)
    assert got[0].dtype == torch.float32 and got[1].dtype == h.dtype and got[2].dtype == w.dtype
    for g, x, b, what in zip(got, want, bound, ("loss", "dh", "dw")):
        within(g, x, b, what)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, v, d", [(1, 1, 1), (1, 2, 8), (3, 257, 63), (129, 1000, 64), (256, 256, 128), (257, 513, 200), (300, 5000, 1001), (64, 40000, 136),
                                     (5, 151936, 64), (1000, 31, 72), (2, 300, 2056), (700, 3000, 520),
                                     (8, 5001, 63), (9, 700, 264), (16, 3001, 520), (17, 90, 31), (24, 20000, 100), (25, 20000, 100), (8, 257, 4100), (128, 600, 72)])
def test_loss_sizes(n, v, d, dtype):
    h, w, t = loss_inputs(n, v, d, dtype, DEV, seed=n + v + d, masked=0.0 if n < 4 else 0.2)
    compare(h, w, t, torch.tensor(UP.get(dtype, 1.0), device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction, smoothing", [("mean", 0.1), ("sum", 0.0), ("none", 0.0), ("none", 0.3)])
def test_loss_reductions(reduction, smoothing, dtype):
    h, w, t = loss_inputs(200, 700, 96, dtype, DEV, seed=5, masked=0.3)
    up = torch.rand(200, device=DEV) if reduction == "none" else torch.tensor(0.5, device=DEV)
    if reduction == "none":
        up[7], up[11] = 0.0, -3.0
    compare(h, w, t, up * UP.get(dtype, 1.0), reduction, smoothing)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 8, 20, 24])
def test_loss_few_rows(n, dtype):
    """The forms of a few rows: masks, each gradient alone, sums over rows, rows of the head with gaps between them."""
    h, w, t = loss_inputs(n, 900, 136, dtype, DEV, seed=40 + n)
    up = torch.rand(n, device=DEV) * UP.get(dtype, 1.0)
    if n > 1:
        t[1], t[n - 1] = -100, 899
        h[1] = float("inf")
    wide = torch.zeros(900, 144, dtype=dtype, device=DEV)
    wide[:, 8:] = w
    clean = torch.where((t == -100)[:, None], 0.0, h)
    want, bound = loss_by_formula(clean, w, t, up, reduction="none", smoothing=0.2)
    for head in (w, wide[:, 8:], wide[:, 8:].T.contiguous().T):
        got = run_loss(h, head, t, up, "none", 0.2)
        for g, x, b, what in zip(got, want, bound, ("loss", "dh", "dw")):
            within(g, x, b, what)
        assert torch.equal(run_loss(h, head, t, up, "none", 0.2, want="w")[1], got[2]) and torch.equal(run_loss(h, head, t, up, "none", 0.2, want="h")[1], got[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", ["all", "all but one", "first", "tail", "odd"])
def test_loss_masks(mask, dtype):
    h, w, t = loss_inputs(530, 300, 64, dtype, DEV, seed=9)
    i = torch.arange(530, device=DEV)
    dead = {"all": i >= 0, "all but one": i != 400, "first": i < 300, "tail": i > 100, "odd": i % 2 == 1}[mask]
    t = torch.where(dead, -100, t)
    want, bound = loss_by_formula(h, w, t)
    h[dead] = float("nan")              # what padded rows hold reaches nothing
    got = run_loss(h, w, t)
    for g, x, b, what in zip(got, want, bound, ("loss", "dh", "dw")):
        within(g, x, b, what)
    assert not got[1][dead].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_strides_and_orders(dtype):
    h, w, t = loss_inputs(70, 400, 48, dtype, DEV, seed=2)
    wide = torch.zeros(70, 61, dtype=dtype, device=DEV)
    wide[:, 3:51] = h                    # rows that begin at odd places
    tall = torch.zeros(400, 56, dtype=dtype, device=DEV)
    tall[:, :48] = w
    compare(wide[:, 3:51], tall[:, :48], t)
    compare(h.T.contiguous().T, w.T.contiguous().T, t.int())
    compare(h[:1].expand(70, 48), w, t)
    odd = torch.zeros(400 * 48 + 1, dtype=dtype, device=DEV)
    odd[1:] = w.flatten()
    compare(h, odd[1:].view(400, 48), t)
    a = run_loss(h.view(7, 10, 48), w, t.view(7, 10), reduction="none")
    b = run_loss(h, w, t, reduction="none")
    assert a[0].shape == (7, 10) and torch.equal(a[0].flatten(), b[0]) and torch.equal(a[1].flatten(0, 1), b[1]) and torch.equal(a[2], b[2])
    compare(h[:1].T.contiguous().T, w, t[:1])                     # a single row may have any stride
    compare(h[:, :1], w[:1, :1], torch.zeros_like(t))
    compare(h[:, 5:6], w[:, 7:8], t)
    one = run_loss(h[0], w, t[0])
    assert one[0].shape == () and one[1].shape == (48,)


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_wanted_gradients(dtype):
    h, w, t = loss_inputs(150, 600, 80, dtype, DEV, seed=4, masked=0.1)
    both = run_loss(h, w, t)
    assert torch.equal(run_loss(h, w, t, want="")[0], both[0])
    assert torch.equal(run_loss(h, w, t, want="h")[1], both[1])
    assert torch.equal(run_loss(h, w, t, want="w")[1], both[2])
    again = run_loss(h, w, t)
    assert all(torch.equal(x, y) for x, y in zip(both, again))
    h.requires_grad_()
    loss = TR.linear_cross_entropy(h, w, t)
    first = torch.autograd.grad(loss, h, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(loss, h)[0]) and torch.equal(first, both[1])
    spread = TR.linear_cross_entropy(h, w, t, reduction="none")
    each = torch.autograd.grad(spread.sum(), h, create_graph=False)[0]          # a gradient of stride 0 comes in
    assert torch.equal(each, run_loss(h.detach(), w, t, reduction="none")[1])


def test_loss_gradient_by_differences():
    h, w, t = loss_inputs(6, 50, 16, torch.float32, DEV, seed=8)
    _, dh, dw = run_loss(h, w, t, reduction="sum")
    g = torch.Generator().manual_seed(1)
    for grad, which in ((dh, 0), (dw, 1)):
        x = (h, w)[which]
        way = torch.randn(x.shape, generator=g).to(DEV)
        e = 2.0 ** -6
        ends = [float(run_loss(*((x + s * e * way, w) if which == 0 else (h, x + s * e * way)), t, reduction="none", want="")[0].double().sum()) for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * e)
        # third derivatives of six rows along a direction of length |way| leave e^2 |way . z'|^3 / 6 each; rounding leaves 2^-20 / e
        reach = (way @ w.T if which == 0 else h @ way.T).abs().max().item()
        assert abs(slope - float((grad * way).sum())) <= 6 * e * e * reach ** 3 / 6 + 2.0 ** -20 * 6 / e


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_wrong_targets(dtype):
    h, w, t = loss_inputs(40, 90, 32, dtype, DEV, seed=6)
    t[3], t[17], t[20] = 90, -7, -100
    loss, dh, dw = run_loss(h, w, t, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 17]] = True
    assert torch.equal(loss.isnan(), bad) and torch.equal(dh.isnan().any(1), bad) and dw.isnan().all() and not dh[20].any()
    assert run_loss(h, w, t, want="")[0].isnan()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [9, 300])
def test_loss_upstream_gradients(n, dtype):
    """Ignored rows have no gradient whatever comes from above; rows with an upstream gradient of 0 have none; sizes far apart keep their rows exact."""
    h, w, t = loss_inputs(n, 400, 72, dtype, DEV, seed=50)
    t[2] = -100
    for bad in (float("inf"), float("nan")):
        _, dh, dw = run_loss(h, w, t, torch.tensor(bad, device=DEV))
        assert not dh[2].any() and dh[0].isnan().all() and dw.isnan().all()
    up = torch.ones(n, device=DEV)
    up[0], up[1] = 0.0, float("nan")
    _, dh, _ = run_loss(h, w, t, up, "none")
    assert not dh[0].any() and not dh[2].any() and dh[1].isnan().all() and dh[3:].isfinite().all()
    up = torch.logspace(0, -4, n, device=DEV)
    compare(h, w, t, up * UP.get(dtype, 1.0), "none")
    assert not run_loss(h, w, t, torch.zeros((), device=DEV))[1].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_far_logits(dtype):
    """Logits of hundreds: the largest carries the softmax, the others vanish; equal logits share it."""
    v, d = 600, 64
    h = torch.zeros(4, d, device=DEV, dtype=dtype)
    h[:3, 0] = torch.tensor([30.0, -30.0, 0.0], device=DEV).to(dtype)
    w = torch.zeros(v, d, device=DEV, dtype=dtype)
    w[:, 0] = torch.linspace(-16, 16, v, device=DEV).to(dtype)
    t = torch.tensor([v - 1, v - 1, 5, 599], device=DEV)
    got = compare(h, w, t, reduction="none")
    assert got[0][0] < 3 and got[0][1] > 900


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_not_finite_inputs(dtype):
    h, w, t = loss_inputs(20, 300, 64, dtype, DEV, seed=11)
    h[4, 5] = float("nan")
    loss, dh, dw = run_loss(h, w, t, reduction="none")
    bad = torch.arange(20, device=DEV) == 4
    assert torch.equal(loss.isnan(), bad) and torch.equal(dh.isnan().all(1), bad) and dw.isnan().all()


def test_loss_on_another_stream_and_in_a_graph():
    h, w, t = loss_inputs(300, 2000, 128, torch.bfloat16, DEV, seed=12, masked=0.2)
    want = run_loss(h, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = run_loss(h, w, t), run_loss(h, w, t, reduction="sum")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a, want)) and not torch.equal(b[0], want[0])
    sh, sw, st = h.clone().requires_grad_(), w.clone().requires_grad_(), t.clone()
    graphs = []
    for reduction in ("mean", "sum"):          # two graphs over the same tensors, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss = TR.linear_cross_entropy(sh, sw, st, reduction=reduction)
            grads = torch.autograd.grad(loss, [sh, sw])
        graphs.append((g, loss, grads, reduction))
    for seed in (13, 14):
        h2, w2, t2 = loss_inputs(300, 2000, 128, torch.bfloat16, DEV, seed=seed, masked=0.5 if seed == 13 else 0.0)
        with torch.no_grad():
            sh.copy_(h2), sw.copy_(w2), st.copy_(t2)
        for g, loss, grads, reduction in graphs:
            g.replay()
            want = run_loss(h2, w2, t2, reduction=reduction)
            assert torch.equal(loss, want[0]) and torch.equal(grads[0], want[1]) and torch.equal(grads[1], want[2])


def test_loss_from_threads():
    """Each pass as the first thing that a thread does on the GPU, and two threads at once."""
    import threading

    from oxibonsai_b200.ops import train_ops

    h, w, t = loss_inputs(40, 500, 64, torch.bfloat16, DEV, seed=15)
    want = run_loss(h, w, t)
    got = {}

    def go(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            loss, kept = train_ops.linear_ce_forward(h, w, t, -100, "mean", 0.0)
            torch.cuda.current_stream().synchronize()
            second = threading.Thread(target=lambda: got.__setitem__((i, "back"), train_ops.linear_ce_backward(w, kept, 40, torch.ones((), device=DEV), "mean", 0.0, True, True)))
            second.start(), second.join()
            got[i, "loss"] = loss
    threads = [threading.Thread(target=go, args=(i,)) for i in range(2)]
    torch.cuda.synchronize()
    [x.start() for x in threads], [x.join() for x in threads]
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i, "loss"], want[0]) and torch.equal(got[i, "back"][0], want[1]) and torch.equal(got[i, "back"][1], want[2])


def test_loss_in_several_pieces():
    """Enough rows that the gradient of the logits goes through several pieces of the vocabulary."""
    h, w, t = loss_inputs(6000, 70000, 64, torch.bfloat16, DEV, seed=21, masked=0.1)
    got = run_loss(h, w, t)
    part = slice(0, 6000, 37)
    live = t != -100
    rows = torch.zeros(6000, device=DEV)
    rows[part] = 1.0
    rows = (rows * live) / live.sum()
    (_, dh, _), (_, bh, _) = loss_by_formula(h[part], w, t[part], rows[part], reduction="none")
    within(got[1][part], dh, bh, "dh")
    z = h.double() @ w[69900:].double().T
    lse = torch.cat([torch.logsumexp(x.double() @ w.double().T, 1) for x in h.split(500)])
    dz = (z - lse[:, None]).exp() - (t[:, None] == torch.arange(69900, 70000, device=DEV)).double()
    dz = torch.where(live[:, None], dz, 0.0) / live.sum()
    want = dz.T @ h.double()
    bound = (dz.abs() * 2.0 ** -7).T @ h.double().abs() + want.abs() * 2.0 ** -8        # the products' errors are well below another half step of dz
    within(got[2][69900:], want, bound, "dw")


def test_loss_refusals_on_cuda():
    h, w, t = loss_inputs(4, 10, 8, torch.bfloat16, DEV)
    for bad, error in ((lambda: TR.linear_cross_entropy(h, w.float(), t), TypeError), (lambda: TR.linear_cross_entropy(h.double(), w.double(), t), TypeError),
                       (lambda: TR.linear_cross_entropy(h, w, t.cpu()), ValueError), (lambda: TR.linear_cross_entropy(h, w.cpu(), t), ValueError)):
        with pytest.raises(error):
            bad()


# ---- many tensors ---------------------------------------------------------------------------------------------------------------------
def ragged(sizes, dtypes, seed=0, odd=False, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        x = (torch.randn(n + 1, generator=g) * scale).to(DEV, dtypes[i % len(dtypes)])
        out.append(x[1:] if odd else x[:n].clone())
    return out


SETS = [([1], False), ([5, 0, 4096, 129], False), ([7, 100003, 8, 1, 300], True), ([33] * 1100, False), ([64] * 513, True), ([3_000_001, 17], False)]


@pytest.mark.parametrize("sizes, odd", SETS)
@pytest.mark.parametrize("types", [[torch.float32], [torch.bfloat16], [torch.float16, torch.float32, torch.bfloat16]])
def test_norm_and_clip(sizes, odd, types):
    grads = ragged(sizes, types, seed=len(sizes), odd=odd)
    want = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    s = TR.GradientSet(grads)
    assert abs(float(s.norm()) - float(want)) <= 2.0 ** -21 * float(want)          # f32 squares and sums of eight: below 8 half steps
    outs = ragged(sizes, types[::-1], seed=1, odd=not odd)
    before = [g.clone() for g in grads]
    n = TR.GradientSet(grads, out=outs).clip(0.5 * float(want))
    assert torch.equal(n, s.norm()) and all(torch.equal(a, b) for a, b in zip(grads, before))
    share = 0.5 * float(want) / (float(want) + 1e-6)
    for g, o in zip(grads, outs):
        x = g.double() * share
        u = max(2.0 ** -20, {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}.get(o.dtype, 0.0))
        assert ((o.double() - x).abs() <= x.abs() * (u + 2.0 ** -20) + 2.0 ** -25).all()
    assert torch.equal(s.clip(2.0 * float(want)), n) and all(torch.equal(a, b) for a, b in zip(grads, before))
    TR.GradientSet(grads, out=outs).clip(2.0 * float(want))
    assert all(torch.equal(o, g.to(o.dtype)) for g, o in zip(grads, outs))
    s.clip(0.5 * float(want))
    for g, b in zip(grads, before):
        x = b.double() * share
        u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}.get(g.dtype, 0.0)
        assert ((g.double() - x).abs() <= x.abs() * (u + 2.0 ** -20) + 2.0 ** -25).all()


def test_norm_of_extremes():
    big = torch.full((1000,), 1e25, device=DEV)                   # squares beyond f32
    assert float(TR.GradientSet([big]).norm()) == pytest.approx(1e25 * 1000 ** 0.5, rel=1e-6)
    small = torch.full((1000,), 1e-30, device=DEV)
    assert float(TR.GradientSet([small]).norm()) == pytest.approx(1e-30 * 1000 ** 0.5, rel=1e-6)
    assert TR.GradientSet([torch.zeros(100, device=DEV)]).norm() == 0
    x = torch.ones(100, device=DEV)
    x[50] = float("nan")
    assert TR.GradientSet([x]).clip(1.0).isnan() and x[0] == 1
    x[50] = float("inf")
    assert TR.GradientSet([x]).clip(1.0).isinf() and x[0] == 0 and x[50].isnan()
    assert TR.GradientSet([torch.empty(0, device=DEV)]).norm().device.type == "cuda"


def test_clip_functions_and_graph():
    ps = [torch.ones(300, 7, device=DEV, requires_grad=True), torch.ones(11, device=DEV, requires_grad=True)]
    for p in ps:
        p.grad = torch.full_like(p, 2.0)
    want = 2.0 * (2111 ** 0.5)
    assert float(TR.global_grad_norm(ps)) == pytest.approx(want, rel=1e-6)
    s = TR.GradientSet([p.grad for p in ps])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n = s.clip(1.0)
    for fill in (2.0, 4.0, 1e-4):
        for p in ps:
            p.grad.fill_(fill)
        g.replay()
        was = fill * 2111 ** 0.5
        assert float(n) == pytest.approx(was, rel=1e-6) and float(ps[1].grad[3]) == pytest.approx(fill * min(1.0, 1.0 / was), rel=1e-5)
    assert float(TR.clip_global_norm(ps, 1.0)) == pytest.approx(1e-4 * 2111 ** 0.5, rel=1e-6)


@pytest.mark.parametrize("sizes, odd", SETS)
@pytest.mark.parametrize("ptype, gtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("kind, max_norm", [(TR.FusedAdamW, 1.0), (TR.FusedAdam, None)])
def test_adam(sizes, odd, ptype, gtype, kind, max_norm):
    params = ragged(sizes, [ptype], seed=1, odd=odd)
    grads = ragged(sizes, [gtype], seed=2, odd=odd, scale=0.1)
    m, v = ragged(sizes, [torch.float32], seed=3, odd=odd, scale=0.01), [x.square() for x in ragged(sizes, [torch.float32], seed=4, odd=odd, scale=0.1)]
    lr, betas, eps, decay = 0.01, (0.9, 0.95), 1e-8, 0.1
    want = adam_by_formula(params, grads, m, v, 8, lr, betas, eps, decay, kind.decoupled, max_norm)
    before, m0 = [p.clone() for p in params], [x.double() for x in m]
    opt = kind(params, lr=lr, betas=betas, eps=eps, weight_decay=decay, grads=grads, state=(m, v), steps=7)
    norm = opt.step(max_norm=max_norm)
    assert opt.t == 8 and (norm is None if max_norm is None else abs(float(norm) - float(want[3])) <= 2.0 ** -21 * float(want[3]))
    u = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[ptype]
    for i, p in enumerate(params):
        # in f32, roundings of 2^-24: the decayed gradient is off by two of its parts, m by four of its parts and v by a dozen of itself and
        # by 2 |g'| times what g' is off by; the update m / sqrt(v) by what m is off by, and by half of v's share and four roundings
        x, extra = before[i].double(), 0.0 if kind.decoupled else decay
        g = grads[i].double() * (1.0 if max_norm is None or float(want[3]) <= max_norm else max_norm / (float(want[3]) + 1e-6)) + extra * x
        gmag = grads[i].double().abs() + extra * x.abs()
        off_m, off_v = 2.0 ** -22 * (m0[i].abs() + gmag), 2.0 ** -20 * (want[2][i] + g.abs() * gmag)
        assert ((m[i].double() - want[1][i]).abs() <= off_m).all() and ((v[i].double() - want[2][i]).abs() <= off_v).all()
        root = (want[2][i] / (1 - betas[1] ** 8)).sqrt() + eps
        off_p = lr / (1 - betas[0] ** 8) / root * (off_m + want[1][i].abs() * (off_v / (2 * want[2][i]) + 2.0 ** -21))
        assert ((p.double() - want[0][i]).abs() <= u * want[0][i].abs() + 2.0 ** -22 * x.abs() + off_p + (2.0 ** -25 if ptype == torch.float16 else 0.0)).all()


def test_adam_without_fixed_gradients():
    g = torch.Generator().manual_seed(5)
    a = [torch.randn(40, 30, generator=g).to(DEV).requires_grad_(), torch.randn(9, generator=g).to(DEV).requires_grad_()]
    b = [x.detach().clone().requires_grad_() for x in a]
    fa, ba = TR.FusedAdamW(a, lr=0.01), TR.AdamW(b, lr=0.01)
    for i in range(4):
        for p, q in zip(a, b):
            x = torch.randn(p.shape, generator=g).to(DEV)
            p.grad, q.grad = (x.T.contiguous().T if x.dim() == 2 else x), x.clone()      # laid out in another order than its parameter
        if i == 1:
            a[1].grad = b[1].grad = None
        n = TR.clip_grad_norm(b, 1.0)
        was = a[0]._version
        assert float(fa.step(max_norm=1.0)) == pytest.approx(n, rel=1e-5) and a[0]._version > was
        ba.step()
    for p, q in zip(a, b):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)
    fa.zero_grad()
    assert fa.step(max_norm=1.0) == 0 and fa.t == 5


def test_adam_follows_replaced_parameters():
    p = torch.ones(1000, device=DEV, requires_grad=True)
    p.grad = torch.ones(1000, device=DEV)
    opt = TR.FusedAdam([p], lr=0.1)
    opt.step()
    old = p.data
    p.data = p.data.clone()
    opt.step()
    assert float(p[0].detach()) < float(old[0]) - 0.05                   # the new memory was stepped, the old one not
    p.data = torch.ones(500, 2, device=DEV)
    p.grad = torch.ones(500, 2, device=DEV)
    with pytest.raises(ValueError):
        opt.step()
    x = torch.full((64,), 3.0, device=DEV)
    s = TR.GradientSet([x])
    x.data = torch.zeros(64, device=DEV)
    assert float(s.norm()) == 24.0                                        # a set keeps the memory that it was made with


def test_adam_in_a_graph():
    p, g = [torch.ones(1000, device=DEV)], [torch.ones(1000, device=DEV)]
    q, lr = [torch.ones(1000, device=DEV)], torch.tensor(0.1, device=DEV)
    opt, plain = TR.FusedAdamW(p, grads=g), TR.FusedAdamW(q, grads=[g[0].clone()])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = opt.step(lr=lr, max_norm=1.0)
    for i in range(3):
        lr.fill_(0.1 / (i + 1))
        graph.replay()
        want = plain.step(lr=0.1 / (i + 1), max_norm=1.0)
        assert torch.equal(n, want) and torch.allclose(p[0], q[0], rtol=2.0 ** -22)
    assert opt.t == 3


def test_a_training_step_together():
    """Head and hidden projection trained for three steps: the loss without logits, clipping and AdamW, against 64-bit torch."""
    torch.manual_seed(0)
    n, v, d = 200, 900, 64
    h, head, t = loss_inputs(n, v, d, torch.float32, DEV, seed=30, masked=0.2)
    proj = torch.eye(d, device=DEV) + 0.01 * torch.randn(d, d, device=DEV)
    ours, theirs = [proj.clone().requires_grad_(), head.clone().requires_grad_()], [proj.double().requires_grad_(), head.double().requires_grad_()]
    a, b = TR.FusedAdamW(ours, lr=1e-3), torch.optim.AdamW(theirs, lr=1e-3, weight_decay=0.01)
    for _ in range(3):
        a.zero_grad(), b.zero_grad()
        loss = TR.linear_cross_entropy(h @ ours[0], ours[1], t, label_smoothing=0.1)
        loss.backward()
        want = torch.nn.functional.cross_entropy(h.double() @ theirs[0] @ theirs[1].T, t, label_smoothing=0.1)
        want.backward()
        assert float(loss.detach()) == pytest.approx(float(want.detach()), rel=1e-5)
        for p, q in zip(ours, theirs):
            assert float((p.grad.double() - q.grad).norm()) <= 1e-4 * float(q.grad.norm())
        norm = torch.nn.utils.clip_grad_norm_(theirs, 0.1)
        assert float(a.step(max_norm=0.1)) == pytest.approx(float(norm), rel=1e-4)
        b.step()
    reg = TR.LoraRegistry(TR.LoraConfig(rank=4))
    reg.add("lin", d, d, seed=1)
    for adapter in reg.adapters.values():
        adapter.to(DEV)
    tr = TR.LoraTrainer(reg, TR.LoraTrainingConfig(lr=0.01, total_steps=3, fused=True))
    while not tr.is_complete():
        s = tr.step(lambda: TR.linear_cross_entropy(reg.apply_adapter("lin", h, h), head, t))
        assert s.grad_norm > 0 and s.loss > 0


# ---- places past 32 bits ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n, v, d", [(530_000, 300, 4096), (24, 530_000, 4096), (600_000, 8192, 64)])
def test_loss_far_places(n, v, d):
    """Hidden states, a head and a piece of the logits' gradient of more than 2^31 values: rows at both ends against the formula."""
    g = torch.Generator(device=DEV).manual_seed(n)
    h = torch.empty(n, d, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    w = torch.empty(v, d, dtype=torch.bfloat16, device=DEV).normal_(0, 1.28 / d ** 0.5, generator=g)
    t = torch.randint(0, v, (n,), generator=g, device=DEV)
    t[n // 2] = -100
    up = torch.rand(n, generator=g, device=DEV)
    loss, dh, dw = run_loss(h, w, t, up, "none")
    ends = torch.tensor(sorted({0, 1, n // 2, n - 2, n - 1}), device=DEV)
    want, bound = loss_by_formula(h[ends], w, t[ends], up[ends], reduction="none")
    within(loss[ends], want[0], bound[0], "loss")
    within(dh[ends], want[1], bound[1], "dh")
    for rows in (slice(0, 2), slice(v - 2, v)):
        total = torch.zeros(2, d, dtype=torch.float64, device=DEV)
        size = torch.zeros(2, d, dtype=torch.float64, device=DEV)
        for a in range(0, n, 20_000):
            x = h[a:a + 20_000].double()
            lse = loss[a:a + 20_000].double() + (x * w[t[a:a + 20_000].clamp_min(0)].double()).sum(1)          # the loss is within its bound above
            q = (t[a:a + 20_000, None] == torch.arange(v, device=DEV)[rows]).double()
            dz = ((x @ w[rows].double().T - lse[:, None]).exp() - q) * torch.where(t[a:a + 20_000] == -100, 0.0, up[a:a + 20_000].double())[:, None]
            total += dz.T @ x
            size += dz.abs().T @ x.abs()
        # dz is rounded by half a step, its exponent is off by less than another, the sums truncate by 2^-23 for each token
        within(dw[rows], total, size * (2.0 ** -7 + n * 2.0 ** -23) + total.abs() * 2.0 ** -8, "dw")


def test_many_values():
    n = 2 ** 31 + 4099
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.empty(n, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    small = torch.ones(5, device=DEV)
    want = sum(float(part.double().square().sum()) for part in x.split(1 << 28)) + 5
    s = TR.GradientSet([x, small])
    tail = x[-4099:].clone()
    norm = s.clip(1.0)
    assert float(norm) == pytest.approx(want ** 0.5, rel=2.0 ** -20)
    assert torch.equal(x[-4099:], (tail.float() * (1.0 / (want ** 0.5 + 1e-6))).to(torch.bfloat16)) or torch.allclose(
        x[-4099:].float(), tail.float() / want ** 0.5, rtol=2.0 ** -7)
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    TR.FusedAdam([p], lr=1.0, grads=[x], state=([m], [v]), eps=0.0).step()
    live = x[-4099:] != 0
    assert torch.equal(p[-4099:][live], -x[-4099:][live].sign()) and torch.allclose(m[-4099:], 0.1 * x[-4099:].float(), rtol=2.0 ** -22)
