"""The training operators without a GPU: their torch forms against the formulas, gradients by differences, refusals."""
import math

import pytest
import torch
from training_operators import adam_by_formula, loss_by_formula, loss_inputs, within

from oxibonsai_b200 import training as TR


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing", [0.0, 0.2])
def test_linear_cross_entropy_against_formula_and_differences(reduction, smoothing, monkeypatch):
    monkeypatch.setattr(TR.linear_loss, "_PIECE", 5)           # several pieces, the last one short
    h, w, t = loss_inputs(9, 13, 6, torch.float64, "cpu", masked=0.3)
    h.requires_grad_(), w.requires_grad_()
    loss = TR.linear_cross_entropy(h, w, t, reduction=reduction, label_smoothing=smoothing)
    want = torch.nn.functional.cross_entropy(h @ w.T, t, reduction=reduction, label_smoothing=smoothing)
    assert torch.allclose(loss, want, rtol=1e-12)
    assert torch.autograd.gradcheck(lambda h, w: TR.linear_cross_entropy(h, w, t, reduction=reduction, label_smoothing=smoothing), (h, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_linear_cross_entropy_types(dtype):
    h, w, t = loss_inputs(33, 70, 24, dtype, "cpu", masked=0.2)
    h.requires_grad_(), w.requires_grad_()
    loss = TR.linear_cross_entropy(h.view(3, 11, 24), w, t.view(3, 11).int())
    loss.backward()
    want, bound = loss_by_formula(h.detach(), w.detach(), t)
    assert loss.dtype == torch.float32 and h.grad.dtype == dtype
    for got, x, b, what in zip((loss.detach(), h.grad, w.grad), want, bound, ("loss", "dh", "dw")):
        within(got, x, b, what)


def test_linear_cross_entropy_masked_rows():
    h, w, t = loss_inputs(6, 20, 8, torch.float32, "cpu")
    t[2], t[5] = -100, -100
    h[2], h[5, 0] = float("nan"), float("inf")                   # padding may hold anything
    h.requires_grad_(), w.requires_grad_()
    loss = TR.linear_cross_entropy(h, w, t)
    loss.backward()
    assert loss.isfinite() and w.grad.isfinite().all() and not h.grad[[2, 5]].any() and h.grad[0].any()
    none = TR.linear_cross_entropy(h, w, torch.full_like(t, -100))
    none.backward()
    assert none.isnan() and TR.linear_cross_entropy(h, w, torch.full_like(t, -100), reduction="sum") == 0
    assert TR.linear_cross_entropy(h, w, torch.where(t == -100, 7, t), ignore_index=7, reduction="none")[2] == 0
    empty = TR.linear_cross_entropy(h[:0], w, t[:0], reduction="sum")
    empty.backward()
    assert empty == 0 and TR.linear_cross_entropy(h[:0], w, t[:0]).isnan() and TR.linear_cross_entropy(h[:0], w, t[:0], reduction="none").shape == (0,)


def test_linear_cross_entropy_has_no_second_derivative():
    h, w, t = loss_inputs(5, 12, 6, torch.float64, "cpu")
    h.requires_grad_(), w.requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(TR.linear_cross_entropy(h, w, t), [h, w], create_graph=True)


def test_next_token_forms():
    h, w, t = loss_inputs(12, 30, 16, torch.float32, "cpu")
    assert torch.allclose(TR.linear_ntp_loss(h, w, t), TR.ntp_loss(h @ w.T, t), rtol=1e-5)
    assert TR.linear_sequence_perplexity(h, w, t) == pytest.approx(TR.sequence_perplexity(h @ w.T, t), rel=1e-5)


def test_linear_cross_entropy_refusals():
    h, w, t = loss_inputs(4, 10, 8, torch.float32, "cpu")
    for bad, error in ((lambda: TR.linear_cross_entropy(h[:, :5], w, t), ValueError), (lambda: TR.linear_cross_entropy(h, w[0], t), ValueError),
                       (lambda: TR.linear_cross_entropy(h, w, t[:3]), ValueError), (lambda: TR.linear_cross_entropy(h, w, t.float()), TypeError),
                       (lambda: TR.linear_cross_entropy(h, w, t, reduction="batch"), ValueError), (lambda: TR.linear_cross_entropy(h.half(), w, t), TypeError),
                       (lambda: TR.linear_cross_entropy(h, w, t, label_smoothing=1.5), ValueError), (lambda: TR.linear_cross_entropy(h.int(), w.int(), t), TypeError),
                       (lambda: TR.linear_cross_entropy(h, w[:0], t), ValueError),
                       (lambda: TR.linear_cross_entropy(h.to("meta"), w.to("meta"), t.to("meta")), ValueError), (lambda: TR.linear_cross_entropy(h, w, t + 10), IndexError),
                       (lambda: TR.linear_cross_entropy(h, w, t - 20), IndexError)):
        with pytest.raises(error):
            bad()


def test_gradient_set():
    a, b = torch.tensor([3.0, 0.0]), torch.tensor([[4.0]], dtype=torch.bfloat16)
    s = TR.GradientSet([a, b, torch.empty(0)])
    assert len(s) == 3 and s.norm() == 5.0 and s.norm().dtype == torch.float32
    out = [torch.zeros(2, dtype=torch.float16), torch.zeros(1, 1), torch.empty(0)]
    assert TR.GradientSet([a, b, torch.empty(0)], out=out).clip(1.0) == 5.0 and a[0] == 3.0
    assert out[0][0] == pytest.approx(0.6, rel=2e-3) and out[1].item() == pytest.approx(0.8, rel=1e-6)
    assert s.clip(10.0) == 5.0 and a[0] == 3.0 and s.clip(0.0) == 5.0 and a[0] == 3.0
    assert s.clip(2.5) == 5.0 and a[0] == pytest.approx(1.5, rel=1e-6)
    a[0] = float("nan")
    assert s.clip(1.0).isnan() and a[1] == 0.0
    assert TR.GradientSet([]).norm() == 0 and TR.GradientSet([]).clip(1.0) == 0
    p = torch.ones(4, requires_grad=True)
    (p * torch.tensor([3.0, 4.0, 0.0, 0.0])).sum().backward()
    q = torch.ones(2, requires_grad=True)
    assert TR.global_grad_norm([p, q]) == 5.0 and TR.clip_global_norm([p, q], 1.0) == 5.0 and TR.grad_norm([p]) == pytest.approx(1.0, rel=1e-5)


def test_written_tensors_count_a_version():
    flat, single = torch.ones(10), torch.ones(3)
    views = [flat[:4], flat[5:]]
    was = [t._version for t in (flat, single)]
    TR.GradientSet(views + [single]).clip(1.0)
    assert flat._version > was[0] and single._version > was[1]
    p = torch.ones(3, requires_grad=True)
    y = (p * p).sum()
    opt = TR.FusedAdam([p], grads=[torch.ones(3)])
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        TR.GradientSet([torch.ones(3)]).clip(1.0)


def test_gradient_set_refusals():
    a = torch.zeros(8)
    for bad, error in ((lambda: TR.GradientSet([a, a]), ValueError), (lambda: TR.GradientSet([a[:5], a[4:]]), ValueError),
                       (lambda: TR.GradientSet([torch.zeros(4, 4)[:, :2]]), ValueError), (lambda: TR.GradientSet([torch.zeros(1).expand(3)]), ValueError),
                       (lambda: TR.GradientSet([a.double()]), TypeError), (lambda: TR.GradientSet([[1.0]]), TypeError),
                       (lambda: TR.GradientSet([a], out=[a[:4]]), ValueError), (lambda: TR.GradientSet([a], out=[]), ValueError),
                       (lambda: TR.GradientSet([a], out=[a.view(torch.bfloat16)[:8]]), ValueError),
                       (lambda: TR.GradientSet([torch.zeros(2, 3)], out=[torch.zeros(3, 2).T]), ValueError),
                       (lambda: TR.GradientSet([torch.zeros(3).to_sparse()]), TypeError)):
        with pytest.raises(error):
            bad()
    TR.GradientSet([a], out=[a])
    TR.GradientSet([torch.zeros(3, 2).T])


@pytest.mark.parametrize("kind, base", [(TR.FusedAdam, TR.Adam), (TR.FusedAdamW, TR.AdamW)])
def test_fused_adam_follows_adam(kind, base):
    g = torch.Generator().manual_seed(3)
    w = [torch.randn(5, 3, generator=g), torch.randn(7, generator=g)]
    a, b = ([x.clone().requires_grad_() for x in w] for _ in range(2))
    fa, ba = kind(a, lr=0.01, weight_decay=0.1), base(b, lr=0.01, weight_decay=0.1)
    for i in range(4):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, generator=g)
            q.grad = p.grad.clone()
        if i == 2:
            a[1].grad = b[1].grad = None
        n = TR.clip_grad_norm(b, 1.0)
        kept = a[0].grad.clone()
        assert fa.step(lr=0.02, max_norm=1.0) == pytest.approx(n, rel=1e-6)
        assert torch.equal(a[0].grad, kept)
        ba.step(lr=0.02)
    assert fa.t == 4
    for p, q in zip(a, b):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-7)
    assert fa.step() is None
    fa.zero_grad()
    assert a[0].grad is None


def test_fused_adam_state_and_refusals():
    p, g = [torch.ones(4, dtype=torch.bfloat16)], [torch.full((4,), 2.0)]
    m, v = [torch.full((4,), 0.5)], [torch.full((4,), 0.25)]
    opt = TR.FusedAdamW(p, lr=0.1, grads=g, state=(m, v), steps=2)
    want = adam_by_formula(p, g, m, v, 3, 0.1, (0.9, 0.999), 1e-8, 0.01, True, 1.0)
    assert opt.step(max_norm=1.0) == 4.0 and opt.t == 3
    assert p[0][0] == want[0][0][0].to(torch.bfloat16) and torch.allclose(m[0].double(), want[1][0]) and torch.allclose(v[0].double(), want[2][0])
    opt.zero_grad()
    assert not g[0].any()
    opt.reset()
    assert opt.t == 0 and not m[0].any() and not v[0].any()
    x = torch.zeros(4)
    for bad, error in ((lambda: TR.FusedAdam([]), ValueError), (lambda: TR.FusedAdam([x, x]), ValueError), (lambda: TR.FusedAdam([x.long()]), TypeError),
                       (lambda: TR.FusedAdam([x], betas=(1.0, 0.9)), ValueError), (lambda: TR.FusedAdam([x], grads=[]), ValueError),
                       (lambda: TR.FusedAdam([x], grads=[torch.zeros(3)]), ValueError), (lambda: TR.FusedAdam([x], grads=[torch.zeros(4).double()]), TypeError),
                       (lambda: TR.FusedAdam([x], state=([torch.zeros(4)], [torch.zeros(3)])), ValueError), (lambda: TR.FusedAdam([x], state=([x], [x])), ValueError),
                       (lambda: TR.FusedAdam([torch.zeros(2, 3)], grads=[torch.zeros(3, 2).T]), ValueError),
                       (lambda: TR.FusedAdam([x]).step(lr=torch.zeros(2)), ValueError), (lambda: TR.FusedAdam([x], grads=[None]), TypeError)):
        with pytest.raises(error):
            bad()


def test_trainer_fused():
    """The whole step of a trainer whose head is frozen: loss without logits, clipping and AdamW, against the tensor-by-tensor trainer."""
    def run(fused):
        torch.manual_seed(0)
        reg = TR.LoraRegistry(TR.LoraConfig(rank=4, alpha=4.0))
        reg.add("lin", 16, 16, seed=3)
        h, w, t = loss_inputs(24, 50, 16, torch.float32, "cpu", masked=0.2)
        tr = TR.LoraTrainer(reg, TR.LoraTrainingConfig(lr=0.05, total_steps=6, warmup_steps=2, max_grad_norm=0.05, fused=fused))
        while not tr.is_complete():
            x = lambda: reg.apply_adapter("lin", h, h)  # noqa: E731
            tr.step(lambda: TR.linear_cross_entropy(x(), w, t) if fused else TR.cross_entropy(x() @ w.T, t))
        return tr
    a, b = run(True), run(False)
    for x, y in zip(a.history, b.history):
        assert x.loss == pytest.approx(y.loss, rel=1e-4) and x.grad_norm == pytest.approx(y.grad_norm, rel=1e-3) and x.lr == y.lr
    assert math.isfinite(a.history[-1].loss)
