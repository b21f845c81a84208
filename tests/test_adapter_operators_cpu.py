"""Low-rank updates, dropout and tuning losses on the CPU: formulas in 64 bits, gradients by differences, refusals."""
import math

import pytest
import torch
from adapter_operators import (loss_inputs, mask_by_formula, philox, policy_by_formula, preference_by_formula, update_by_formula, update_inputs)
from training_operators import within

from oxibonsai_b200 import training as TR

TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


def run_update(x, base, dy, a, b, scales, ids, **kw):
    x, base, a, b = (None if t is None else t.detach().requires_grad_() for t in (x, base, a, b))
    y = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales, **kw)
    grads = torch.autograd.grad(y, [t for t in (x, a, b, base) if t is not None], dy)
    assert base is None or torch.equal(grads[3], dy)
    return (y.detach(), *grads[:3])


def compare(got, want, names):
    for g, w, b, what in zip(got, *want, names):
        within(g, w, b, what)


def test_philox_known_answers():
    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("seed", [0, 5, 2 ** 32 + 7, 2 ** 63 + 11, 2 ** 64 - 1])
def test_dropout_bits(seed):
    x = torch.ones(5, 21, dtype=torch.float64)
    y = TR.dropout(x, 0.3, seed=seed)
    places = [(r, c) for r in range(5) for c in range(21)]
    assert torch.equal((y != 0).flatten(), mask_by_formula(places, 0.3, seed))
    steps = round(0.7 * 65536)
    assert torch.equal(y[y != 0], torch.full_like(y[y != 0], 65536 / steps))


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_values_and_gradient(dtype):
    x = torch.randn(3, 7, 33, dtype=torch.float64).to(dtype)
    x[0, 0, 0] = float("nan")
    seed = next(s for s in range(100) if not mask_by_formula([(0, 0)], 0.5, s).item())
    x.requires_grad_()
    y = TR.dropout(x, 0.5, seed=seed)
    mask = y != 0
    assert y.dtype == dtype and torch.equal(y, torch.where(mask, x * 2, 0.0)) and 0.3 < mask.double().mean() < 0.7
    up = torch.randn(x.shape, dtype=torch.float64).to(dtype)
    assert torch.equal(torch.autograd.grad(y, x, up)[0], torch.where(mask, up * 2, 0.0))
    assert torch.equal(TR.dropout(x.detach().view(21, 33), 0.5, seed=torch.tensor(seed)).view(x.shape), y.detach())
    turned = x.detach().transpose(0, 2)
    assert torch.equal(TR.dropout(turned, 0.5, seed=7).nan_to_num(), TR.dropout(turned.contiguous(), 0.5, seed=7).nan_to_num())
    one = torch.ones(4, 4, dtype=torch.float64, requires_grad=True)
    grad, = torch.autograd.grad(TR.dropout(one, 0.5, seed=1).square().sum(), one, create_graph=True)
    assert torch.autograd.grad(grad.sum(), one)[0].max() == 8.0


def test_dropout_ends():
    x = torch.randn(4, 9)
    assert TR.dropout(x, 0.0, seed=1) is x and TR.dropout(x, 0.7, seed=1, training=False) is x
    assert not TR.dropout(torch.full((4, 9), float("inf")), 1.0, seed=1).any()
    assert torch.equal(TR.dropout(x, 1e-6, seed=1), x)               # less than half a step of 2^-16
    assert TR.dropout(x[:0], 0.5).shape == (0, 9)
    torch.manual_seed(3)
    a = TR.dropout(x, 0.5)
    torch.manual_seed(3)
    assert torch.equal(a, TR.dropout(x, 0.5)) and not torch.equal(a, TR.dropout(x, 0.5))


@pytest.mark.parametrize("kw, error", [(dict(p=1.5), ValueError), (dict(p=float("nan")), ValueError), (dict(seed=-1), ValueError), (dict(seed=2 ** 64), ValueError),
                                       (dict(seed=1.0), ValueError), (dict(seed=torch.tensor(1, dtype=torch.int32)), ValueError),
                                       (dict(seed=torch.tensor([1, 2])), ValueError), (dict(x=torch.ones(3, dtype=torch.int32)), TypeError),
                                       (dict(x=torch.ones(())), ValueError), (dict(x=torch.ones(3, device="meta")), ValueError)])
def test_dropout_refusals(kw, error):
    with pytest.raises(error):
        TR.dropout(**{"x": torch.ones(3, 4), "p": 0.5, **kw})


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, out, rank, adapters", [(1, 1, 1, 1, 0), (5, 9, 7, 3, 0), (17, 20, 33, 4, 3), (6, 8, 8, 8, 9)])
def test_update(n, d, out, rank, adapters, dtype):
    x, base, dy, a, b, scales, ids = update_inputs(n, d, out, rank, adapters, dtype, "cpu", seed=n, bare=0.2)
    want = update_by_formula(x, base, dy, a, b, scales, ids)
    compare(run_update(x, base, dy, a, b, scales, ids), want, ("y", "dx", "da", "db"))
    want = update_by_formula(x, None, dy, a, b, torch.full_like(scales, 0.5), ids)
    got = run_update(x, None, dy, a, b, 0.5, None if ids is None else ids.int())
    compare(got, want, ("y", "dx", "da", "db"))
    if not adapters:
        flat = run_update(x, None, dy, a[0], b[0], 0.5, None)
        assert all(torch.equal(p, q.view(p.shape)) for p, q in zip(flat, got))


@pytest.mark.parametrize("p", [0.3, 1.0])
def test_update_with_dropout_is_dropout_and_update(p):
    x, base, dy, a, b, scales, ids = update_inputs(12, 20, 9, 4, 3, torch.float64, "cpu", bare=0.2)
    got = run_update(x, base, dy, a, b, scales, ids, dropout=p, seed=77)
    x1 = x.detach().requires_grad_()
    a1, b1 = a.detach().requires_grad_(), b.detach().requires_grad_()
    y = TR.low_rank_update(TR.dropout(x1, p, seed=77), a1, b1, base=base, ids=ids, scale=scales)
    two = (y.detach(), *torch.autograd.grad(y, (x1, a1, b1), dy))
    assert all(torch.allclose(g, w, rtol=1e-12, atol=1e-12) for g, w in zip(got, two))


def test_update_gradients_by_differences():
    x, base, dy, a, b, scales, ids = update_inputs(7, 6, 5, 3, 2, torch.float64, "cpu", bare=0.2)
    args = [t.requires_grad_() for t in (x, a, b, base)]
    assert torch.autograd.gradcheck(lambda x, a, b, base: TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales, dropout=0.4, seed=3), args)


def test_update_shapes_and_out():
    x, base, dy, a, b, scales, ids = update_inputs(12, 10, 6, 3, 4, torch.float32, "cpu", bare=0.3)
    y = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales)
    assert torch.equal(y[ids < 0], base[ids < 0])
    assert torch.equal(TR.low_rank_update(x.view(3, 4, 10), a, b, base=base.view(3, 4, 6), ids=ids.view(3, 4), scale=scales), y.view(3, 4, 6))
    one = TR.low_rank_update(x[0], a, b, base=base[0], ids=ids[0], scale=scales)
    assert one.shape == (6,) and torch.allclose(one, y[0])
    none = TR.low_rank_update(x[:0].requires_grad_(), a, b, base=base[:0], ids=ids[:0], scale=scales)
    assert none.shape == (0, 6)
    held = base.clone()
    version = held._version
    assert TR.low_rank_update(x, a, b, base=held, ids=ids, scale=scales, out=held) is held and torch.equal(held, y) and held._version > version


def test_update_refusals():
    x, base, dy, a, b, scales, ids = update_inputs(6, 8, 5, 3, 4, torch.float32, "cpu")
    ok = dict(x=x, a=a, b=b, base=base, ids=ids, scale=scales)
    bad = [dict(x=x[:, :7]), dict(a=a[0]), dict(b=b[:3]), dict(base=base[:, :4]), dict(ids=None), dict(ids=ids[:5]), dict(scale=scales[:2]),
           dict(scale=scales.double()), dict(scale=scales.clone().requires_grad_()), dict(dropout=1.1), dict(dropout=0.5, seed=-4), dict(out=base[:5]),
           dict(out=base.double()), dict(out=base.T.contiguous().T), dict(out=torch.empty(5).expand(6, 5)), dict(x=x[0, 0]),
           dict(a=torch.zeros(4, 129, 8), b=torch.zeros(4, 5, 129)), dict(a=a[:, :0], b=b[:, :, :0]), dict(a=a[:0], b=b[:0], scale=scales[:0]),
           dict(a=torch.zeros(4097, 1, 8), b=torch.zeros(4097, 5, 1), scale=1.0)]
    for change in bad:
        with pytest.raises(ValueError):
            TR.low_rank_update(**{**ok, **change})
    wide = torch.zeros(6, 5)
    for change in (dict(x=x.double()), dict(base=base.half()), dict(ids=ids.float()), dict(x=x.int(), a=a.int(), b=b.int(), base=base.int())):
        with pytest.raises(TypeError):
            TR.low_rank_update(**{**ok, **change})
    with pytest.raises(IndexError):
        TR.low_rank_update(**{**ok, "ids": torch.full_like(ids, 4)})
    with pytest.raises(ValueError, match="without gradients"):
        TR.low_rank_update(**{**ok, "x": x.clone().requires_grad_(), "out": wide})
    block = torch.zeros(6, 8)
    with pytest.raises(ValueError, match="shares memory"):
        TR.low_rank_update(**{**ok, "x": block, "out": block[:, :5]})
    with pytest.raises(ValueError, match="shares memory"):
        TR.low_rank_update(**{**ok, "base": block[:, 1:6], "out": block[:, :5]})
    z = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(TR.low_rank_update(**{**ok, "x": z}).sum(), z, create_graph=True)


def test_bank_and_fused_adapter():
    bank = TR.AdapterBank(12, 7, rank=4, count=3, dtype=torch.float32, device="cpu")
    adapters = [TR.LoraAdapter(12, 7, TR.LoraConfig(rank=r, alpha=6.0), seed=r) for r in (2, 4)]
    for a in adapters:
        torch.nn.init.normal_(a.B)
    bank.set(0, adapters[0])
    bank.set(2, adapters[1])
    x, base, ids = torch.randn(5, 12), torch.randn(5, 7), torch.tensor([0, 2, -1, 1, 0])
    y = bank(x, base, ids)
    for i, e in enumerate(ids.tolist()):
        want = base[i] if e in (-1, 1) else adapters[e // 2](x[i], base[i])
        assert torch.allclose(y[i], want, atol=1e-5)
    bank.clear(0)
    assert torch.equal(bank(x, base, torch.zeros(5, dtype=torch.int64)), base) and bank.nbytes == 4 * (3 * 4 * 19 + 3)
    for call in (lambda: bank.set(3, adapters[0]), lambda: bank.clear(-1)):
        with pytest.raises(IndexError):
            call()
    for r, d in ((5, 12), (2, 11)):
        with pytest.raises(ValueError):
            bank.set(0, TR.LoraAdapter(d, 7, TR.LoraConfig(rank=r)))
    fused = TR.LoraAdapter(12, 7, TR.LoraConfig(rank=4, alpha=6.0, fused=True, dropout=0.5), seed=4)
    fused.load_state_dict(adapters[1].state_dict())
    fused.eval()
    assert torch.allclose(fused(x, base), adapters[1](x, base), atol=1e-5) and torch.allclose(fused.apply_delta(x), adapters[1].apply_delta(x), atol=1e-5)
    fused.train()
    torch.manual_seed(1)
    first = fused(x, base)
    torch.manual_seed(1)
    assert torch.equal(first, fused(x, base)) and not torch.equal(first, fused(x, base))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind, smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("average, reduction", [(False, "mean"), (True, "sum"), (False, "none")])
def test_preference(kind, smoothing, average, reduction, dtype):
    logps, _, ref, mask, _ = loss_inputs(10, 13, dtype, "cpu", seed=2)
    mask[3] = False
    up = torch.rand(5, dtype=torch.float64).to(torch.float64 if dtype == torch.float64 else torch.float32) if reduction == "none" else None
    want = preference_by_formula(logps, ref, mask, 0.3, kind, smoothing, average, reduction, up)
    logps[~mask] = float("nan")
    logps.requires_grad_()
    got = TR.preference_loss(logps, ref, mask, beta=0.3, kind=kind, label_smoothing=smoothing, average=average, reduction=reduction)
    grad, = torch.autograd.grad(got.loss, logps, up)
    compare((*(t.detach() for t in got), grad), want, ("loss", "chosen", "rejected", "gradient"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["tokens", "sequences", "sum", "none"])
@pytest.mark.parametrize("per_token, weight", [(True, 0.1), (False, 0.0)])
def test_policy(reduction, per_token, weight, dtype):
    logps, old, ref, mask, gain = loss_inputs(6, 11, dtype, "cpu", seed=4)
    mask[2] = False
    gain = gain if per_token else gain[:, 0]
    gain[0] = 0.0
    up = torch.rand(6, 11, dtype=torch.float64).to(torch.float64 if dtype == torch.float64 else torch.float32) if reduction == "none" else None
    want = policy_by_formula(logps, old, gain, mask, ref, (0.2, 0.3), weight, reduction, up)
    logps[~mask], old[~mask] = float("nan"), float("inf")
    logps.requires_grad_()
    got = TR.policy_loss(logps, old, gain, mask=mask, ref_logps=ref, clip=(0.2, 0.3), kl_weight=weight, reduction=reduction)
    grad, = torch.autograd.grad(got.loss, logps, up)
    compare((*(t.detach() for t in got), grad), want, ("loss", "kl", "clipped", "gradient"))


def test_policy_by_differences():
    logps, old, ref, mask, gain = loss_inputs(4, 9, torch.float64, "cpu", seed=8)
    near = (torch.exp(logps - old) - 0.8).abs().minimum((torch.exp(logps - old) - 1.3).abs())
    mask &= near > 1e-3
    for reduction in ("tokens", "sequences", "none"):
        assert torch.autograd.gradcheck(lambda l: TR.policy_loss(l, old, gain, mask=mask, ref_logps=ref, clip=(0.2, 0.3), kl_weight=0.1, reduction=reduction).loss,
                                        logps.requires_grad_())
    for kind in TR.tuning_loss.train_ops.PREFERENCE_KINDS:
        assert torch.autograd.gradcheck(lambda l: TR.preference_loss(l, ref, mask, beta=0.4, kind=kind).loss, logps)


def test_policy_on_policy_and_empty():
    logps, _, ref, mask, gain = loss_inputs(3, 5, torch.float64, "cpu")
    logps.requires_grad_()
    r = TR.policy_loss(logps, None, gain, mask=mask)
    assert torch.allclose(torch.autograd.grad(r.loss, logps)[0], torch.where(mask, -gain.double(), 0.0) / mask.sum()) and r.kl == 0 and r.clipped == 0
    r = TR.policy_loss(logps, None, gain, mask=torch.zeros_like(mask), reduction="sequences")
    assert r.loss.isnan() and not torch.autograd.grad(r.loss, logps)[0].any()
    assert TR.policy_loss(logps[:0], None, gain[:0], reduction="none").loss.shape == (0, 5)
    assert TR.policy_loss(logps[:, :0], None, gain[:, 0], reduction="sum").loss == 0
    assert TR.preference_loss(logps[:0], None).loss.isnan()
    assert math.isclose(float(TR.preference_loss(logps[:2, :0].detach(), None).loss), math.log(2), rel_tol=1e-6)


def test_loss_refusals():
    logps, old, ref, mask, gain = loss_inputs(4, 6, torch.float32, "cpu")
    for change in (dict(logps=logps[0]), dict(ref_logps=ref[:, :5]), dict(ref_logps=ref.double()), dict(mask=mask.float()), dict(mask=mask[:2]), dict(kind="other"),
                   dict(beta=0.0), dict(beta=float("inf")), dict(label_smoothing=-0.1), dict(label_smoothing=0.1, kind="ipo"), dict(reduction="tokens"),
                   dict(logps=logps[:3], ref_logps=ref[:3], mask=mask[:3]), dict(ref_logps=ref.clone().requires_grad_())):
        with pytest.raises(ValueError):
            TR.preference_loss(**{**dict(logps=logps, ref_logps=ref, mask=mask), **change})
    with pytest.raises(TypeError):
        TR.preference_loss(logps.int(), ref.int())
    for change in (dict(old_logps=old[:3]), dict(ref_logps=ref.half()), dict(advantages=gain[:, :3]), dict(advantages=gain.int()),
                   dict(advantages=gain.clone().requires_grad_()), dict(old_logps=old.clone().requires_grad_()), dict(clip=(1.5, 0.2)), dict(clip=(0.1, -0.2)),
                   dict(clip=(0.1,)), dict(kl_weight=0.1, ref_logps=None), dict(kl_weight=float("nan")), dict(reduction="mean"), dict(mask=mask.int())):
        with pytest.raises(ValueError):
            TR.policy_loss(**{**dict(logps=logps, old_logps=old, advantages=gain, mask=mask, ref_logps=ref), **change})


def test_operators_beside_a_default_device():
    """What the operators make themselves lies where their inputs do, whatever device a program has made the default."""
    x, base, dy, a, b, scales, ids = update_inputs(9, 12, 10, 3, 2, torch.float32, "cpu", seed=1, bare=0.2)
    one = a[:1].clone(), b[:1].clone()

    def run():
        logps = torch.ones_like(x).requires_grad_()
        loss = TR.policy_loss(logps, None, x[:, 0]).loss
        return [TR.dropout(x, 0.5, seed=3), *run_update(x, base, dy, a, b, scales, ids, dropout=0.5, seed=3), *run_update(x, None, dy, *one, 0.5, None), loss.detach(),
                *torch.autograd.grad(loss, logps)]

    torch.manual_seed(5)
    drawn, want = TR.dropout(x, 0.5), run()
    torch.manual_seed(5)
    with torch.device("meta"):
        again, got = TR.dropout(x, 0.5), run()
    assert torch.equal(drawn, again) and all(torch.equal(g, w) for g, w in zip(got, want))


def test_seeded_dropout_in_a_segment_that_runs_again():
    x, _, _, a, b, scales, _ = update_inputs(6, 16, 12, 4, 0, torch.float64, "cpu", seed=2, bare=0.0)

    def segment(v):
        return TR.dropout(TR.low_rank_update(v, a, b, scale=scales, dropout=0.5, seed=7).tanh(), 0.25, seed=8)

    grads = []
    for run in (segment, lambda v: TR.checkpoint(segment, v)):
        v = x.clone().requires_grad_()
        y = run(v)
        grads.append(torch.autograd.grad(y.square().sum(), v)[0])
    assert grads[0].any() and torch.equal(*grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_preference_margins_that_overflow_an_exponential(dtype):
    x = torch.tensor([[5000.0], [-5000.0], [0.0], [0.0]], dtype=dtype, requires_grad=True)
    for smoothing, loss, slopes in ((0.0, [0.0, 5000.0], [0.0, -1.0]), (0.25, [1250.0, 3750.0], [0.25, -0.75])):
        got = TR.preference_loss(x, None, beta=1.0, label_smoothing=smoothing, reduction="none")
        grad, = torch.autograd.grad(got.loss, x, torch.ones(2, dtype=dtype))
        assert got.loss.tolist() == loss and grad.flatten().tolist() == [*slopes, *(-s for s in slopes)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("weight", [0.0, 0.5])
def test_policy_advantages_of_zero_beside_infinite_ratios(dtype, weight):
    x = torch.tensor([[800.0, 800.0, 800.0, -800.0]], dtype=dtype, requires_grad=True)
    got = TR.policy_loss(x, torch.zeros_like(x), torch.tensor([[0.0, 1.0, -1.0, -1.0]]), ref_logps=x.detach(), kl_weight=weight, reduction="none")
    grad, = torch.autograd.grad(got.loss, x, torch.ones_like(x))
    assert got.loss.tolist() == [[0.0, pytest.approx(-1.2), float("inf"), pytest.approx(0.8)]] and grad.tolist() == [[0.0, 0.0, float("inf"), 0.0]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_hinge_at_its_corner(dtype):
    for margin, slope in ((1.0, 0.0), (1.0 - 2.0 ** -24, -0.5), (1.5, 0.0)):
        x = torch.tensor([[2 * margin], [0.0]], dtype=dtype, requires_grad=True)
        r = TR.preference_loss(x, None, beta=0.5, kind="hinge")
        assert float(r.loss.detach()) == max(0.0, 1.0 - margin) and torch.autograd.grad(r.loss, x)[0].flatten().tolist() == [slope, -slope]
    assert TR.preference_loss(torch.tensor([[float("nan")], [0.0]], dtype=dtype), None, kind="hinge").loss.isnan()


def test_update_leaves_the_sign_of_zeros_in_rows_without_an_adapter():
    x, base, _, a, b, scales, ids = update_inputs(9, 16, 10, 4, 3, torch.float32, "cpu", bare=0.4)
    ids[::2], base[:, ::2] = -1, -0.0
    y = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales)
    assert torch.equal(y[ids < 0].view(torch.int32), base[ids < 0].view(torch.int32))


def test_preference_differences_are_not_rounded():
    logps, ref = torch.full((2, 1025), -1.0), torch.full((2, 1025), -2.0 ** -30)
    logps[:, 0], ref[:, 0] = 1024, 0
    logps[1], ref[1] = 0, 0
    assert float(TR.preference_loss(logps, ref, beta=1.0).chosen_rewards[0]) == 2.0 ** -20


def test_forward_mode():
    """Tangents are right or refused, and those of what has no gradient are refused."""
    import torch.autograd.forward_ad as fw
    x, base, _, a, b, scales, ids = update_inputs(4, 16, 8, 2, 3, torch.float64, "cpu")
    logps, old, ref, mask, gain = loss_inputs(4, 6, torch.float64, "cpu")
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        y = TR.low_rank_update(dual(x), a, b, base=base, ids=ids, scale=scales)
        tangent = TR.low_rank_update(torch.ones_like(x), a, b, ids=ids, scale=scales)
        assert torch.allclose(fw.unpack_dual(y).tangent, tangent)
        for loss in (lambda v: TR.preference_loss(v, ref, mask).loss, lambda v: TR.policy_loss(v, old, gain, mask=mask, ref_logps=ref, kl_weight=0.1).loss):
            v = logps.clone().requires_grad_()
            grad, = torch.autograd.grad(loss(v), v)
            assert torch.allclose(fw.unpack_dual(loss(dual(logps))).tangent, grad.sum())
        with pytest.raises(NotImplementedError):
            TR.dropout(dual(x), 0.5, seed=1)
        for call in (lambda: TR.low_rank_update(x, a, b, ids=ids, scale=dual(scales)), lambda: TR.preference_loss(logps, dual(ref), mask),
                     lambda: TR.policy_loss(logps, dual(old), gain), lambda: TR.policy_loss(logps, old, dual(gain)), lambda: TR.policy_loss(logps, old, gain, ref_logps=dual(ref)),
                     lambda: TR.low_rank_update(x, a, b, ids=ids, scale=scales, out=dual(torch.empty_like(base)))):
            with pytest.raises(ValueError):
                call()


def test_update_out_with_a_history_is_refused():
    x, base, _, a, b, scales, ids = update_inputs(5, 12, 7, 4, 2, torch.float32, "cpu")
    w = torch.ones(5, 7, requires_grad=True)
    for out in (w, w * 2, w[:]):
        with pytest.raises(ValueError):
            TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales, out=out)
    assert torch.equal(w.detach(), torch.ones_like(w))
    want = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales)
    with torch.no_grad():
        assert torch.equal(TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales, out=w), want)


def test_adapter_takes_a_seed():
    config = dict(rank=4, alpha=6.0, dropout=0.5)
    fused, plain = (TR.LoraAdapter(12, 7, TR.LoraConfig(**config, fused=f)).double() for f in (True, False))
    torch.nn.init.normal_(fused.B)
    plain.load_state_dict(fused.state_dict())
    x, base = torch.randn(5, 12, dtype=torch.float64), torch.randn(5, 7, dtype=torch.float64)
    want = TR.low_rank_update(TR.dropout(x, 0.5, seed=9), fused.A, fused.B, base=base, scale=1.5)
    for adapter in (fused, plain):
        registry = TR.LoraRegistry()
        registry.adapters["attn_q"] = adapter
        for seed in (9, torch.tensor(9)):
            assert torch.allclose(adapter(x, base, seed=seed), want) and torch.allclose(base + adapter.apply_delta(x, seed=seed), want)
            assert torch.allclose(registry.apply_adapter("attn_q", x, base, seed=seed), want)
        assert not torch.allclose(adapter(x, base, seed=10), want)
        adapter.eval()
        assert torch.allclose(adapter(x, base, seed=9), adapter(x, base))


@pytest.mark.parametrize("fused", [True, False])
def test_adapter_in_a_segment_that_runs_again(fused):
    """The update is linear in x: the product of x and its gradient is the sum of the results, with the same mask in both passes alone."""
    adapter = TR.LoraAdapter(12, 7, TR.LoraConfig(rank=4, fused=fused, dropout=0.5)).double()
    torch.nn.init.normal_(adapter.B)
    x, base = torch.rand(5, 12, dtype=torch.float64) + 0.5, torch.zeros(5, 7, dtype=torch.float64)

    class Segment(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.adapter = adapter

        def forward(self, t):
            return self.adapter(t, base)

    for run in (*(lambda v, s=s: TR.checkpoint(lambda t: adapter(t, base, seed=s), v) for s in (None, 5, torch.tensor(6))), TR.CheckpointedPipeline([Segment()])):
        v = x.clone().requires_grad_()
        y = run(v)
        drawn = torch.get_rng_state()
        grad, = torch.autograd.grad(y.sum(), v)
        assert torch.equal(drawn, torch.get_rng_state())                  # the second run draws nothing new
        assert abs(float(y.detach().sum() - (grad * x).sum())) <= 1e-9
    with_parameters = TR.CheckpointedPipeline([Segment()])
    v = x.clone().requires_grad_()
    y = with_parameters(v)
    adapter.zero_grad()
    y.sum().backward()
    assert abs(float((adapter.B.grad * adapter.B).sum().detach() - y.detach().sum())) <= 1e-9


@pytest.mark.parametrize("reduction", ["tokens", "sequences", "sum"])
def test_policy_sums_are_float64(reduction):
    """Losses of 2^27, 1 and -2^27: the 1 is lost where they are added in float32.  Gradients are rounded three times, by 2^-24 each."""
    logps = torch.zeros(2, 3, requires_grad=True)
    gain = torch.tensor([[-2.0 ** 27, -1.0, 2.0 ** 27]] * 2)
    loss = TR.policy_loss(logps, None, gain, reduction=reduction).loss
    each = 1.0 if reduction == "sum" else 1 / 6
    assert loss.dtype == torch.float32 and float(loss.detach()) == float(torch.tensor(2 * each, dtype=torch.float32))
    assert torch.allclose(torch.autograd.grad(loss, logps)[0], -gain * each, rtol=2.0 ** -22, atol=0.0)
