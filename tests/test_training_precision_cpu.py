"""The bounds that the head loss's kernels are held to: three bfloat16 parts of a float32 operand keep them, two parts, or parts paired
wrongly, do not; nor does a hidden gradient that is added over pieces of the vocabulary in 16 bits."""
import pytest
import torch
from training_precision import gradient_case, logits_case, loss_and_gradients, parts, pieces_case, plain, product


def three(a, b):
    return product(a, b, 3)


def two(a, b):
    return product(a, b, 2)


def paired_wrongly(a, b):          # the third part of b meets a's second
    x, y = parts(a, 3), parts(b, 3)
    return x[0] @ y[0] + x[0] @ y[1] + x[1] @ y[0] + x[1] @ y[1] + x[1] @ y[2] + x[2] @ y[0]


def outside(got, want, bound):
    return ((got - want).abs() > bound).any()


@pytest.mark.parametrize("n, v, d", [(30, 8, 64), (200, 8, 64), (200, 300, 130)])
def test_bounds_of_the_loss_tell_three_parts_from_two(n, v, d):
    h, w, t, bound = logits_case(n, v, d, "cpu", seed=n)
    want = loss_and_gradients(h, w, t, torch.ones(n), plain)[0]
    assert not outside(loss_and_gradients(h, w, t, torch.ones(n), three)[0], want, bound)
    assert outside(loss_and_gradients(h, w, t, torch.ones(n), two)[0], want, bound)
    assert outside(loss_and_gradients(h, w, t, torch.ones(n), paired_wrongly)[0], want, bound)


@pytest.mark.parametrize("which, n, v, d, live", [("h", 30, 2, 64, 30), ("h", 200, 2, 1001, 150), ("w", 30, 2, 64, 2), ("w", 200, 64, 130, 2)])
def test_bounds_of_the_gradients_tell_three_parts_from_two(which, n, v, d, live):
    h, w, t, up, bound = gradient_case(which, n, v, d, live, "cpu", seed=n)
    i = 1 if which == "h" else 2
    want = loss_and_gradients(h, w, t, up, plain)[i]
    assert not outside(loss_and_gradients(h, w, t, up, three)[i], want, bound)
    assert outside(loss_and_gradients(h, w, t, up, two)[i], want, bound)
    assert outside(loss_and_gradients(h, w, t, up, paired_wrongly)[i], want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_bounds_of_pieces_tell_float32_sums_from_16_bit_ones(dtype):
    v, piece = 2 ** 17, 2 ** 13
    _, w, t, want, bound = pieces_case(40, v, 64, dtype, "cpu", seed=1)
    for kind in (torch.float32, torch.float16, torch.bfloat16):
        total = torch.zeros(40, 64, dtype=kind)
        for c in range(0, v, piece):
            inside = ((t >= c) & (t < c + piece)).float()[:, None]
            total = (total.float() + w[c:c + piece].double().sum(0).float() / v - inside * w[t].float()).to(kind)
        got = total.to(dtype).double()
        assert bool(outside(got, want, bound)) == (kind != torch.float32), kind
