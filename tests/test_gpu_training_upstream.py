"""Upstream gradients of single tokens that are infinite, or far below the others', and what they do to the other tokens."""
import pytest
import torch
from training_operators import loss_by_formula, loss_inputs, within

from oxibonsai_b200 import training as TR

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gradients(h, w, t, up):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    return torch.autograd.grad(TR.linear_cross_entropy(h, w, t, reduction="none"), [h, w], up)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [9, 300])
def test_infinite_upstream_gradients_stay_with_their_rows(n, dtype):
    h, w, t = loss_inputs(n, 400, 72, dtype, DEV, seed=60)
    t[2] = -100
    up = (torch.rand(n, device=DEV) + 0.1) * (1024.0 if dtype == torch.float16 else 1.0)
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    bad[[0, 4, 7]] = True
    (_, want, _), (_, bound, _) = loss_by_formula(h, w, t, torch.where(bad, 0.0, up), reduction="none")
    up[0], up[2], up[4], up[7] = float("inf"), float("inf"), -float("inf"), float("nan")          # the second is an ignored token's
    dh, dw = gradients(h, w, t, up)
    assert not dh[bad].isfinite().any() and not dw.isfinite().any()
    within(dh[~bad], want[~bad], bound[~bad], "dh")
    # nothing finite above 0 beside it
    up = torch.zeros(n, device=DEV)
    up[4] = float("inf")
    dh, _ = gradients(h, w, t, up)
    assert not dh[4].isfinite().any() and not dh[:4].any() and not dh[5:].any()
    # of an ignored token alone: no gradient at all
    up[2], up[4] = float("inf"), 0.0
    dh, dw = gradients(h, w, t, up)
    assert not dh.any() and not dw.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_upstream_gradients_far_apart(dtype):
    n = 300
    h, w, t = loss_inputs(n, 400, 72, dtype, DEV, seed=61)
    up = 4096.0 * 2.0 ** -torch.linspace(0, 24, n, device=DEV)
    dh, _ = gradients(h, w, t, up)
    (_, want, _), (_, bound, _) = loss_by_formula(h, w, t, up, reduction="none")
    if dtype == torch.float16:          # half a step of dz: 2^-40 of the largest upstream gradient
        bound = bound + 4096.0 * 2.0 ** -40 * w.double().abs().sum(0)
    within(dh, want, bound, "dh")
