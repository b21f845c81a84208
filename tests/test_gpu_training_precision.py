"""The head loss's kernels against bounds of the arithmetic itself: float32 operands in three parts, sums over pieces of the vocabulary."""
import pytest
import torch
from training_operators import loss_by_formula, loss_inputs, within
from training_precision import gradient_case, logits_case, loss_and_gradients, pieces_case, plain

from oxibonsai_b200 import training as TR

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def run(h, w, t, up, reduction="none"):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = TR.linear_cross_entropy(h, w, t, reduction=reduction)
    return (loss.detach(), *torch.autograd.grad(loss, [h, w], up))


# up to 24 rows on the CUDA cores, up to 128 with the head's rows across the tile, more with the tokens'; the last two in several pieces of the vocabulary
@pytest.mark.parametrize("n, v, d", [(5, 8, 64), (20, 300, 130), (30, 8, 64), (128, 300, 130), (200, 8, 64), (200, 300, 130), (129, 2000, 1001), (100, 50001, 2048), (200, 50001, 2048)])
def test_float32_losses(n, v, d):
    h, w, t, bound = logits_case(n, v, d, DEV, seed=n + v)
    want = loss_and_gradients(h, w, t, torch.ones(n, device=DEV), plain)[0]
    with torch.no_grad():
        within(TR.linear_cross_entropy(h, w, t, reduction="none"), want, bound, "loss")


@pytest.mark.parametrize("which, n, v, d, live", [("h", 3, 2, 64, 3), ("h", 20, 2, 1001, 11), ("h", 30, 2, 64, 30), ("h", 200, 2, 1001, 150), ("h", 300, 4, 520, 300),
                                                  ("w", 3, 2, 64, 2), ("w", 20, 64, 130, 1), ("w", 30, 2, 64, 2), ("w", 200, 64, 130, 2), ("w", 300, 2048, 72, 3)])
def test_float32_gradients(which, n, v, d, live):
    h, w, t, up, bound = gradient_case(which, n, v, d, live, DEV, seed=n)
    i = 1 if which == "h" else 2
    within(run(h, w, t, up)[i], loss_and_gradients(h, w, t, up, plain)[i], bound, "gradient")


@pytest.mark.parametrize("n", [100, 200])
def test_float32_gradients_over_a_packed_head_in_pieces(n):
    h, w, t = loss_inputs(n, 50001, 2048, torch.float32, DEV, seed=n, masked=0.1)
    up = torch.rand(n, device=DEV)
    want, bound = loss_by_formula(h, w, t, up, reduction="none")
    for got, x, b, what in zip(run(h, w, t, up), want, bound, ("loss", "dh", "dw")):
        within(got, x, b, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_hidden_gradient_over_many_pieces(dtype):
    n, v = 20_000, 2 ** 17                        # at least 10 pieces of the vocabulary
    h, w, t, want, bound = pieces_case(n, v, 64, dtype, DEV, seed=3)
    t[::7] = -100
    live = (t != -100)[:, None]
    within(run(h, w, t, torch.ones((), device=DEV), "sum")[1], torch.where(live, want, 0.0), bound, "dh")
