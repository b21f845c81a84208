"""The loss of a head over no tokens at all."""
import pytest
import torch

from oxibonsai_b200 import training as TR


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_no_tokens_give_zero_gradients(reduction, dtype):
    for shape in ((0, 6), (2, 0, 6)):
        h, w = torch.ones(shape, dtype=dtype, requires_grad=True), torch.ones(11, 6, dtype=dtype, requires_grad=True)
        loss = TR.linear_cross_entropy(h, w, torch.zeros(shape[:-1], dtype=torch.int64), reduction=reduction)
        assert loss.shape == (shape[:-1] if reduction == "none" else ()) and loss.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
        dh, dw = torch.autograd.grad(loss.sum(), [h, w])
        assert dh.shape == h.shape and dh.dtype == dw.dtype == dtype
        assert not dw.any() and (reduction != "mean" or loss.isnan())


def test_no_tokens_and_a_head_that_is_not_finite():
    h, w = torch.ones(0, 3, requires_grad=True), torch.full((4, 3), float("nan"), requires_grad=True)
    loss = TR.linear_cross_entropy(h, w, torch.zeros(0, dtype=torch.int64), reduction="sum")
    assert loss == 0
    loss.backward()
    assert not w.grad.any()
