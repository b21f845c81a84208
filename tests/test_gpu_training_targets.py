"""Targets with gaps or repeats in memory, through the kernels."""
import pytest
import torch
from training_operators import loss_inputs

from oxibonsai_b200 import training as TR

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [7, 150])
def test_strided_targets(n, dtype):
    h, w, t = loss_inputs(n, 300, 72, dtype, DEV, seed=70, masked=0.2)
    h.requires_grad_(), w.requires_grad_()

    def run(targets):
        loss = TR.linear_cross_entropy(h, w, targets, reduction="none")
        return (loss.detach(), *torch.autograd.grad(loss.sum(), [h, w]))
    want, same = run(t), run(torch.full_like(t, int(t[0])))
    for targets in (torch.stack([t, (t + 1).clamp_min(0)], 1)[:, 0], t.repeat_interleave(3)[::3], t.int().repeat_interleave(2)[::2], torch.stack([t] * 4, 1).T[1]):
        assert all(torch.equal(a, b) for a, b in zip(run(targets), want))
    assert all(torch.equal(a, b) for a, b in zip(run(t[:1].expand(n)), same))
