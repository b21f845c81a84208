"""Targets with gaps or repeats in memory: the kernels read them side by side."""
import pytest
import torch

from oxibonsai_b200 import training as TR


@pytest.mark.parametrize("make", [lambda t: torch.stack([t, t + 1], 1)[:, 0], lambda t: t[:1].expand(8), lambda t: t.repeat(2)[::2], lambda t: t.int().repeat(3)[::3],
                                  lambda t: torch.stack([t, t])[0], lambda t: t.int()])
def test_targets_are_handed_on_side_by_side(make, monkeypatch):
    seen = []
    apply = TR.linear_loss._LinearCrossEntropy.apply
    monkeypatch.setattr(TR.linear_loss._LinearCrossEntropy, "apply", lambda *a: (seen.append(a[2]), apply(*a))[1])
    h, w, t = torch.randn(8, 6), torch.randn(11, 6), make(torch.arange(8) % 9)
    loss = TR.linear_cross_entropy(h, w, t, reduction="none")
    assert torch.allclose(loss, torch.nn.functional.cross_entropy(h @ w.T, t.long(), reduction="none"), atol=1e-5)
    assert seen[0].is_contiguous() and seen[0].dtype == torch.int64
