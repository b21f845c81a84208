"""Sizes and overlaps that the training operators refuse, or take, without a GPU."""
import pytest
import torch

from oxibonsai_b200 import training as TR


@pytest.mark.parametrize("rows, vocab, width", [(4, 2 ** 30, 1), (4, 2 ** 31 - 10000, 1), (2 ** 30, 4, 1)])
def test_loss_refuses_sizes_whose_sums_pass_32_bits(rows, vocab, width):
    """The kernels add a piece or a tile of rows to a row's number: sizes end where such a sum may not fit an int any more."""
    h, w = (torch.zeros(1, 1).expand(n, width) for n in (rows, vocab))
    with pytest.raises(ValueError, match="2\\^30"):
        TR.linear_cross_entropy(h, w, torch.zeros(1, dtype=torch.int64).expand(rows))


@pytest.mark.parametrize("kind", [TR.FusedAdam, TR.FusedAdamW])
def test_adam_refuses_fixed_gradients_that_share_memory_with_what_it_writes(kind):
    flat = torch.zeros(64)
    other, m, v = torch.zeros(8), torch.zeros(8), torch.zeros(8)
    for p, g, state in (([flat[:8]], [flat[4:12]], None), ([flat[:8]], [flat[:8]], None), ([other, flat[:8]], [flat[6:14], torch.zeros(8)], None),
                        ([flat[8:16]], [flat[:16][4:12]], None), ([other], [m], ([m], [v])), ([other], [v], ([m], [v]))):
        with pytest.raises(ValueError, match="memory"):
            kind(p, grads=g, state=state)
    kind([flat[:8], flat[16:24]], grads=[flat[8:16], flat[24:32]])
    kind([flat[:8], flat[16:24]], grads=[flat[8:16], flat[8:16]])          # gradients are only read
    kind([flat[:0], flat[:8]], grads=[flat[:0], other])


def test_norm_of_parameters_that_are_listed_twice():
    p, q = torch.ones(4, requires_grad=True), torch.ones(2, requires_grad=True)
    p.grad, tied = torch.full((4,), 3.0), torch.ones(2, 2, requires_grad=True)
    tied.grad = p.grad.view(2, 2)
    assert TR.global_grad_norm([p, q, p]) == pytest.approx(TR.grad_norm([p, q, p])) and TR.global_grad_norm([p, tied]) == pytest.approx(72 ** 0.5)
    assert TR.global_grad_norm([q]) == 0 and TR.global_grad_norm([]).dtype == torch.float32
    with pytest.raises(ValueError, match="memory"):
        TR.clip_global_norm([p, p], 1.0)          # would scale the same values twice
    assert torch.equal(p.grad, torch.full((4,), 3.0))
    for grad, error in ((torch.ones(4).double(), TypeError), (torch.ones(4).to_sparse(), TypeError)):
        z = torch.ones(4, dtype=grad.dtype, requires_grad=True)
        z.grad = grad
        with pytest.raises(error):
            TR.global_grad_norm([z])
