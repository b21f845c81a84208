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
