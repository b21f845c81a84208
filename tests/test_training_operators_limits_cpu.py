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
