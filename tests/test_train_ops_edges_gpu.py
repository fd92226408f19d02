"""The training operators at the ends of their ranges: calls that their documentation allows or refuses."""
import pytest
import torch

from tests.helpers import rel_l2
from tests.test_train_ops_gpu import TYPES, U, _kept64, _norm64, _rand, _rounded, _within

pytestmark = pytest.mark.gpu


def test_statistics_of_no_pixels_are_zero():
    from spgt_b200 import ops
    for shape in ((2, 0, 12), (0, 5, 12)):
        dirt = [torch.full((128,), float('nan'), device='cuda') for _ in range(64)]     # what the next small allocation holds
        del dirt
        y, stats, _ = ops.group_norm(torch.empty(shape, device='cuda'), 3, None, None)
        assert y.shape == shape and stats.shape == (shape[0], 3, 2) and torch.equal(stats, torch.zeros_like(stats))
