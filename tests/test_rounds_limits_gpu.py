"""The operators of a drafted round at their limits, on the GPU."""

from types import SimpleNamespace

import pytest
import torch

from test_rounds_gpu import attend, batch, kernel_set, kernels, tiled, within  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dim", [64, 128])
def test_weights_in_two_parts_whatever_the_batch(tiled, dim):
    """Within the limits of weights in two parts, also where the prompt's keys would go in wide tiles."""
    case = batch(torch.bfloat16, 16, 2, dim, 16, 1104, tuple(range(0, 90, 6)), (5,) * 15, seed=70)
    got = attend(tiled, case, two_part_weights=True)
    within(SimpleNamespace(wide_prefix_tiles=False), case, got)
