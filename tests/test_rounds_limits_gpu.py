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


def within_surroundings(kernels, case):
    """`within` for an output that lies inside a larger buffer, of which nothing else is written."""
    rows, width = case["q"].shape
    room = torch.full(((rows + 2) * width,), 7.0, dtype=case["q"].dtype, device=DEV)
    attend(kernels, case, out=room[width:-width].view(rows, width))
    assert bool((room[:width] == 7.0).all()) and bool((room[-width:] == 7.0).all())
    within(kernels, case, room[width:-width].view(rows, width))


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dim", [16, 80, 128, 160, 176, 192, 256])
def test_heads_of_every_width_stay_in_their_places(kernels, dtype, dim, rows):
    """Widths that the join's lanes divide among them in different ways, few rows (a block a row) and many (a wave a row)."""
    counts = (2, 1, 2) if rows == 5 else (4,) * 75
    case = batch(dtype, 8 if rows == 5 else 16, 2 if rows == 5 else 8, dim, 16, 64, tuple(3 * i % 40 for i in range(len(counts))), counts, seed=71)
    within_surroundings(kernels, case)
