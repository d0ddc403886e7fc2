"""The operators of a drafted round at their limits, on the GPU."""

from types import SimpleNamespace

import pytest
import torch

from test_rounds_gpu import attend, batch, kernel_set, kernels, place_both, tiled, within  # noqa: F401  (fixtures among them)

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


# ---- a step's layout --------------------------------------------------------------------------------------------------------

PROMPT = [7, 901, 33]           # three pages of sixteen tokens


@pytest.mark.parametrize("lengths,counts,held", [
    ((48, 0), (1, 3), (0, 0)), ((0, 48), (3, 1), (0, 0)),       # a request without tokens beside one that starts behind the prompt
    ((70, 0), (1, 3), (5, 0)), ((47, 70), (1, 0), (0, 5)),      # the same beside one that holds pages
    ((0, 0), (3, 2), (0, 0)), ((0, 2), (3, 2), (0, 0)), ((5, 0), (1, 60), (0, 0)),      # two that bring the same places
])
def test_nobody_writes_into_a_prompt_that_others_have(kernels, lengths, counts, held):
    assert place_both(kernels, lengths, counts, held, 16, prefix=PROMPT) == -4
    assert place_both(kernels, lengths, counts, held, 16, prefix=PROMPT, rows=[4, 1], table_rows=5) == -4


def test_a_prompt_is_written_where_nobody_has_it_yet(kernels):
    assert place_both(kernels, [0], [60], [0], 16, prefix=PROMPT) == 1
    assert place_both(kernels, [0, 3, 40], [3, 30, 8], [0, 0, 0], 16, prefix=PROMPT) == 0
    assert place_both(kernels, [48, 0, 70], [1, 0, 2], [0, 0, 5], 16, prefix=PROMPT) == 1        # one that brings nothing
    prompt = list(range(50, 175))
    lengths = torch.randperm(2000, generator=torch.Generator().manual_seed(3))[:1500].tolist()
    assert place_both(kernels, lengths, [1] * 1500, [0] * 1500, 16, prefix=prompt) == 0
    lengths[1400] = lengths[3]
    assert place_both(kernels, lengths, [1] * 1500, [0] * 1500, 16, prefix=prompt) == -4
