"""The operators of a drafted round at their limits, on the GPU."""

import math
from types import SimpleNamespace

import pytest
import torch

from ampere_kv_engine_amd.kernels.hip import KernelError
from test_rounds_gpu import attend, batch, drafted, ints, kernel_set, kernels, place_both, tiled, within  # noqa: F401  (fixtures among them)

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


def put_value(case, request, position, kv_head, dim, value):
    """At one dim of a token's value; position counts from the request's first token, the prompt's among them."""
    page = case["page"]
    case["v"][int(case["table"][request, position // page]), kv_head, dim, position % page] = value


def expect_reached(case, got, finite, reached, values):
    """Elements that see a value that is not finite are that value (or NaN, of two), whatever its weight; the others are as without it."""
    got, finite = got.view_as(reached).float(), finite.view_as(reached).float()
    assert bool((got[~reached].isfinite()).all())
    assert float((got[~reached] - finite[~reached]).abs().max()) <= float(torch.finfo(case["q"].dtype).eps) * float(finite.abs().max())
    want = values[reached]
    assert torch.equal(got[reached].nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("scale", [None, 2.0], ids=["mild", "far"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite_in_places_that_all_see(tiled, dtype, scale, value):
    """In the prompt and among own keys, of a token each and of drafts: everybody who sees the place gets what the formula gives - its
    weight, however small, is no nought.  (`far`: scores some hundred apart, whose weights are less than 32 bits hold.)"""
    heads, kv_heads, dim, shared = 8, 2, 128, 1104
    counts = (1, 3, 1)
    case = batch(dtype, heads, kv_heads, dim, 16, shared, (300, 7, 60), counts, seed=72, scale=scale)
    finite = attend(tiled, case)
    put_value(case, 0, 700, 0, 5, value)                       # of the prompt, seen by all
    put_value(case, 0, shared + 200, 1, 9, value)              # among the first request's own
    put_value(case, 1, shared + 3, 1, 77, value)               # among the second's, seen by its three tokens
    put_value(case, 2, shared + 59, 1, 100, -value)            # of the third's
    put_value(case, 2, 4, 1, 100, value)                       # which the prompt has there too: of both signs is NaN
    case_values = torch.zeros(5, heads, dim, device=DEV)
    reached = torch.zeros(5, heads, dim, dtype=torch.bool, device=DEV)
    for tokens, of_heads, d, v in ((slice(0, 5), slice(0, 4), 5, value), (slice(0, 1), slice(4, 8), 9, value), (slice(1, 4), slice(4, 8), 77, value),
                                   (slice(0, 5), slice(4, 8), 100, value), (slice(4, 5), slice(4, 8), 100, math.nan)):
        reached[tokens, of_heads, d] = True
        case_values[tokens, of_heads, d] = v
    expect_reached(case, attend(tiled, case), finite, reached, case_values)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_values_near_the_largest(tiled, dtype):
    """A segment's first keys of scores far below the others': weights above one times values of 2^100 stay in range."""
    case = batch(dtype, 8, 2, 64, 16, 2048, (20, 40), (2, 1), seed=73)
    case["q"] = torch.ones_like(case["q"])
    case["k"].fill_(0.0)
    case["k"][case["table"][0, 60:].clamp(min=0).long()] = 3.0         # scores of 24, weights of 2^34 beside those of the first keys
    case["v"] *= 2.0 ** 100
    within(tiled, case, attend(tiled, case))


def test_the_prompt_is_found_without_the_first_request(tiled):
    """The first request has ended and its row is cleared, or is none any more: the prompt's pages are given by themselves."""
    case = batch(torch.bfloat16, 8, 2, 64, 16, 1104, (3, 40, 9, 5), (0, 1, 2, 1), seed=74)
    good = attend(tiled, case)
    within(tiled, case, good)
    pages = case["table"][0, :1104 // 16].to(DEV)
    table = case["table"].clone()
    table[0] = -1
    assert bool(attend(tiled, case, block_table=table.to(DEV)).isnan().all())
    for changes in (dict(), dict(rows=ints([-1, 1, 2, 3])), dict(rows=ints([0, 1, 2, 3]), prefix_pages=torch.cat((pages, ints([-5, 7]))))):
        assert torch.equal(attend(tiled, case, **{**dict(block_table=table.to(DEV), prefix_pages=pages), **changes}), good)
    wrong = pages.clone()
    wrong[30] = case["k"].shape[0]
    assert bool(attend(tiled, case, prefix_pages=wrong).isnan().all())
    out = torch.empty(4, 512, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(KernelError, match="out and prefix_pages share memory"):
        attend(tiled, case, prefix_pages=out.view(torch.int32).view(-1)[:69], out=out)


# ---- drafted tokens ---------------------------------------------------------------------------------------------------------

def verified(kernels, logits, tokens, starts, temperature, uniforms, draft):
    requests, places = uniforms.shape
    kept, chosen = ints([99] * requests), torch.full((requests, places), 99, dtype=torch.int32, device=DEV)
    kernels.verify_drafts(logits.to(DEV), tokens.to(DEV), ints(starts), temperature.to(DEV), uniforms.to(DEV), kept, chosen,
                          draft_logits=draft.to(DEV) if draft is not None else None)
    return kept.tolist(), chosen.tolist()


@pytest.mark.parametrize("with_draft", [True, False], ids=["drawn", "looked-up"])
def test_a_temperature_that_is_no_number_has_no_next_token(kernels, with_draft):
    """Nothing is kept and nothing chosen; the requests beside it get what they get."""
    logits, tokens, starts, temperature, uniforms, draft = drafted(5000, (3, 3, 1, 0, 3), 3, with_draft, 80, temperatures=(1.0, 0.0))
    kept, chosen = verified(kernels, logits, tokens, starts, temperature, uniforms, draft)
    temperature[[0, 2, 3]] = math.nan
    now_kept, now_chosen = verified(kernels, logits, tokens, starts, temperature, uniforms, draft)
    for r in range(5):
        if r in (0, 2, 3):
            assert now_kept[r] == 0 and now_chosen[r] == [-1, -1, -1]
        else:
            assert now_kept[r] == kept[r] and now_chosen[r] == chosen[r]


@pytest.mark.parametrize("with_draft", [True, False], ids=["drawn", "looked-up"])
@pytest.mark.parametrize("place", [0, 1, 2])
def test_a_random_number_that_is_none_ends_the_walk(kernels, with_draft, place):
    """The walk ends without a next token at a draft whose number is NaN, and where the token would be drawn with one.  Numbers that
    nobody looks at - of places behind the walk's end, of greedy requests - change nothing."""
    for seed in range(8):
        logits, tokens, starts, temperature, uniforms, draft = drafted(700, (3, 2, 3, 3, 1), 3, with_draft, 90 + seed, temperatures=(1.0, 0.7, 0.0))
        if seed % 2 and not with_draft:                     # (the best token as the draft, and numbers that keep it)
            uniforms[:, :2] = 0.0
        kept, chosen = verified(kernels, logits, tokens, starts, temperature, uniforms, draft)
        numbers = uniforms.clone()
        numbers[:, place] = math.nan
        now_kept, now_chosen = verified(kernels, logits, tokens, starts, temperature, numbers, draft)
        for r, rows in enumerate((3, 2, 3, 3, 1)):
            if float(temperature[r]) == 0 or place < 2 and (place > kept[r] or place >= rows - 1):
                assert now_kept[r] == kept[r] and now_chosen[r] == chosen[r]
            elif place == 2:                                # the number for the token
                assert now_kept[r] == kept[r] and now_chosen[r] == chosen[r][:kept[r]] + [-1] * (3 - kept[r])
            else:                                           # a draft's
                assert now_kept[r] == place and now_chosen[r] == chosen[r][:place] + [-1] * (3 - place)


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
