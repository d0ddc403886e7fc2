"""The operators of a drafted round at their limits, on the GPU."""

import math
from types import SimpleNamespace

import pytest
import torch

from ampere_kv_engine_amd.kernels.hip import KernelError
from ampere_kv_engine_amd.kernels.hip_rounds import cut_own, cut_prefix
from plain import rounds_plain
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


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,shared,counts", [
    (32, 32, 5200, (1, 2)),             # segments of 12 stages of 64 keys, the last of 9 and a half steps of 32 and 16 keys more
    (64, 64, 4000, (2, 0, 1)),          # 16 stages, the last segment 29 steps
    (64, 64, 4144, (1, 1)),             # 18 stages, the last segment 21 steps and 16 keys
    (128, 128, 2992, (1,)),             # 24 stages, the last segment 45 steps and 16 keys
    (64, 8, 12288, (10, 10, 10, 10)),   # two tiles of 256 columns, the second with 64
], ids=lambda v: str(v).replace(" ", ""))
def test_wide_tiles_go_round_their_rings(kernel_set, dim, heads, kv_heads, shared, counts):
    """Segments long enough that every slot of the rings is filled again, several times."""
    rows = sum(counts) * heads // kv_heads
    segments, keys = cut_prefix(256, rows, kv_heads, shared, kernel_set.compute_units, False)
    assert keys >= 10 * 64 and segments > 1
    case = batch(torch.bfloat16, heads, kv_heads, dim, 16, shared, tuple(5 * i for i in range(len(counts))), counts, seed=75 + dim)
    kernel_set.wide_prefix_tiles = True
    try:
        within(kernel_set, case, attend(kernel_set, case))
    finally:
        kernel_set.wide_prefix_tiles = None


@pytest.mark.parametrize("scale", [None, 1.0], ids=["mild", "far"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,dim,shared,own,counts,bound", [
    (2, 64, 26000, (3, 40), (2, 1), 0),                                   # a block a row: more than a hundred segments of the prompt
    (2, 32, 64, (30000, 9000, 10), (1, 2, 1), 0),                         # the same of own keys
    (32, 16, 320, (30000,) + (70, 3) * 15 + (500,), (2,) * 32, 0),        # a wave a row, 79 segments and the prompt's
    (32, 16, 320, (7, 3) * 16, (2,) * 32, 40000),                         # the same where nobody holds what the bound allows
], ids=["prompt", "own", "own-waves", "bound"])
def test_joins_of_more_segments_than_lanes(kernels, dtype, scale, heads, dim, shared, own, counts, bound):
    case = batch(dtype, heads, 1, dim, 16, shared, own, counts, seed=76, scale=scale)
    changes = {}
    if bound:
        table = torch.full((len(counts), bound // 16), -1, dtype=torch.int32)
        table[:, :case["table"].shape[1]] = case["table"]
        changes = dict(block_table=table.to(DEV), max_seq_len=bound)
    most = (bound or max(case["lengths"])) - shared
    segments = (cut_prefix(32, sum(counts) * heads, 1, shared, kernels.compute_units, dtype == torch.float32)[0]
                + cut_own(len(counts), max(counts) * heads, 1, most, kernels.compute_units)[0])
    assert segments > 64 and (sum(counts) * heads >= 8 * kernels.compute_units) == (heads == 32)
    within(kernels, case, attend(kernels, case, **changes))


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


def place_cleared(kernels, lengths, counts, held, page, tokens, free, cursor=0, prefix=None):
    requests = len(lengths)
    outs = {name: torch.full((n,), -99, dtype=torch.int32, device=DEV) for name, n in dict(
        q_start=requests + 1, seq_lens=requests, held_after=requests, cursor_after=1, positions=tokens, seq_of_token=tokens, slot_map=tokens, status=1).items()}
    table = torch.full((max(requests, 1), 9), -1, dtype=torch.int32, device=DEV)
    kernels.place_tokens(ints(lengths), ints(counts), ints(held), ints(free), ints([cursor]), table, page, *outs.values(),
                         prefix_pages=ints(prefix) if prefix else None, clear_rest=True)
    return {name: t.tolist() for name, t in outs.items()}, table.tolist()


@pytest.mark.parametrize("tokens", [5, 6, 3000])
def test_slots_behind_the_last_token_are_cleared(kernels, tokens):
    outs, _ = place_cleared(kernels, [16, 3], [2, 3], [1, 1], 16, tokens, [8, 9], prefix=None)
    assert outs["status"] == [1] and outs["q_start"] == [0, 2, 5] and outs["slot_map"][:2] == [128, 129]
    assert outs["slot_map"][5:] == [-1] * (tokens - 5) and outs["positions"][5:] == [-99] * (tokens - 5)


@pytest.mark.parametrize("why,changes", [(-1, dict(free=[])), (-1, dict(cursor=5)), (-2, dict(lengths=[16, 200], held=[1, 13])), (-3, dict(tokens=4)),
                                         (-4, dict(lengths=[16, -3])), (-4, dict(lengths=[0, 48], held=[0, 3], prefix=[1, 2, 3]))])
def test_a_step_that_cannot_be_laid_out_brings_nothing(kernels, why, changes):
    arguments = dict(lengths=[16, 3], counts=[2, 3], held=[1, 1], page=16, tokens=2500, free=[8, 9], cursor=0)
    arguments.update(changes)
    outs, table = place_cleared(kernels, **arguments)
    assert outs["status"] == [why] and outs["q_start"] == [0, 0, 0] and outs["slot_map"] == [-1] * arguments["tokens"]
    assert outs["seq_lens"] == arguments["lengths"] and outs["held_after"] == arguments["held"] and outs["cursor_after"] == [arguments["cursor"]]
    assert table == [[-1] * 9] * 2


def test_cleared_layouts_of_nobody(kernels):
    outs, _ = place_cleared(kernels, [], [], [], 16, 4, [8, 9])
    assert outs["status"] == [0] and outs["q_start"] == [0] and outs["slot_map"] == [-1] * 4
    outs, _ = place_cleared(kernels, [], [], [], 16, 4, [8, 9], cursor=3)
    assert outs["status"] == [-1] and outs["q_start"] == [0] and outs["slot_map"] == [-1] * 4 and outs["cursor_after"] == [3]


def test_rounds_of_changing_counts(kernels):
    """Rounds whose counts change and one that brings more than there is room for, nothing read back, eagerly and recorded: the pages hold
    what the host puts there, and the refused round leaves pages, output and lengths alone."""
    heads, kv_heads, dim, page, requests, places, shared, vocab = 4, 2, 64, 16, 4, 4, 32, 300
    generator = torch.Generator().manual_seed(31)
    normal = lambda *shape: torch.randn(shape, generator=generator)
    pool, tokens = 14, requests * places
    pages = normal(pool, kv_heads, page, dim), normal(pool, kv_heads, dim, page)
    counts = [[4, 4, 4, 4], [1, 3, 0, 4], [4, 1, 4, 0], [60, 60, 60, 60], [0, 2, 1, 3], [0, 0, 0, 0], [2, 1, 4, 1]]      # (the fourth has no room)
    rounds = [dict(q=2 * normal(tokens, heads * dim), k=normal(tokens, kv_heads, dim), v=normal(tokens, kv_heads, dim),
                   logits=normal(tokens, vocab), fed=torch.randint(0, vocab, (tokens,), generator=generator, dtype=torch.int32),
                   counts=torch.tensor(c, dtype=torch.int32)) for c in counts]
    start = dict(lengths=ints([shared] * requests), held=ints([0] * requests), cursor=ints([0]), table=torch.full((requests, 8), -1, dtype=torch.int32, device=DEV),
                 k_pages=pages[0].to(DEV), v_pages=pages[1].to(DEV))
    at = {name: t.clone() for name, t in start.items()}
    inputs = {name: t.to(DEV) for name, t in rounds[0].items()}
    free, prompt, heat = ints(list(range(2, pool))), ints([0, 1]), torch.zeros(requests, device=DEV)
    empty = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)
    made = dict(q_start=empty(requests + 1), seq_lens=empty(requests), held_after=empty(requests), cursor_after=empty(1), positions=empty(tokens),
                seq_of_token=empty(tokens), slot_map=empty(tokens), status=empty(1))
    out, kept, chosen = torch.zeros_like(inputs["q"]), empty(requests), torch.zeros(requests, places, dtype=torch.int32, device=DEV)
    numbers = torch.rand(requests, places, generator=generator).to(DEV)

    def one_round():
        kernels.place_tokens(at["lengths"], inputs["counts"], at["held"], free, at["cursor"], at["table"], page, *made.values(), prefix_pages=prompt, clear_rest=True)
        kernels.kv_write(inputs["k"], inputs["v"], made["slot_map"], at["k_pages"], at["v_pages"])
        kernels.attention_shared_prefix(inputs["q"], at["k_pages"], at["v_pages"], at["table"], made["q_start"], made["seq_lens"], shared, heads, kv_heads, dim,
                                        dim ** -0.5, out, max_seq_len=8 * page, max_new_tokens=places, prefix_pages=prompt)
        kernels.verify_drafts(inputs["logits"], inputs["fed"], made["q_start"], heat, numbers, kept, chosen)
        at["lengths"].copy_(made["seq_lens"])
        at["held"].copy_(made["held_after"])
        at["cursor"].copy_(made["cursor_after"])

    def run(step):
        for name, t in start.items():
            at[name].copy_(t)
        for t in (out, kept, chosen):
            t.fill_(7)
        results = []
        for one in rounds:
            for name, t in one.items():
                inputs[name].copy_(t)
            out.fill_(7)
            step()
            results.append({name: t.clone() for name, t in dict(at, out=out, kept=kept, chosen=chosen, **made).items()})
        return results

    eager = run(one_round)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one_round()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one_round()
    for _ in range(2):
        for a, b in zip(eager, run(graph.replay)):
            for name in a:
                if name not in ("positions", "seq_of_token"):      # (behind the last token they are those of earlier rounds)
                    assert torch.equal(a[name], b[name]), name

    lengths, held, cursor, table = [shared] * requests, [0] * requests, 0, [[-1] * 8 for _ in range(requests)]
    k, v = pages[0].clone(), pages[1].clone()
    for number, (one, brings, got) in enumerate(zip(rounds, counts, eager)):
        if number == 3:
            assert int(got["status"]) < 0 and bool((got["out"] == 7).all())
            assert got["kept"].tolist() == [0] * requests and bool((got["chosen"] == -1).all())
        else:
            placed = rounds_plain.place(lengths, brings, held, list(range(2, pool)), cursor, table, page, list(range(requests)), [0, 1])
            lengths, held, cursor = placed["seq_lens"], placed["held_after"], placed["cursor_after"][0]
            for n, slot in enumerate(placed["slot_map"]):
                k[slot // page, :, slot % page] = one["k"][n]
                v[slot // page, :, :, slot % page] = one["v"][n]
            brought = sum(brings)
            assert got["slot_map"].tolist() == placed["slot_map"] + [-1] * (tokens - brought)
            assert bool((got["out"][brought:] == 7).all()) and bool(got["out"][:brought].isfinite().all())
            case = dict(q=one["q"][:brought], k=k, v=v, table=torch.tensor(table, dtype=torch.int32), starts=placed["q_start"], lengths=lengths,
                        heads=heads, kv_heads=kv_heads, dim=dim, page=page, shared=shared, scale=dim ** -0.5)
            if brought:
                within(kernels, case, got["out"][:brought])
        assert torch.equal(got["k_pages"].cpu(), k) and torch.equal(got["v_pages"].cpu(), v)
        assert got["lengths"].tolist() == lengths and got["held"].tolist() == held and got["cursor"].tolist() == [cursor]


def test_slots_that_do_not_fit_are_none(kernels):
    """The last slot of 31 bits, the first behind it, and pages whose slots would come round to others' again."""
    fits = 2 ** 31 // 16 - 1
    outs, _ = place_cleared(kernels, [15, 0, 0, 0], [2, 16, 1, 1], [1, 0, 0, 0], 16, 20, [fits, fits, 2 ** 28, 2 ** 31 - 1])
    assert outs["status"] == [4]
    assert outs["slot_map"] == [-1, 16 * fits] + list(range(16 * fits, 16 * fits + 16)) + [-1, -1]
    assert max(outs["slot_map"]) == 2 ** 31 - 1
