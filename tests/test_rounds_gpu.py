"""Rounds of drafted tokens over a shared prompt, on the GPU: attention, verification and layout against 64 bits."""

import math

import pytest
import torch

from ampere_kv_engine_amd.kernels.hip import KernelError
from ampere_kv_engine_amd.kernels.hip_rounds import wide_tiles, wide_tiles_fit
from plain import rounds_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def kernel_set():
    from ampere_kv_engine_amd.kernels.hip import HipKernels
    return HipKernels(DEV)


@pytest.fixture(params=[False, True], ids=["narrow", "wide"])
def tiled(kernel_set, request):
    """The kernel set with a prompt's keys for tiles of 32 columns or, where heads and pages allow it, of 256."""
    kernel_set.wide_prefix_tiles = request.param
    yield kernel_set
    kernel_set.wide_prefix_tiles = None


@pytest.fixture
def kernels(kernel_set):
    return kernel_set


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- attention ------------------------------------------------------------------------------------------------------------

def batch(dtype, heads, kv_heads, dim, page, shared, own, counts, seed=0, scale=None, spare=3):
    """Pages in no order; request r brings counts[r] tokens and holds shared + own[r] + counts[r] after the step."""
    generator = torch.Generator().manual_seed(seed)
    lengths = [shared + o + c for o, c in zip(own, counts)]
    shared_pages = shared // page
    total = shared_pages + sum(-(-n // page) - shared_pages for n in lengths) + spare
    order = torch.randperm(total, generator=generator).to(torch.int32)
    width = max(-(-n // page) for n in lengths) + 1
    table = torch.full((len(counts), width), -7, dtype=torch.int32)
    taken = shared_pages
    for r, n in enumerate(lengths):
        table[r, :shared_pages] = order[:shared_pages]
        own_pages = -(-n // page) - shared_pages
        table[r, shared_pages:shared_pages + own_pages] = order[taken:taken + own_pages]
        taken += own_pages
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    normal = lambda *shape: torch.randn(shape, generator=generator)
    case = dict(heads=heads, kv_heads=kv_heads, dim=dim, page=page, shared=shared, lengths=lengths, starts=starts,
                scale=scale or dim ** -0.5, table=table,
                k=normal(total, kv_heads, page, dim).to(dtype), v=normal(total, kv_heads, dim, page).to(dtype),
                q=(2 * normal(starts[-1], heads * dim)).to(dtype))
    return case


def clear_behind(case, value):
    """Puts `value` wherever a page's places lie behind its request's last token."""
    for r, n in enumerate(case["lengths"]):
        if n % case["page"]:
            id = int(case["table"][r, n // case["page"]])
            case["k"][id, :, n % case["page"]:] = value
            case["v"][id, :, :, n % case["page"]:] = value
    free = set(range(case["k"].shape[0])) - set(case["table"].flatten().tolist())
    for id in free:
        case["k"][id], case["v"][id] = value, value


def attend(kernels, case, **changes):
    q = case["q"].to(DEV)
    out = torch.full_like(q, 7.0)
    arguments = dict(q=q, k_pages=case["k"].to(DEV), v_pages=case["v"].to(DEV), block_table=case["table"].to(DEV), q_start=ints(case["starts"]),
                     seq_lens=ints(case["lengths"]), shared=case["shared"], q_heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                     scale=case["scale"], out=out, max_seq_len=max(case["lengths"]),
                     max_new_tokens=max(1, max(b - a for a, b in zip(case["starts"], case["starts"][1:]))))
    arguments.update(changes)
    kernels.attention_shared_prefix(**arguments)
    return arguments["out"]


def within(kernels, case, got, rows=None):
    """Every element within what rounding allows.  A score is a sum of `dim` products in 32 bits: off by (dim + 2) 2^-24 of the sum of
    |q||k|, times the scale; a weight's relative error is that, 2^-22 for its power and as much for its reference point's scaling
    (exponents up to some tens, 2^-24 relative each: 2^-18); sums of n weights in order add n 2^-24, bfloat16 weights in two parts 2^-16.
    Numerator and denominator both carry it; the output's own rounding comes last.
    Tiles of many columns round the prompt's weights once, p' = p (1 + d) with |d| <= u = 2^-8, and divide by the sum of what they
    multiplied: sum p' v / sum p' - out = sum p d (v - out) / sum p', at most u / (1 - u) sum p (|v| + |out|) / sum p."""
    want, weighed, product = rounds_plain.attention(case["q"], case["k"], case["v"], case["table"], case["starts"], case["lengths"],
                                                    case["heads"], case["kv_heads"], case["dim"], case["scale"])
    dtype, dim, most = case["q"].dtype, case["dim"], max(case["lengths"])
    relative = (dim + 2) * 2.0 ** -24 * case["scale"] * product + 2.0 ** -18 + most * 2.0 ** -24
    if dtype == torch.bfloat16:
        relative = relative + 2.0 ** -16
    allowed = 2 * relative * weighed * 1.01 + torch.finfo(dtype).eps / 2 * want.abs() * 1.01
    wide = kernels.wide_prefix_tiles
    if wide is None:
        wide = wide_tiles(len(case["q"]) * case["heads"] // case["kv_heads"], case["kv_heads"], case["shared"], kernels.compute_units)
    if wide and wide_tiles_fit(dim, case["page"], dtype):
        allowed = allowed + 2.0 ** -8 / (1 - 2.0 ** -8) * (weighed + want.abs()) * 1.01
    got = got.double().cpu()
    if rows is not None:
        got, want, allowed = got[rows], want[rows], allowed[rows]
    assert bool((got.isnan() == want.isnan()).all())
    over = ((got - want).abs() - allowed).nan_to_num(nan=-1.0)
    assert float(over.max()) <= 0, f"{float(over.max()):.3g} over what rounding allows, {float((got - want).abs().max()):.3g} off"


SHAPES = [
    # heads, kv_heads, dim, page, shared, own, counts
    (4, 2, 16, 8, 64, (0, 5, 17), (1, 1, 1)),
    (16, 4, 128, 16, 512, (22, 22), (1, 1)),
    (8, 8, 64, 16, 160, (0, 1, 200, 33), (1, 3, 0, 2)),
    (6, 2, 32, 32, 320, (3, 77), (2, 5)),
    (40, 8, 128, 16, 176, (9, 300, 0, 64, 31), (5, 1, 4, 3, 2)),
    (12, 1, 48, 8, 200, (13,), (3,)),
    (10, 2, 80, 64, 128, (100, 7), (4, 1)),
    (6, 3, 96, 16, 0, (0, 40, 130), (1, 2, 1)),          # nothing is shared
    (4, 1, 192, 16, 48, (5, 60), (2, 1)),
    (8, 2, 256, 16, 272, (20, 3, 150), (1, 8, 1)),
    (64, 8, 128, 16, 544, tuple(7 * i for i in range(14)), (5,) * 14),
    (32, 2, 64, 128, 1024, (0, 260, 11), (1, 70, 33)),   # more rows of a request than a tile holds
    (34, 1, 64, 16, 96, (2, 3), (1, 2)),                 # a group wider than a tile
    (16, 4, 128, 16, 1600, tuple(3 + 5 * i for i in range(40)), (1,) * 40),
    (2, 2, 64, 16, 160, (70,), (64,)),                   # the first tile sees nothing of the last segment, the second does
    (16, 2, 256, 16, 128, (9, 40), (5, 6)),
    # several segments of more requests than lanes, some that bring nothing
    (2, 1, 16, 8, 64, tuple(0 if i % 3 else 5 * i for i in range(150)), tuple((2 * i) % 3 for i in range(150))),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"h{s[0]}x{s[1]}d{s[2]}p{s[3]}s{s[4]}r{len(s[5])}")
def test_attention_matches_64_bits(tiled, dtype, shape):
    heads, kv_heads, dim, page, shared, own, counts = shape
    case = batch(dtype, heads, kv_heads, dim, page, shared, own, counts, seed=heads + dim)
    clear_behind(case, math.nan)          # what no token holds is never looked at
    within(tiled, case, attend(tiled, case))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_attention_finds_rows_of_a_persistent_table(tiled, dtype):
    case = batch(dtype, 8, 2, 64, 16, 96, (3, 40, 0), (2, 1, 1), seed=5)
    rows = [4, 0, 2]
    table = torch.full((6, case["table"].shape[1] + 2), -1, dtype=torch.int32)
    for r, row in enumerate(rows):
        table[row, :case["table"].shape[1]] = case["table"][r]
    within(tiled, case, attend(tiled, case, block_table=table.to(DEV), rows=ints(rows), max_seq_len=table.shape[1] * 16, max_new_tokens=9))


def test_attention_leaves_rows_behind_the_last_request(tiled):
    case = batch(torch.bfloat16, 8, 2, 64, 16, 64, (3, 40), (2, 1), seed=6)
    q = torch.cat((case["q"], torch.full((5, 8 * 64), math.nan, dtype=torch.bfloat16)))
    out = attend(tiled, case, q=q.to(DEV), out=torch.full((8, 512), 7.0, dtype=torch.bfloat16, device=DEV))
    within(tiled, case, out[:3])
    assert bool((out[3:] == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite_reach_only_who_sees_them(tiled, dtype, value):
    """A drafted token's value is not finite: the tokens before it, in the same tile, do not see it."""
    case = batch(dtype, 8, 2, 128, 16, 64, (3, 40), (4, 3), seed=7)
    finite = attend(tiled, case)
    position = case["lengths"][0] - 2                      # the third of the first request's four tokens
    id = int(case["table"][0, position // 16])
    case["v"][id, 1, 5, position % 16] = value             # one dim of the second kv head
    got = attend(tiled, case).view(7, 8, 128)
    reached = torch.zeros(7, 8, 128, dtype=torch.bool, device=DEV)
    reached[2:4, 4:, 5] = True
    assert torch.equal(got[~reached], finite.view(7, 8, 128)[~reached])
    assert bool((got[reached].isnan() if math.isnan(value) else got[reached] == value).all())


def test_keys_that_are_not_finite_reach_only_who_sees_them(tiled):
    case = batch(torch.bfloat16, 8, 2, 64, 16, 64, (3, 40), (4, 3), seed=8)
    finite = attend(tiled, case)
    position = case["lengths"][0] - 2
    case["k"][int(case["table"][0, position // 16]), 0, position % 16] = math.nan
    got = attend(tiled, case).view(7, 8, 64)
    reached = torch.zeros(7, 8, 64, dtype=torch.bool, device=DEV)
    reached[2:4, :4] = True
    assert torch.equal(got[~reached], finite.view(7, 8, 64)[~reached])
    assert bool(got[reached].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_scores_far_apart(tiled, dtype):
    """Scores of some hundreds: all but one key of a segment, and all but one segment, underflow."""
    case = batch(dtype, 4, 1, 64, 16, 512, (130, 3), (2, 1), seed=9)
    case["q"] *= 40
    case["k"] *= 4
    within(tiled, case, attend(tiled, case))


def test_what_the_host_cannot_see_is_answered_with_nan(tiled):
    case = batch(torch.bfloat16, 8, 2, 64, 16, 64, (3, 40, 9, 5), (2, 1, 1, 1), seed=10)
    good = attend(tiled, case)
    within(tiled, case, good)
    table = case["table"].clone()
    table[0, 4] = case["k"].shape[0]                        # a page outside the pool: the first request's own
    out = attend(tiled, case, block_table=table.to(DEV))
    assert bool(out[:2].isnan().all()) and torch.equal(out[2:], good[2:])
    table = case["table"].clone()
    table[:, 1] = -1                                        # the same in the prompt
    assert bool(attend(tiled, case, block_table=table.to(DEV)).isnan().all())
    out = attend(tiled, case, max_seq_len=80)             # the second request is longer than that
    assert bool(out[2].isnan().all()) and torch.equal(out[[0, 1, 3, 4]], good[[0, 1, 3, 4]])
    out = attend(tiled, case, rows=ints([0, 1, 4, 3]))      # a row that the table does not have
    assert bool(out[3].isnan().all()) and torch.equal(out[[0, 1, 2, 4]], good[[0, 1, 2, 4]])
    assert bool(attend(tiled, case, rows=ints([-1, 1, 2, 3])).isnan().all())        # the prompt is read from the first
    out = attend(tiled, case, q_start=ints([0, 2, 3, 4, 9]))                        # more tokens than there are
    assert bool(out[4].isnan().all()) and torch.equal(out[:4], good[:4])
    out = attend(tiled, case, max_new_tokens=1)
    assert bool(out[:2].isnan().all()) and torch.equal(out[2:], good[2:])
    out = attend(tiled, case, seq_lens=ints([case["lengths"][0], 64, case["lengths"][2], case["lengths"][3]]))   # within the prompt
    assert bool(out[2].isnan().all()) and torch.equal(out[[0, 1, 3, 4]], good[[0, 1, 3, 4]])


def test_a_request_gives_the_same_whatever_stands_beside_it(tiled):
    """The prompt's product has a column per row of the batch: no column reaches another."""
    case = batch(torch.bfloat16, 8, 2, 128, 16, 640, tuple(range(0, 150, 6)), (1,) * 25, seed=11)
    good = attend(tiled, case)
    case["q"][::2] = math.nan
    out = attend(tiled, case)
    assert torch.equal(out[1::2], good[1::2]) and bool(out[::2].isnan().all())


def test_attention_in_a_pool_of_many_gigabytes(tiled):
    """Pages whose places lie beyond 2^31 elements and 2^32 bytes."""
    case = batch(torch.bfloat16, 16, 4, 128, 16, 512, (20, 300, 5), (2, 1, 3), seed=61)
    pages, far = len(case["k"]), 300_000
    pools = {}
    for name in ("k", "v"):
        pool = torch.empty((far + pages, *case[name].shape[1:]), dtype=torch.bfloat16, device=DEV)
        pool[far:] = case[name].to(DEV)
        pools[name + "_pages"] = pool
    assert pools["k_pages"].numel() > 2 ** 31
    table = torch.where(case["table"] >= 0, case["table"] + far, case["table"])
    near = attend(tiled, case)
    within(tiled, case, near)
    assert torch.equal(attend(tiled, case, block_table=table.to(DEV), **pools), near)


def test_attention_recorded(tiled):
    """A recorded call, replayed over changed queries and lengths with eager calls in between, gives what the eager call does."""
    case = batch(torch.bfloat16, 16, 4, 128, 16, 512, (20, 300, 5), (2, 1, 3), seed=62)
    q, lengths, out = case["q"].to(DEV), ints(case["lengths"]), torch.empty_like(case["q"], device=DEV)
    pages = dict(k_pages=case["k"].to(DEV), v_pages=case["v"].to(DEV), block_table=case["table"].to(DEV), q_start=ints(case["starts"]))
    run = lambda to: attend(tiled, case, q=q, seq_lens=lengths, out=to, **pages)
    run(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tiled.attention_shared_prefix(q, seq_lens=lengths, shared=512, q_heads=16, kv_heads=4, head_dim=128, scale=case["scale"], out=out,
                                      max_seq_len=max(case["lengths"]), max_new_tokens=3, **pages)
    for turn in range(3):
        q.mul_(-0.9)
        lengths.sub_(ints([1, 2, 0]))
        want = run(torch.empty_like(out))
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_attention_agrees_with_the_engines_own(kernels):
    """The same requests through `HipKernels.attention`."""
    from types import SimpleNamespace
    case = batch(torch.bfloat16, 16, 4, 128, 16, 512, (22, 70, 5), (1, 1, 1), seed=12)
    q = case["q"].to(DEV)
    other = torch.empty_like(q)
    ctx = SimpleNamespace(q_start=ints(case["starts"]), seq_lens=ints(case["lengths"]), num_seqs=3, num_decode_seqs=3, host_q_start=case["starts"],
                          host_seq_lens=case["lengths"], max_seq_len=max(case["lengths"]), num_tokens=3)
    meta = SimpleNamespace(block_table=case["table"].to(DEV), width=case["table"].shape[1])
    kernels.attention(q, case["k"].to(DEV), case["v"].to(DEV), ctx, meta, 16, 4, 128, case["scale"], None, other)
    within(kernels, case, attend(kernels, case))
    within(kernels, case, other)


# ---- drafted tokens ---------------------------------------------------------------------------------------------------------

def verify_both(kernels, logits, tokens, starts, temperature, uniforms, draft=None):
    requests, places = uniforms.shape
    kept = torch.full((requests,), 99, dtype=torch.int32, device=DEV)
    chosen = torch.full((requests, places), 99, dtype=torch.int32, device=DEV)
    kernels.verify_drafts(logits.to(DEV), tokens.to(DEV), ints(starts), temperature.to(DEV), uniforms.to(DEV), kept, chosen,
                          draft_logits=draft.to(DEV) if draft is not None else None)
    want = rounds_plain.verify(logits, tokens, starts, temperature, uniforms, draft)
    assert kept.tolist() == want[0]
    assert chosen.tolist() == want[1]
    return kept, chosen


def drafted(vocab, counts, places, with_draft, seed, temperatures=(1.0, 0.7, 0.0), spread=2.5):
    generator = torch.Generator().manual_seed(seed)
    requests = len(counts)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    logits = spread * torch.randn(starts[-1], vocab, generator=generator)
    tokens = torch.randint(0, vocab, (starts[-1],), generator=generator, dtype=torch.int32)
    draft = None
    if with_draft and places > 1:
        draft = torch.randn(requests, places - 1, vocab, generator=generator)
        for r in range(requests):
            for i in range(min(counts[r], places) - 1):
                draft[r, i] = logits[starts[r] + i] + 0.5 * draft[r, i]
                tokens[starts[r] + i + 1] = int(torch.multinomial(torch.softmax(draft[r, i].double(), 0), 1, generator=generator))
    else:
        for r in range(requests):
            for i in range(counts[r] - 1):
                if (r + i) % 4:
                    tokens[starts[r] + i + 1] = int(logits[starts[r] + i].argmax())
    temperature = torch.tensor([temperatures[r % len(temperatures)] for r in range(requests)])
    return logits, tokens, starts, temperature, torch.rand(requests, places, generator=generator), draft


@pytest.mark.parametrize("with_draft", [True, False], ids=["drawn", "looked-up"])
@pytest.mark.parametrize("vocab,counts,places", [(1, (1, 2), 2), (3, (2, 3, 1, 0, 3), 3), (64, (1,), 1), (1000, (4, 1, 2, 3, 4, 0, 4, 4), 4),
                                                 (8192, (2, 2), 2), (8197, (3, 3, 3), 3), (32768, (4, 4, 4), 4), (50001, (8, 1, 5, 7), 8),
                                                 (151936, (5, 5, 2, 5), 5), (700, (20, 33), 33)])
def test_verification_matches_64_bits(kernels, vocab, counts, places, with_draft):
    for seed in range(4):
        verify_both(kernels, *drafted(vocab, counts, places, with_draft, seed))


@pytest.mark.parametrize("with_draft", [True, False], ids=["drawn", "looked-up"])
def test_verification_of_many_small_batches(kernels, with_draft):
    """Every place of the walk and many draws, flat and peaked."""
    for seed in range(30):
        verify_both(kernels, *drafted(517, (5, 3, 4, 5, 5, 1, 5, 2), 5, with_draft, 100 + seed, spread=0.3 if seed % 2 else 6.0))


def test_draft_logits_place_by_place(kernels):
    logits, tokens, starts, temperature, uniforms, draft = drafted(5000, (4, 3, 4), 4, True, 3)
    by_place = draft.transpose(0, 1).contiguous().transpose(0, 1)
    assert not by_place.is_contiguous()
    verify_both(kernels, logits, tokens, starts, temperature, uniforms, by_place)


@pytest.mark.parametrize("vocab", [700, 20000, 20001])
def test_numbers_at_the_ends(kernels, vocab):
    """Random numbers of 0, just below 1 and 1; masked ids of minus infinity at both ends of the vocabulary."""
    logits, tokens, starts, temperature, uniforms, draft = drafted(vocab, (3, 3, 3, 3), 3, True, 4, temperatures=(1.0, 0.3))
    logits[:, :9] = logits[:, -300:] = -math.inf
    draft[:, :, -100:] = -math.inf
    for value in (0.0, 1 - 2.0 ** -24, 1.0):
        for at in range(3):
            numbers = uniforms.clone()
            numbers[:, at] = value
            verify_both(kernels, logits, tokens, starts, temperature, numbers, draft)
            verify_both(kernels, logits, tokens, starts, temperature, numbers)


def test_a_draft_model_that_leaves_nothing(kernels):
    """q = p: every draft is kept; and where one is not kept all the same - a draft of no weight - nothing is left of p, and p is drawn from."""
    logits, tokens, starts, temperature, uniforms, _ = drafted(3000, (3, 3, 3), 3, False, 5, temperatures=(1.0,))
    draft = torch.stack([logits[s:s + 2] for s in starts[:-1]])
    kept, _ = verify_both(kernels, logits, tokens, starts, temperature, uniforms, draft)
    assert kept.tolist() == [2, 2, 2]
    logits[::3, 17] = -math.inf
    draft[:, 0, 17] = -math.inf
    tokens[1::3] = 17
    kept, chosen = verify_both(kernels, logits, tokens, starts, temperature, uniforms, draft)
    assert kept.tolist() == [0, 0, 0] and bool((chosen[:, 0] >= 0).all())


@pytest.mark.parametrize("with_draft", [True, False], ids=["drawn", "looked-up"])
@pytest.mark.parametrize("t", [1e-45, 1e-30, 1e-20, 1e-12, 1e-8, 1e-4, 1e4, 1e20, 1e28])
def test_temperatures_far_from_one(kernels, with_draft, t):
    """Cold rows are all on their largest logits (equal ones share it), warm ones nearly even; in each, minus infinity has no weight."""
    vocab, counts = 9001, (3, 2, 3, 3, 1)
    logits, tokens, starts, temperature, uniforms, draft = drafted(vocab, counts, 3, with_draft, 21)
    temperature = torch.full_like(temperature, t)
    uniforms[:, -1] = torch.tensor([0.0, 0.3137, 0.5171, 0.7, 0.999])
    logits[0, [5, 4100, 9000]] = logits[0].max()                  # one row's largest three times, in several parts
    logits[starts[1]] = torch.finfo(torch.float32).min            # rows of nothing but the lowest value, and masks below it
    logits[starts[1], 100:] = -math.inf
    logits[starts[2], ::2] = -math.inf
    logits[starts[3]] = -math.inf
    logits[starts[3], 4097] = -3.4e38
    if draft is not None:
        draft[1, 0, 7:] = -math.inf
        draft[2, 0] = logits[starts[2]]
    verify_both(kernels, logits, tokens, starts, temperature, uniforms, draft)


def test_ties_go_to_the_lowest_id(kernels):
    logits, tokens, starts, temperature, uniforms, _ = drafted(20000, (3, 3), 3, False, 6, temperatures=(0.0,))
    logits[:, [77, 9000, 19999]] = 50.0
    tokens[1], tokens[2], tokens[4] = 77, 9000, 9000
    kept, chosen = verify_both(kernels, logits, tokens, starts, temperature, uniforms)
    assert kept.tolist() == [1, 0] and chosen.tolist() == [[77, 77, -1], [77, -1, -1]]


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("place", [0, 1, 2])
def test_rows_without_a_next_token(kernels, value, place):
    for t in (1.0, 0.0):
        logits, tokens, starts, temperature, uniforms, draft = drafted(9000, (3, 3), 3, True, 7, temperatures=(t,))
        logits[place, 8500] = value
        verify_both(kernels, logits, tokens, starts, temperature, uniforms, draft)
        logits, tokens, starts, temperature, uniforms, draft = drafted(9000, (3, 3), 3, True, 7, temperatures=(t,))
        draft[0, min(place, 1), 8500] = value
        verify_both(kernels, logits, tokens, starts, temperature, uniforms, draft)
        logits[starts[1] + place] = -math.inf
        verify_both(kernels, logits, tokens, starts, temperature, uniforms, draft)


def test_logits_of_many_gigabytes(kernels):
    """Rows beyond 2^31 logits, and requests that do not begin at the first row."""
    vocab, before = 151936, 14200
    logits, tokens, starts, temperature, uniforms, draft = drafted(vocab, (2, 3), 3, True, 63)
    all_logits = torch.empty((before + len(logits), vocab), device=DEV)
    all_logits[before:] = logits.to(DEV)
    assert before * vocab > 2 ** 31
    all_tokens = torch.cat([torch.zeros(before, dtype=torch.int32), tokens])
    kept, chosen = ints([9, 9]), torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    kernels.verify_drafts(all_logits, all_tokens.to(DEV), ints([s + before for s in starts]), temperature.to(DEV), uniforms.to(DEV), kept, chosen,
                          draft_logits=draft.to(DEV))
    want = rounds_plain.verify(logits, tokens, starts, temperature, uniforms, draft)
    assert kept.tolist() == want[0] and chosen.tolist() == want[1]


def test_drafts_that_are_no_ids(kernels):
    logits, tokens, starts, temperature, uniforms, draft = drafted(600, (3, 3, 3), 3, True, 8)
    tokens[1], tokens[4], tokens[8] = -1, 600, 2 ** 31 - 1
    verify_both(kernels, logits, tokens, starts, temperature, uniforms, draft)
    verify_both(kernels, logits, tokens, starts, temperature, uniforms)


def test_verification_is_distributed_as_the_target(kernels):
    """One draft: the first chosen token's law is the target's.  20,000 requests, 8 ids; the counts' squared differences, over their
    expectations, stay below the 1 - 1e-6 point of chi-squared with 7 degrees (40.5)."""
    generator = torch.Generator().manual_seed(9)
    requests, vocab = 20000, 8
    p, q = torch.randn(vocab, generator=generator), torch.randn(vocab, generator=generator)
    logits = p.expand(2 * requests, vocab).contiguous().to(DEV)
    draft = q.expand(requests, 1, vocab).to(DEV)
    tokens = torch.zeros(2 * requests, dtype=torch.int32)
    tokens[1::2] = torch.multinomial(torch.softmax(q.double(), 0), requests, replacement=True, generator=generator).to(torch.int32)
    uniforms = torch.rand(requests, 2, generator=generator)
    kept = torch.empty(requests, dtype=torch.int32, device=DEV)
    chosen = torch.empty(requests, 2, dtype=torch.int32, device=DEV)
    kernels.verify_drafts(logits, tokens.to(DEV), ints(list(range(0, 2 * requests + 1, 2))), torch.ones(requests, device=DEV), uniforms.to(DEV),
                          kept, chosen, draft_logits=draft)
    counts = torch.bincount(chosen[:, 0].long().cpu(), minlength=vocab).double()
    expected = torch.softmax(p.double(), 0) * requests
    assert float(((counts - expected) ** 2 / expected).sum()) < 40.5


# ---- a step's layout --------------------------------------------------------------------------------------------------------

def place_both(kernels, lengths, counts, held, page, prefix=None, rows=None, table_rows=None, width=None, spare_tokens=0, free=None, cursor=3, seed=0):
    """Runs the call; where it succeeds everything is compared.  Returns (status, outputs, their values before)."""
    generator = torch.Generator().manual_seed(seed)
    requests = len(lengths)
    row_of = rows if rows is not None else list(range(requests))
    table_rows = table_rows or max(row_of, default=0) + 1
    width = width or max([-(-(n + c) // page) for n, c in zip(lengths, counts)] + [len(prefix or ()), 1]) + 2
    table = torch.randint(0, 5000, (table_rows, width), generator=generator, dtype=torch.int32)
    free = free if free is not None else torch.randperm(6000, generator=generator)[:3 + sum(-(-(n + c) // page) for n, c in zip(lengths, counts))].tolist()
    tokens = sum(counts) + spare_tokens
    sizes = dict(q_start=requests + 1, seq_lens=requests, held_after=requests, cursor_after=1, positions=tokens, seq_of_token=tokens, slot_map=tokens, status=1)
    outs = {name: torch.full((n,), -99, dtype=torch.int32, device=DEV) for name, n in sizes.items()}
    on_device = table.to(DEV)
    kernels.place_tokens(ints(lengths), ints(counts), ints(held), ints(free), ints([cursor]), on_device, page, *outs.values(),
                         rows=ints(rows) if rows is not None else None, prefix_pages=ints(prefix) if prefix is not None else None)
    status = int(outs["status"])
    if status < 0:
        assert torch.equal(on_device.cpu(), table)
        assert all(bool((t == -99).all()) for name, t in outs.items() if name != "status")
        return status
    line = table.tolist()
    want = rounds_plain.place(lengths, counts, held, free, cursor, line, page, row_of, prefix)
    for name, values in want.items():
        got = outs[name].tolist()
        assert got[:len(values)] == values, name
        assert all(x == -99 for x in got[len(values):]), name
    assert on_device.tolist() == line
    return status


@pytest.mark.parametrize("page", [1, 8, 16, 24])
def test_layout_of_mixed_requests(kernels, page):
    lengths, counts = [0, 5, 16, 17, 31, 40, 100, 0], [1, 3, 0, 40, 1, 16, 1, 0]
    held = [-(-n // page) for n in lengths]
    held[5] += 2                                            # pages asked for ahead
    assert place_both(kernels, lengths, counts, held, page) >= 0
    assert place_both(kernels, lengths, counts, held, page, rows=[9, 3, 4, 0, 7, 1, 2, 5], table_rows=11, spare_tokens=6) >= 0


def test_layout_of_forked_requests(kernels):
    lengths, counts, held = [48, 70, 48, 48], [5, 2, 1, 0], [0, 5, 0, 0]
    assert place_both(kernels, lengths, counts, held, 16, prefix=[7, 901, 33]) == 2
    assert place_both(kernels, [40, 0], [3, 2], [0, 0], 16, prefix=[7, 901, 33], rows=[2, 0]) == 0


@pytest.mark.parametrize("requests", [1, 63, 256, 257, 600, 4096])
def test_layout_of_many_requests(kernels, requests):
    generator = torch.Generator().manual_seed(requests)
    lengths = torch.randint(0, 90, (requests,), generator=generator).tolist()
    counts = torch.randint(0, 9, (requests,), generator=generator).tolist()
    counts[requests // 2] = 300
    held = [-(-n // 8) for n in lengths]
    rows = torch.randperm(requests + 5, generator=generator)[:requests].tolist()
    assert place_both(kernels, lengths, counts, held, 8, rows=rows, table_rows=requests + 5, free=list(range(10 + requests * 13 + 40))) >= 0


def test_layout_of_long_prompts(kernels):
    assert place_both(kernels, [0] * 7, [1, 20000, 333, 0, 4097, 1, 12000], [0] * 7, 16) >= 0


def test_layouts_that_cannot_be_made(kernels):
    assert place_both(kernels, [16, 16], [1, 1], [1, 1], 16, free=[5, 6, 7, 8]) == -1
    assert place_both(kernels, [16, 16], [1, 1], [1, 1], 16, free=[5, 6, 7, 8], cursor=-1) == -1
    assert place_both(kernels, [16, 16], [1, 1], [1, 1], 16, free=[5, 6, 7, 8], cursor=2) == 2
    assert place_both(kernels, [16, 30], [1, 40], [1, 2], 16, width=4) == -2
    assert place_both(kernels, [16, 30], [1, 4], [1, 2], 16, rows=[0, 5], table_rows=5) == -2
    assert place_both(kernels, [16, 30], [1, 4], [1, 2], 16, rows=[0, -1], table_rows=5) == -2
    assert place_both(kernels, [16, 30, 1], [1, 4, 1], [1, 2, 1], 16, rows=[3, 1, 3], table_rows=5) == -2
    assert place_both(kernels, [16, 30], [1, 4], [1, 2], 16, spare_tokens=-1) == -3
    assert place_both(kernels, [16, -1], [1, 4], [1, 2], 16) == -4
    assert place_both(kernels, [16, 30], [1, 4], [1, -2], 16) == -4
    assert place_both(kernels, [16, 30], [1, 4], [1, 1], 16) == -4            # thirty tokens on one page
    assert place_both(kernels, [16, 2 ** 31 - 1], [1, 4], [1, 2], 16, width=9, free=[1] * 9) == -4


def test_layout_without_requests(kernels):
    assert place_both(kernels, [], [], [], 16) == 0
    assert place_both(kernels, [3], [0], [1], 16) == 0


# ---- a run of them ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("every", [3, 1])
def test_rounds_follow_each_other_on_the_device(kernels, every):
    """(Every `every`-th token is the best one behind the token before it: a draft that a greedy request keeps.)  Three rounds with nothing
    read back in between - place, write keys and values, attend, verify -, eagerly and recorded, against the same on the host."""
    heads, kv_heads, dim, page, vocab, requests, places = 8, 2, 64, 16, 500, 5, 4
    generator = torch.Generator().manual_seed(21)
    shared, pool = 64, 64
    prompt = list(range(4))
    normal = lambda *shape: torch.randn(shape, generator=generator)
    k_pages, v_pages = normal(pool, kv_heads, page, dim), normal(pool, kv_heads, dim, page)
    rounds = [dict(q=2 * normal(requests * places, heads * dim), k=normal(requests * places, kv_heads, dim), v=normal(requests * places, kv_heads, dim),
                   logits=2 * normal(requests * places, vocab), uniforms=torch.rand(requests, places, generator=generator),
                   tokens=torch.randint(0, vocab, (requests * places,), generator=generator, dtype=torch.int32)) for _ in range(3)]
    for one in rounds:
        for n in range(0, requests * places, every):
            one["tokens"][n] = int(one["logits"][max(n - 1, 0)].argmax())
    temperature = torch.tensor([1.0, 0.0, 0.7, 0.0, 1.0])

    state = dict(lengths=ints([shared] * requests), held=ints([0] * requests), cursor=ints([0]), free=ints(list(range(4, pool))),
                 table=torch.full((requests, 12), -1, dtype=torch.int32, device=DEV), prompt=ints(prompt), counts=ints([places] * requests),
                 k=k_pages.to(DEV), v=v_pages.to(DEV))
    at = {name: t.clone() for name, t in state.items()}
    inputs = {name: t.to(DEV) for name, t in rounds[0].items()}
    empty = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)
    made = dict(q_start=empty(requests + 1), seq_lens=empty(requests), held_after=empty(requests), cursor_after=empty(1),
                positions=empty(requests * places), seq_of_token=empty(requests * places), slot_map=empty(requests * places), status=empty(1))
    out, kept, chosen = torch.zeros_like(inputs["q"]), empty(requests), torch.zeros(requests, places, dtype=torch.int32, device=DEV)
    heat = temperature.to(DEV)

    def one_round():
        kernels.place_tokens(at["lengths"], at["counts"], at["held"], at["free"], at["cursor"], at["table"], page, *made.values(), prefix_pages=at["prompt"])
        kernels.kv_write(inputs["k"], inputs["v"], made["slot_map"], at["k"], at["v"])
        kernels.attention_shared_prefix(inputs["q"], at["k"], at["v"], at["table"], made["q_start"], made["seq_lens"], shared, heads, kv_heads, dim,
                                        dim ** -0.5, out, max_seq_len=12 * page, max_new_tokens=places)
        kernels.verify_drafts(inputs["logits"], inputs["tokens"], made["q_start"], heat, inputs["uniforms"], kept, chosen)
        at["lengths"].add_(kept).add_(1)                    # the last token and the kept drafts stay
        at["held"].copy_(made["held_after"])
        at["cursor"].copy_(made["cursor_after"])

    def run(step):
        for name, t in state.items():
            at[name].copy_(t)
        results = []
        for one in rounds:
            for name, t in one.items():
                inputs[name].copy_(t)
            step()
            results.append([t.clone() for t in (out, kept, chosen, made["slot_map"], made["status"])])
        return results

    eager = run(one_round)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        one_round()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one_round()
    for _ in range(2):
        recorded = run(graph.replay)
        for a, b in zip(eager, recorded):
            assert all(torch.equal(x, y) for x, y in zip(a, b))

    # the same on the host
    all_kept = 0
    lengths, held, cursor, table = [shared] * requests, [0] * requests, 0, [[-1] * 12 for _ in range(requests)]
    k, v = k_pages.clone(), v_pages.clone()
    for one, (got, got_kept, got_chosen, got_slots, got_status) in zip(rounds, eager):
        placed = rounds_plain.place(lengths, [places] * requests, held, list(range(4, pool)), cursor, table, page, list(range(requests)), prompt)
        assert got_slots.tolist() == placed["slot_map"] and got_status.tolist() == placed["status"]
        for n, slot in enumerate(placed["slot_map"]):
            k[slot // page, :, slot % page] = one["k"][n]
            v[slot // page, :, :, slot % page] = one["v"][n]
        case = dict(q=one["q"], k=k, v=v, table=torch.tensor(table, dtype=torch.int32), starts=placed["q_start"], lengths=placed["seq_lens"],
                    heads=heads, kv_heads=kv_heads, dim=dim, page=page, shared=shared, scale=dim ** -0.5)
        within(kernels, case, got)
        want = rounds_plain.verify(one["logits"], one["tokens"], placed["q_start"], temperature, one["uniforms"])
        assert got_kept.tolist() == want[0] and got_chosen.tolist() == want[1]
        all_kept += sum(want[0])
        lengths = [n + x + 1 for n, x in zip(lengths, want[0])]
        held, cursor = placed["held_after"], placed["cursor_after"][0]
    assert every == 3 or all_kept >= 2 * 3 * (places - 1)     # (two requests are greedy)


def test_calls_on_two_streams_at_once(kernels):
    """Two batches on two streams, many times over: neither finds the other's sums."""
    cases = [batch(torch.bfloat16, 16, 4, 128, 16, 512, (20, 33, 5), (2, 1, 3), seed=30 + i) for i in range(2)]
    good = [attend(kernels, case) for case in cases]
    drafts = [drafted(30000, (3, 4), 4, True, 40 + i) for i in range(2)]
    want = [rounds_plain.verify(*d) for d in drafts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    arguments = []
    for case, (logits, tokens, starts, temperature, uniforms, draft) in zip(cases, drafts):
        q = case["q"].to(DEV)
        arguments.append((
            dict(q=q, k_pages=case["k"].to(DEV), v_pages=case["v"].to(DEV), block_table=case["table"].to(DEV), q_start=ints(case["starts"]),
                 seq_lens=ints(case["lengths"]), shared=512, q_heads=16, kv_heads=4, head_dim=128, scale=case["scale"], out=torch.empty_like(q),
                 max_seq_len=max(case["lengths"]), max_new_tokens=3),
            dict(logits=logits.to(DEV), tokens=tokens.to(DEV), q_start=ints(starts), temperature=temperature.to(DEV), uniforms=uniforms.to(DEV),
                 kept=ints([9, 9]), chosen=torch.zeros(2, 4, dtype=torch.int32, device=DEV), draft_logits=draft.to(DEV))))
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (attention, verify) in zip(streams, arguments):
            with torch.cuda.stream(stream):
                kernels.attention_shared_prefix(**attention)
                kernels.verify_drafts(**verify)
    torch.cuda.synchronize()
    for (attention, verify), out, (kept, chosen) in zip(arguments, good, want):
        assert torch.equal(attention["out"], out)
        assert verify["kept"].tolist() == kept and verify["chosen"].tolist() == chosen


@pytest.mark.parametrize("first,second", [("lengths", "seq_lens"), ("held", "held_after"), ("cursor", "cursor_after"), ("positions", "slot_map"),
                                          ("free_pages", "status"), ("table", "status")])
def test_layout_refuses_what_shares_memory(kernels, first, second):
    vector = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)
    arguments = dict(lengths=vector(3), counts=vector(3), held=vector(3), free_pages=vector(9), cursor=vector(1), table=vector(12).view(3, 4),
                     page_size=16, q_start=vector(4), seq_lens=vector(3), held_after=vector(3), cursor_after=vector(1), positions=vector(5),
                     seq_of_token=vector(5), slot_map=vector(5), status=vector(1))
    arguments[second] = arguments[first].view(-1)[:len(arguments[second])]
    with pytest.raises(KernelError, match="share memory"):
        kernels.place_tokens(**arguments)


def test_attention_and_verification_refuse_what_shares_memory(kernels):
    case = batch(torch.bfloat16, 8, 2, 64, 16, 64, (3, 40), (2, 1), seed=50)
    q = case["q"].to(DEV)
    with pytest.raises(KernelError, match="out and q share memory"):
        attend(kernels, case, q=q, out=q)
    pages = case["k"].to(DEV)
    with pytest.raises(KernelError, match="out and k_pages share memory"):
        attend(kernels, case, k_pages=pages, out=pages.view(-1)[1024:1024 + 3 * 512].view(3, 512))
    logits, tokens, starts, temperature, uniforms, draft = drafted(100, (3, 2, 3), 3, True, 51)
    tokens, chosen = tokens.to(DEV), torch.zeros(3, 3, dtype=torch.int32, device=DEV)
    arguments = dict(logits=logits.to(DEV), tokens=tokens, q_start=ints(starts), temperature=temperature.to(DEV), uniforms=uniforms.to(DEV),
                     kept=ints([0, 0, 0]), chosen=chosen, draft_logits=draft.to(DEV))
    for changes in (dict(kept=tokens[2:5]), dict(kept=chosen.view(-1)[6:9]), dict(tokens=chosen.view(-1)[:8])):
        with pytest.raises(KernelError, match="share memory"):
            kernels.verify_drafts(**{**arguments, **changes})
