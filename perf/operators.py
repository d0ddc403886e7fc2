"""Rounds of requests that share a prompt and are fed drafted tokens: the three operators such a round is made of besides the
model's products, at the layer sizes that `bench.py` and the tests know.

  place      the step's layout on the device: from the requests' lengths and the number of tokens each brings, the pages they
             take from the pool, their block tables, and the position, request and cache slot of every token.
  attention  every token attends to the prompt that all requests share and to its own request's tokens behind it, both in
             pages of the cache; a request brings its last token and the tokens drafted behind it.
  verify     the drafted tokens against the target's probabilities, from given random numbers: how many are kept, and the
             token that follows them.

A case is one call of one operator over a batch of requests.  Outputs are whole: the attention's rows, the kept tokens, every
table and map.  Lengths follow from the case alone (spread evenly over their logarithm where it says `ragged`); what is in
the caches, the logits, the order of pages and the random numbers from the seed.
"""

from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda:0"


def listed() -> list[dict]:
    bf16, f32 = "bfloat16", "float32"
    return [
        # two answers to one short prompt from a small model: the smallest call, launches and latency
        dict(name="attention small b2", kind="attention", dtype=bf16, heads=16, kv_heads=4, dim=128, page=16, requests=2, shared=512,
             own_tokens=23, drafts=0, ragged=False),
        # eight answers sampled from one long prompt, a token each: the headline's batch and context
        dict(name="attention b8 8192", kind="attention", dtype=bf16, heads=32, kv_heads=8, dim=128, page=16, requests=8, shared=8192,
             own_tokens=256, drafts=0, ragged=False),
        # a full batch over one long document, answers of different lengths
        dict(name="attention b64 32768", kind="attention", dtype=bf16, heads=32, kv_heads=8, dim=128, page=16, requests=64,
             shared=32768, own_tokens=2048, drafts=0, ragged=True),
        # a served batch as it comes: an odd number of requests with no, some or four drafted tokens, another head count
        dict(name="attention b27 drafts", kind="attention", dtype=bf16, heads=40, kv_heads=8, dim=128, page=16, requests=27,
             shared=16000, own_tokens=2000, drafts=4, ragged=True),
        # a full batch with four drafted tokens each: so many queries that the products weigh more than the reads
        dict(name="attention b64 drafts 32b", kind="attention", dtype=bf16, heads=64, kv_heads=8, dim=128, page=16, requests=64,
             shared=8192, own_tokens=512, drafts=4, ragged=False),
        # the 32-bit path, which results are checked with
        dict(name="attention f32 b5", kind="attention", dtype=f32, heads=16, kv_heads=4, dim=128, page=16, requests=5, shared=2000,
             own_tokens=77, drafts=2, ragged=True),
        # one user of a small model, drafts from a small model of its own
        dict(name="verify small b1", kind="verify", requests=1, drafts=3, vocab=32768, draft="model", temperature="0.7", ragged=False),
        # a full batch with four drafted tokens each from a draft model: the logits are what counts
        dict(name="verify b64", kind="verify", requests=64, drafts=4, vocab=151936, draft="model", temperature="1.0", ragged=False),
        # a served batch whose drafts are looked up in the text (no probabilities of their own), greedy and drawn requests together
        dict(name="verify b27 looked up", kind="verify", requests=27, drafts=7, vocab=151936, draft="none", temperature="mixed",
             ragged=True),
        # a decode round: one token for each of a few requests
        dict(name="place b8", kind="place", requests=8, longest=8192, new=1, page=16, shared=0, fresh=0, ragged=False),
        # a full batch with drafted tokens, where every fourth request has just been forked from the shared prompt
        dict(name="place b500 drafts", kind="place", requests=500, longest=4000, new=5, page=16, shared=1600, fresh=4, ragged=True),
        # the prompts of a whole batch fed at once
        dict(name="place prompts", kind="place", requests=64, longest=1, new=16384, page=16, shared=0, fresh=0, ragged=True),
    ]


def _spread(rng, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    """Batches of 1 to 64 requests over prompts of 64 to 32,768 shared tokens with up to 2,048 of their own and up to seven
    drafted ones (32-bit: up to 8 requests, 4,096 shared tokens, the small head count); logits of 1,000 to 151,936 ids for up to
    64 requests; layouts of up to 512 requests and 65,536 new tokens."""
    kind = rng.choice(("attention", "attention", "verify", "place"))
    if kind == "attention":
        dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
        small = dtype == "float32"
        heads, kv_heads, dim = (16, 4, 128) if small else rng.choice(((16, 4, 128), (32, 8, 128), (40, 8, 128), (64, 8, 128), (16, 4, 64)))
        requests, drafts = _spread(rng, 1, 8 if small else 64), rng.choice((0, 0, 1, 2, 4, 7))
        page = rng.choice((16, 16, 32))
        most = 4096 if small else 32768
        # (no more queries times keys, and no more keys in all, than the largest listed cases have)
        most = max(64, min(most, 64 * 32 * 32768 // (requests * (1 + drafts) * heads)))
        held = 512 if small else max(16, min(2048 if drafts < 5 else 512, 20000 // requests))
        return dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests,
                    shared=_spread(rng, 64, most) // page * page, own_tokens=_spread(rng, 8, held), drafts=drafts,
                    ragged=rng.random() < 0.6)
    if kind == "verify":
        drafts = rng.randrange(0, 6)
        return dict(kind=kind, requests=_spread(rng, 1, 64 if drafts < 5 else 50), drafts=drafts,
                    vocab=rng.choice((151936, 32768, _spread(rng, 1000, 151936))), draft=rng.choice(("model", "none")),
                    temperature=rng.choice(("0", "0.7", "1.0", "mixed")), ragged=rng.random() < 0.5)
    requests = _spread(rng, 1, 512)
    shared = rng.choice((0, 0, 1)) * _spread(rng, 16, 2048) // 32 * 32
    return dict(kind=kind, requests=requests, longest=_spread(rng, 1, 16000), new=_spread(rng, 1, 65536 // requests),
                page=rng.choice((16, 16, 32, 8)), shared=shared, fresh=rng.choice((2, 3, 7)) if shared else 0, ragged=rng.random() < 0.6)


# ---- lengths ------------------------------------------------------------------------------------------------------------

def _even(low: int, high: int, count: int) -> list[int]:
    """`count` lengths spread evenly over the logarithm."""
    if count == 1:
        return [high]
    return [int(round(low * (high / low) ** (i / (count - 1)))) for i in range(count)]


def _lengths(case) -> tuple[list[int], list[int]]:
    """(tokens a request holds after the step, tokens it brings) of every request of an attention case, of which the new ones
    and what stands between them and the shared prompt are its own."""
    count, most = case["requests"], 1 + case["drafts"]
    new = [1 + (3 * r + 1) % most if case["ragged"] else most for r in range(count)]
    held = _even(min(4, case["own_tokens"]), case["own_tokens"], count) if case["ragged"] else [case["own_tokens"]] * count
    held = held[1::2] + held[0::2]                  # (long and short ones in no order)
    return [case["shared"] + h + n for h, n in zip(held, new)], new


def _rows(case) -> list[int]:
    """Tokens a request brings in a verify case: the last one and its drafts."""
    return [1 + (5 * r + 2) % (1 + case["drafts"]) if case["ragged"] else 1 + case["drafts"] for r in range(case["requests"])]


def _layout(case) -> tuple[list[int], list[int], list[int]]:
    """(tokens held before, tokens brought, pages held before) of every request of a place case.  Every `fresh`-th request
    holds the shared prompt's tokens and no page yet."""
    count, page = case["requests"], case["page"]
    before = _even(min(7, case["longest"]), case["longest"], count) if case["ragged"] else [case["longest"]] * count
    new = _even(1, case["new"], count) if case["ragged"] else [case["new"]] * count
    before = [case["shared"] + n for n in before[1::2] + before[0::2]]
    held = [-(-n // page) for n in before]
    for r in range(count):
        if case["fresh"] and r % case["fresh"] == 1:
            before[r], held[r] = case["shared"], 0
    return before, new, held


def _starts(counts: list[int]) -> list[int]:
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _int(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


# ---- what a user's program holds ----------------------------------------------------------------------------------------

def prepare(case, seed):
    state = dict(case=case, **{"attention": _attention_inputs, "verify": _verify_inputs, "place": _place_inputs}[case["kind"]](case, seed))
    if own:
        from ampere_kv_engine_amd.kernels.hip import HipKernels
        state["kernels"] = HipKernels(DEVICE)
    return state


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 31)


def _attention_inputs(case, seed):
    """A layer's pages, in no order, as the engine keeps them (keys [page_size, dim], values [dim, page_size]), and the
    step's encoded queries.  A query has a few times a key's size: heads look at some of their keys."""
    generator = _generator(seed)
    dtype, page = getattr(torch, case["dtype"]), case["page"]
    lengths, new = _lengths(case)
    shared_pages = case["shared"] // page
    width = max(-(-n // page) for n in lengths)
    pages = shared_pages + sum(-(-n // page) - shared_pages for n in lengths) + 3
    order = torch.randperm(pages, generator=generator, device=DEVICE).to(torch.int32)
    table = torch.full((case["requests"], width), -1, dtype=torch.int32, device=DEVICE)
    table[:, :shared_pages] = order[:shared_pages]
    taken = shared_pages
    for r, n in enumerate(lengths):
        own_pages = -(-n // page) - shared_pages
        table[r, shared_pages:shared_pages + own_pages] = order[taken:taken + own_pages]
        taken += own_pages
    normal = lambda *shape: torch.randn(shape, generator=generator, dtype=torch.float32, device=DEVICE).to(dtype)
    k_pages = normal(pages, case["kv_heads"], page, case["dim"])
    v_pages = normal(pages, case["kv_heads"], case["dim"], page)
    q = (2.0 * torch.randn(sum(new), case["heads"] * case["dim"], generator=generator, device=DEVICE)).to(dtype)
    return dict(q=q, k_pages=k_pages, v_pages=v_pages, table=table, q_start=_int(_starts(new)), seq_lens=_int(lengths),
                out=torch.empty_like(q))


def _verify_inputs(case, seed):
    """Logits as a step leaves them, float32.  The draft model's are the target's blurred, and it has drawn the tokens; without
    one, the drafts are the target's best token or, every third, another one.  A draft model is run once per drafted place
    for all requests, so its logits lie place by place."""
    generator = _generator(seed)
    requests, drafts, vocab = case["requests"], case["drafts"], case["vocab"]
    rows = _rows(case)
    starts = _starts(rows)
    logits = torch.randn(starts[-1], vocab, generator=generator, device=DEVICE) * 2.5
    temperature = [0.0 if (case["temperature"] == "mixed" and r % 3 == 2) else 0.8 if case["temperature"] == "mixed"
                   else float(case["temperature"]) for r in range(requests)]
    tokens = torch.randint(0, vocab, (starts[-1],), generator=generator, device=DEVICE, dtype=torch.int32)
    draft_logits = None
    if case["draft"] == "model" and drafts:
        by_place = torch.empty(drafts, requests, vocab, device=DEVICE)
        for r in range(requests):
            for i in range(rows[r] - 1):
                by_place[i, r] = logits[starts[r] + i] + 0.6 * torch.randn(vocab, generator=generator, device=DEVICE)
                noise = -torch.log(-torch.log(torch.rand(vocab, generator=generator, device=DEVICE).clamp(1e-20, 1 - 1e-7)))
                tokens[starts[r] + i + 1] = (by_place[i, r] + temperature[r] * noise).argmax()
            by_place[rows[r] - 1:, r] = 0.0                 # (places without a draft: never read)
        draft_logits = by_place.transpose(0, 1)
    elif drafts:
        best = logits.argmax(dim=1).to(torch.int32)
        for r in range(requests):
            for i in range(rows[r] - 1):
                if (r + i) % 3:
                    tokens[starts[r] + i + 1] = best[starts[r] + i]
    uniforms = torch.rand(requests, drafts + 1, generator=generator, device=DEVICE)
    return dict(logits=logits, tokens=tokens, q_start=_int(starts), temperature=torch.tensor(temperature, device=DEVICE),
                uniforms=uniforms, draft_logits=draft_logits, kept=torch.empty(requests, dtype=torch.int32, device=DEVICE),
                chosen=torch.empty(requests, drafts + 1, dtype=torch.int32, device=DEVICE))


def _place_inputs(case, seed):
    """The requests' lengths and tables as they lie on the device, and the pool's free pages in the order in which they are
    handed out."""
    generator = _generator(seed)
    before, new, held = _layout(case)
    page, requests = case["page"], case["requests"]
    shared_pages = case["shared"] // page
    width = max(-(-(b + n) // page) for b, n in zip(before, new)) + 5
    needed = sum(max(0, -(-(b + n) // page) - max(h, shared_pages)) for b, n, h in zip(before, new, held))
    used = shared_pages + sum(max(0, h - shared_pages) for h in held)
    order = torch.randperm(used + needed + 40, generator=generator, device=DEVICE).to(torch.int32)
    table = torch.full((requests + 3, width), -1, dtype=torch.int32, device=DEVICE)
    rows = torch.randperm(requests + 3, generator=generator, device=DEVICE)[:requests].to(torch.int32)
    host_rows, taken = rows.tolist(), shared_pages
    for r in range(requests):
        if held[r]:
            table[host_rows[r], :shared_pages] = order[:shared_pages]
            table[host_rows[r], shared_pages:held[r]] = order[taken:taken + held[r] - shared_pages]
            taken += held[r] - shared_pages
    tokens, empty = sum(new), lambda n: torch.empty(n, dtype=torch.int32, device=DEVICE)
    return dict(lengths=_int(before), counts=_int(new), held=_int(held), free_pages=order[used:].contiguous(), cursor=_int([11]),
                table=table, rows=rows, prefix_pages=order[:shared_pages].contiguous() if shared_pages else None,
                q_start=empty(requests + 1), seq_lens=empty(requests), held_after=empty(requests), cursor_after=empty(1),
                positions=empty(tokens), seq_of_token=empty(tokens), slot_map=empty(tokens), status=empty(1))


def run(state):
    if own:
        return {"attention": _attention_own, "verify": _verify_own, "place": _place_own}[state["case"]["kind"]](state)
    return {"attention": _attention_plain, "verify": _verify_plain, "place": _place_plain}[state["case"]["kind"]](state)


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _attention_own(state):
    case = state["case"]
    state["kernels"].attention_shared_prefix(
        state["q"], state["k_pages"], state["v_pages"], state["table"], state["q_start"], state["seq_lens"], case["shared"],
        case["heads"], case["kv_heads"], case["dim"], case["dim"] ** -0.5, state["out"],
        max_seq_len=state["table"].shape[1] * case["page"], max_new_tokens=1 + case["drafts"])
    return state["out"]


def _verify_own(state):
    state["kernels"].verify_drafts(state["logits"], state["tokens"], state["q_start"], state["temperature"], state["uniforms"],
                                   state["kept"], state["chosen"], draft_logits=state["draft_logits"])
    return [state["kept"], state["chosen"]]


def _place_own(state):
    state["kernels"].place_tokens(
        state["lengths"], state["counts"], state["held"], state["free_pages"], state["cursor"], state["table"],
        state["case"]["page"], state["q_start"], state["seq_lens"], state["held_after"], state["cursor_after"],
        state["positions"], state["seq_of_token"], state["slot_map"], state["status"], rows=state["rows"],
        prefix_pages=state["prefix_pages"])
    return [state[name] for name in PLACED]


PLACED = ("q_start", "seq_lens", "held_after", "cursor_after", "positions", "seq_of_token", "slot_map", "status", "table")


# ---- the same in elementary operations ------------------------------------------------------------------------------------

def _attention_plain(state):
    """The shared keys once for all queries, every request's own ones in a batch padded to the longest; one softmax over both."""
    case = state["case"]
    kv, dim, page, shared = case["kv_heads"], case["dim"], case["page"], case["shared"]
    group, requests = case["heads"] // kv, case["requests"]
    q = state["q"].float().view(-1, kv, group, dim)
    tokens = q.shape[0]
    table = state["table"].long()
    starts, lengths = state["q_start"].long(), state["seq_lens"].long()
    token = torch.arange(tokens, device=DEVICE)
    request = torch.searchsorted(starts, token, right=True) - 1
    position = lengths[request] - starts[request + 1] + token
    of_prefix = table[0, :shared // page]
    keys = state["k_pages"][of_prefix].float().permute(1, 3, 0, 2).reshape(kv, dim, shared)
    values = state["v_pages"][of_prefix].float().permute(1, 0, 3, 2).reshape(kv, shared, dim)
    scale = dim ** -0.5
    flat = q.permute(1, 0, 2, 3).reshape(kv, tokens * group, dim)
    first = torch.bmm(flat, keys.contiguous()).view(kv, tokens, group, shared) * scale
    # every request's own tokens: rows padded to the most tokens a request brings, keys to the longest table row
    own_table = table[:, shared // page:].clamp(min=0)
    span = own_table.shape[1] * page
    own_keys = state["k_pages"][own_table].float().permute(0, 2, 4, 1, 3).reshape(requests * kv, dim, span)
    own_values = state["v_pages"][own_table].float().permute(0, 2, 1, 4, 3).reshape(requests * kv, span, dim)
    most = 1 + case["drafts"]
    place = token - starts[request]
    padded = torch.zeros(requests, kv, most, group, dim, device=DEVICE)
    padded[request, :, place] = q
    second = torch.bmm(padded.view(requests * kv, most * group, dim), own_keys.contiguous()).view(requests, kv, most, group, span) * scale
    second = second[request, :, place].permute(1, 0, 2, 3)              # [kv, tokens, group, span]
    hidden = shared + torch.arange(span, device=DEVICE)[None] > position[:, None]
    second = second.masked_fill(hidden[None, :, None], -math.inf)
    top = torch.maximum(first.amax(-1), second.amax(-1))[..., None]
    first, second = torch.exp(first - top), torch.exp(second - top)
    total = first.sum(-1) + second.sum(-1)
    out = torch.bmm(first.view(kv, tokens * group, shared), values).view(kv, tokens, group, dim)
    weights = torch.zeros(requests, kv, most, group, span, device=DEVICE)
    weights[request, :, place] = second.permute(1, 0, 2, 3)
    seen = torch.arange(span, device=DEVICE)[None] < (lengths - shared)[:, None]
    own_values = own_values.view(requests, kv, span, dim).masked_fill(~seen[:, None, :, None], 0.0).view(requests * kv, span, dim)
    behind = torch.bmm(weights.view(requests * kv, most * group, span), own_values).view(requests, kv, most, group, dim)
    out = (out + behind[request, :, place].permute(1, 0, 2, 3)) / total[..., None]
    return out.permute(1, 0, 2, 3).reshape(tokens, case["heads"] * dim).to(state["q"].dtype)


def _log_weights(logits, temperature):
    """What a row's probabilities are the exponentials of, up to a common factor, in 64 bits (the sums of a row's many small
    probabilities are compared with a random number): 0 at the largest."""
    x = logits.double()
    return (x - x.amax(-1, keepdim=True)) / temperature[:, None].double()


def _verify_plain(state):
    logits, tokens, uniforms, q_logits = state["logits"], state["tokens"].long(), state["uniforms"], state["draft_logits"]
    requests, places = uniforms.shape
    vocab = logits.shape[1]
    starts = state["q_start"].long()
    rows = starts[1:] - starts[:-1]
    everyone = torch.arange(requests, device=DEVICE)
    greedy = state["temperature"] <= 0
    temperature = torch.where(greedy, torch.ones_like(state["temperature"]), state["temperature"])
    alive = torch.ones(requests, dtype=torch.bool, device=DEVICE)
    kept = torch.zeros(requests, dtype=torch.long, device=DEVICE)
    row_request = torch.searchsorted(starts, torch.arange(logits.shape[0], device=DEVICE), right=True) - 1
    weights = torch.exp(_log_weights(logits, temperature[row_request]))
    p = weights / weights.sum(-1, keepdim=True)
    best = logits.argmax(-1)
    for i in range(places - 1):
        row = (starts[:-1] + i).clamp(max=logits.shape[0] - 1)
        drafted = tokens[(row + 1).clamp(max=logits.shape[0] - 1)]
        p_at = p[row, drafted]
        if q_logits is not None:
            w = torch.exp(_log_weights(q_logits[:, i], temperature))
            q_at = w[everyone, drafted] / w.sum(-1)
        else:
            q_at = torch.ones_like(p_at)
        fine = torch.where(greedy, best[row] == drafted, uniforms[:, i].double() * q_at < p_at)
        alive = alive & (i + 1 < rows) & fine
        kept += alive
    last = starts[:-1] + kept
    rejected = kept + 1 < rows
    rest = p[last]
    if places > 1:
        drafted = tokens[(last + 1).clamp(max=logits.shape[0] - 1)]
        place = kept.clamp(max=places - 2)
        if q_logits is not None:
            w = torch.exp(_log_weights(q_logits[everyone, place], temperature))
            q = w / w.sum(-1, keepdim=True)
        else:
            q = torch.zeros_like(rest)
            q[everyone, drafted] = 1.0
        left = torch.where(rejected[:, None], (rest - q).clamp(min=0), rest)
        rest = torch.where((left.sum(-1) > 0)[:, None], left, rest)
    upto = torch.cumsum(rest, dim=-1)
    drawn = (upto <= (uniforms[:, -1].double() * upto[:, -1])[:, None]).sum(-1)
    final = torch.arange(vocab, device=DEVICE).expand(requests, -1).masked_fill(rest <= 0, -1).amax(-1)
    token = torch.where(greedy, best[last], torch.minimum(drawn, final))
    place = torch.arange(places, device=DEVICE)[None]
    drafted = tokens[(starts[:-1, None] + 1 + place).clamp(max=logits.shape[0] - 1)]
    chosen = torch.where(place < kept[:, None], drafted, torch.where(place == kept[:, None], token[:, None], -1))
    return [kept.to(torch.int32), chosen.to(torch.int32)]


def _place_plain(state):
    page, rows, table = state["case"]["page"], state["rows"].long(), state["table"]
    before, new, held = state["lengths"].long(), state["counts"].long(), state["held"].long()
    free, prefix = state["free_pages"], state["prefix_pages"]
    shared = prefix.shape[0] if prefix is not None else 0
    after = before + new
    fresh = held == 0
    had = torch.where(fresh, torch.full_like(held, shared), held)
    has = torch.maximum(had, (after + page - 1) // page)
    upto = torch.cumsum(has - had, 0)
    # every place of every request's row: the page it had, the prompt's for a fresh one, or its share of the free pages
    place = torch.arange(table.shape[1], device=DEVICE)[None]
    number = state["cursor"].long() + (upto - has + had)[:, None] + place - had[:, None]
    line = table[rows]
    if shared:
        line = torch.where(fresh[:, None] & (place < shared), prefix[place.clamp(max=shared - 1)], line)
    taken = (place >= had[:, None]) & (place < has[:, None])
    line = torch.where(taken, free[number.clamp(min=0, max=free.shape[0] - 1)], line)
    table[rows] = line
    starts = torch.cat((torch.zeros(1, dtype=torch.long, device=DEVICE), torch.cumsum(new, 0)))
    token = torch.arange(state["positions"].shape[0], device=DEVICE)
    request = torch.searchsorted(starts, token, right=True) - 1
    position = before[request] + token - starts[request]
    slot = line[request, position // page].long() * page + position % page
    i32 = torch.int32
    return [starts.to(i32), after.to(i32), has.to(i32), (state["cursor"] + upto[-1]).to(i32), position.to(i32), request.to(i32),
            slot.to(i32), upto[-1:].to(i32), table]


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "attention":
        lengths, new = _lengths(case)
        size = 4 if case["dtype"] == "float32" else 2
        keys = case["shared"] + sum(n - case["shared"] for n in lengths)
        seen = sum(sum(n - i for i in range(m)) for n, m in zip(lengths, new))
        return dict(bytes=size * case["dim"] * (2 * keys * case["kv_heads"] + 2 * sum(new) * case["heads"]),
                    flops=4 * case["dim"] * case["heads"] * seen)
    if case["kind"] == "verify":
        rows = _rows(case)
        read = sum(rows) + (sum(rows) - len(rows) if case["draft"] == "model" else 0)
        return dict(bytes=4 * case["vocab"] * read, flops=4 * case["vocab"] * read)
    before, new, held = _layout(case)
    shared = case["shared"] // case["page"]
    pages = sum(max(0, -(-(b + n) // case["page"]) - max(h, shared)) for b, n, h in zip(before, new, held))
    forked = shared * sum(h == 0 for h in held)
    return dict(bytes=4 * (7 * len(new) + 3 * sum(new) + 2 * pages + forked + shared), flops=4 * sum(new))


# ---- the same in 64 bits, request by request ------------------------------------------------------------------------------

def exact(case, seed):
    return {"attention": _attention_exact, "verify": _verify_exact, "place": _place_exact}[case["kind"]](case, seed)


def _attention_exact(case, seed):
    state = _attention_inputs(case, seed)
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // kv
    q = state["q"].double().view(-1, kv, group, dim)
    out = torch.empty_like(q)
    lengths, new = _lengths(case)
    row = 0
    for r, (length, count) in enumerate(zip(lengths, new)):
        pages = state["table"][r, :-(-length // page)].long()
        for h in range(kv):
            keys = state["k_pages"][pages, h].reshape(-1, dim)[:length].double()
            values = state["v_pages"][pages, h].transpose(1, 2).reshape(-1, dim)[:length].double()
            for i in range(count):
                seen = length - count + i + 1
                scores = (keys[:seen] @ q[row + i, h].T) / math.sqrt(dim)
                out[row + i, h] = torch.softmax(scores, dim=0).T @ values[:seen]
        row += count
    return out.view(-1, case["heads"] * dim)


def _verify_exact(case, seed):
    state = _verify_inputs(case, seed)
    tokens, uniforms = state["tokens"].tolist(), state["uniforms"].double().tolist()
    kept, chosen = [], []
    row = 0
    for r, rows in enumerate(_rows(case)):
        t = float(state["temperature"][r])
        answer, rest = [], None
        for i in range(rows):
            x = state["logits"][row + i].double()
            p = None if t == 0 else torch.softmax(x / t, dim=0)
            best = int(x.argmax())
            if i + 1 == rows:
                rest = p
                break
            drafted = tokens[row + i + 1]
            if t == 0:
                if best != drafted:
                    break
            else:
                if state["draft_logits"] is not None:
                    q = torch.softmax(state["draft_logits"][r, i].double() / t, dim=0)
                else:
                    q = torch.nn.functional.one_hot(torch.tensor(drafted, device=DEVICE), x.shape[0]).double()
                if not uniforms[r][i] * float(q[drafted]) < float(p[drafted]):
                    rest = (p - q).clamp(min=0)
                    rest = rest if float(rest.sum()) > 0 else p
                    break
            answer.append(drafted)
        kept.append(len(answer))
        if t == 0:
            answer.append(best)
        else:
            upto = rest.cumsum(0)
            answer.append(min(int((upto <= uniforms[r][-1] * upto[-1]).sum()), int(rest.nonzero().max())))
        chosen.append(answer + [-1] * (uniforms[r].__len__() - len(answer)))
        row += rows
    return [_int(kept), _int(chosen)]


def _place_exact(case, seed):
    state = _place_inputs(case, seed)
    page, table = case["page"], state["table"].cpu().numpy().copy()
    free, rows = state["free_pages"].tolist(), state["rows"].tolist()
    prefix = state["prefix_pages"].tolist() if state["prefix_pages"] is not None else []
    cursor = int(state["cursor"])
    begin, starts, after, has, positions, owners, slots = cursor, [0], [], [], [], [], []
    for r, (length, count, pages) in enumerate(zip(*_layout(case))):
        if pages == 0:
            table[rows[r], :len(prefix)] = prefix
            pages = len(prefix)
        while pages * page < length + count:
            table[rows[r], pages] = free[cursor]
            pages, cursor = pages + 1, cursor + 1
        for position in range(length, length + count):
            positions.append(position)
            owners.append(r)
            slots.append(int(table[rows[r], position // page]) * page + position % page)
        starts.append(len(positions))
        after.append(length + count)
        has.append(pages)
    return [_int(x) for x in (starts, after, has, [cursor], positions, owners, slots, [cursor - begin])] + [torch.from_numpy(table).to(DEVICE)]
