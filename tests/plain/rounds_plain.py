"""Attention over a shared prompt, the verification of drafted tokens and a step's layout in 64 bits, request by request."""

import math

import torch


def attention(q, k_pages, v_pages, table, starts, lengths, q_heads, kv_heads, dim, scale):
    """(out, reach): out [tokens, q_heads * dim] in float64, and for every element the weights' sum of |v| (what relative errors of
    the weights act on) and the largest sum of |q||k| over a row's keys (what rounding of a score acts on)."""
    page = k_pages.shape[2]
    group = q_heads // kv_heads
    q = q.double().view(-1, q_heads, dim)
    out = torch.full_like(q, math.nan)
    weighed, product = torch.zeros_like(out), torch.zeros_like(out)
    for r, length in enumerate(lengths):
        count = starts[r + 1] - starts[r]
        if count == 0:
            continue
        pages = table[r, :-(-length // page)].long()
        if bool(((pages < 0) | (pages >= k_pages.shape[0])).any()):
            continue
        keys = k_pages[pages].double().permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :length]
        values = v_pages[pages].double().permute(1, 0, 3, 2).reshape(kv_heads, -1, dim)[:, :length]
        for i in range(count):
            seen = length - count + i + 1
            row = starts[r] + i
            for h in range(q_heads):
                k, v = keys[h // group, :seen], values[h // group, :seen]
                weights = torch.softmax(k @ q[row, h] * scale, dim=0)
                out[row, h] = weights @ v
                weighed[row, h] = weights @ v.abs()
                product[row, h] = (k.abs() @ q[row, h].abs()).max()
    shape = (q.shape[0], q_heads * dim)
    return out.view(shape), weighed.view(shape), product.view(shape)


def verify(logits, tokens, starts, temperature, uniforms, draft=None):
    """(kept, chosen) as `HipKernels.verify_drafts` has them."""
    vocab = logits.shape[1]
    places = uniforms.shape[1]
    kept, chosen = [], []

    def fine(x, drawn):
        return not bool(x.isnan().any()) and float(x.max()) > -math.inf and not (drawn and float(x.max()) == math.inf)

    for r in range(uniforms.shape[0]):
        first, rows = starts[r], min(starts[r + 1] - starts[r], places)
        t = float(temperature[r])
        drawn = t > 0
        answer, token = [], -1
        for i in range(rows):
            x = logits[first + i].double()
            if not fine(x, drawn):
                break
            p = torch.softmax(x / t, dim=0) if drawn else None
            best = int((x == x.max()).nonzero()[0])
            if i + 1 < rows:
                id = int(tokens[first + i + 1])
                q = None
                if drawn and draft is not None:
                    if not fine(draft[r, i].double(), True):
                        break
                    q = torch.softmax(draft[r, i].double() / t, dim=0)
                real = 0 <= id < vocab
                keep = real and (float(uniforms[r, i]) * (float(q[id]) if q is not None else 1.0) < float(p[id]) if drawn else best == id)
                if keep:
                    answer.append(id)
                    continue
                if drawn:
                    left = p.clone()
                    if q is not None:
                        left = (p - q).clamp(min=0)
                    elif real:
                        left[id] = 0
                    if float(left.sum()) > 0:
                        p = left
            if not drawn:
                token = best
            else:
                upto = p.cumsum(0)
                token = min(int((upto <= float(uniforms[r, -1]) * float(upto[-1])).sum()), int(p.nonzero().max()))
            break
        kept.append(len(answer))
        chosen.append((answer + [token] if rows else []) + [-1] * (places - len(answer) - (1 if rows else 0)))
    return kept, chosen


def place(lengths, counts, held, free, cursor, table, page, rows, prefix):
    """Dict of the outputs of `HipKernels.place_tokens`; `table` (nested lists) is changed in place."""
    out = dict(q_start=[0], seq_lens=[], held_after=[], positions=[], seq_of_token=[], slot_map=[])
    start = cursor
    for r, (length, count, pages) in enumerate(zip(lengths, counts, held)):
        line = table[rows[r]]
        if pages == 0 and prefix:
            line[:len(prefix)] = prefix
            pages = len(prefix)
        while pages * page < length + count:
            line[pages] = free[cursor]
            pages, cursor = pages + 1, cursor + 1
        for position in range(length, length + count):
            out["positions"].append(position)
            out["seq_of_token"].append(r)
            id = line[position // page]
            out["slot_map"].append(id * page + position % page if id >= 0 else -1)
        out["q_start"].append(len(out["positions"]))
        out["seq_lens"].append(length + count)
        out["held_after"].append(pages)
    out["cursor_after"], out["status"] = [cursor], [cursor - start]
    return out
