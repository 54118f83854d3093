"""Plain forms, in 64 bits and one row at a time, of what a beam search needs besides the model."""

from __future__ import annotations

import math

import torch


def attention_row(q, k, v, scale):
    """One query ``[heads, size]`` over keys and values ``[kv heads, tokens, size]``: the result and, per feature, the sum of
    the weighed values' magnitudes (what a rounding of the weights is measured against)."""
    share = q.shape[0] // k.shape[0]
    k, v = k.double().repeat_interleave(share, 0), v.double().repeat_interleave(share, 0)
    weights = torch.softmax(torch.einsum("hd,htd->ht", q.double(), k) * scale, -1)
    return torch.einsum("ht,htd->hd", weights, v), torch.einsum("ht,htd->hd", weights, v.abs())


def beam_select(logits, scores, beams, ended=None, lengths=None, end_token=None, length_penalty=0.0, vocab_limit=None):
    """Dict of lists as ``CudaOps.beam_select`` describes them."""
    groups, in_beams = scores.shape
    limit = vocab_limit or logits.shape[1]
    out = {name: [None] * (groups * beams) for name in ("tokens", "parents", "scores", "ranks", "ended", "lengths")}
    for g in range(groups):
        candidates = []
        for b in range(in_beams):
            r = g * in_beams + b
            x = logits[r, :limit].double().cpu()
            x = torch.where(torch.isnan(x), torch.tensor(-math.inf, dtype=torch.float64), x)
            before = float(scores[g, b])
            made = max(0, int(lengths[r])) if lengths is not None else 0
            if ended is not None and int(ended[r]):
                mine = [(before if j == 0 else -math.inf, end_token, made) for j in range(beams)]
            else:
                top = float(x.max())
                if math.isinf(top):
                    total = math.nan
                else:
                    total = top + math.log(float(torch.exp(x - top).sum()))
                order = sorted(range(limit), key=lambda t: (-float(x[t]), t))[:beams]
                mine = [(before + (float(x[t]) - total), t, made + 1) for t in order]
            for j, (value, t, n) in enumerate(mine):
                value = -math.inf if math.isnan(value) else value
                weighed = value / max(1, n) ** length_penalty if length_penalty else value
                candidates.append((-weighed, b, j, value, t, n))
        chosen = sorted(candidates, key=lambda c: c[:3])[:beams]
        keeps, others = {}, []
        for rank, c in enumerate(chosen):
            if c[1] in keeps:
                others.append(rank)
            else:
                keeps[c[1]] = rank
        for row in range(beams):
            rank = keeps[row] if row in keeps else others.pop(0)
            _, b, _, value, t, n = chosen[rank]
            at = g * beams + row
            out["tokens"][at], out["parents"][at], out["scores"][at], out["ranks"][at] = t, g * beams + b, value, rank
            out["ended"][at] = int(bool((ended is not None and int(ended[g * in_beams + b])) or t == end_token))
            out["lengths"][at] = n
    return out


def beam_reorder(parents, lengths, block_tables, k_pages, v_pages, slots=None, states=()):
    """In place, on host tensors."""
    for r, p in enumerate(parents.tolist()):
        if p == r or not 0 <= p < len(parents) or int(parents[p]) != p:
            continue
        for table, k, v in zip(block_tables, k_pages, v_pages):
            page_tokens = k.shape[-2]
            full, used = divmod(int(lengths[p]), page_tokens)
            table[r, :full] = table[p, :full]
            if used and full < table.shape[1] and int(table[r, full]) >= 0 and int(table[p, full]) >= 0:
                for x in (k, v):
                    if x is not None:
                        x[..., int(table[r, full]), :, :used, :] = x[..., int(table[p, full]), :, :used, :]
        for x in states:
            x[int(slots[r])] = x[int(slots[p])]


def step_tables(pages, page_tokens, ctx_before, q_len, num_tokens, rows=None):
    """Lists: token_request, positions, req_q_start, block tables, cache rows."""
    before, fresh = ctx_before.tolist(), [max(0, n) for n in q_len.tolist()]
    rows = list(range(len(before))) if rows is None else rows.tolist()
    request, positions, start = [], [], []
    for r, (b, n) in enumerate(zip(before, fresh)):
        start.append(len(request))
        request += [r] * n
        positions += range(b, b + n)
    tables, slots = [], []
    for pool, size in zip(pages, page_tokens):
        width = pool.shape[1]
        table = [[int(pool[rows[r], c]) if c * size < before[r] + fresh[r] else -1 for c in range(width)] for r in range(len(rows))]
        slot = []
        for r, p in zip(request, positions):
            page = table[r][p // size] if p // size < width else -1
            slot.append(page * size + p % size if page >= 0 else -1)
        tables.append(table)
        slots.append(slot)
    real = min(len(request), num_tokens)
    pad = num_tokens - real
    return (request[:real] + [0] * pad, positions[:real] + [-1] * pad, start, tables, [s[:real] + [-1] * pad for s in slots])


def search(last_logits, prompt, beams, max_tokens, length_penalty=0.0, end_token=None, vocab_limit=None):
    """Beam search one hypothesis at a time: ``last_logits(tokens)`` gives the logits behind them.  Best first:
    ``(tokens, log probability, ended)``."""
    made = [([], 0.0, False)]
    for _ in range(max_tokens):
        candidates = []
        for ids, score, over in made:
            if over:
                candidates.append((ids, score, True))
                continue
            x = last_logits(list(prompt) + ids).double()
            x = torch.log_softmax(x[: vocab_limit or x.numel()], -1)
            for t in torch.topk(x, min(beams, x.numel())).indices.tolist():
                candidates.append((ids + [t], score + float(x[t]), t == end_token))
        candidates.sort(key=lambda c: -c[1] / len(c[0]) ** length_penalty)
        made = candidates[:beams]
        if all(over for _, _, over in made):
            break
    return made
