"""What a beam search on the GPU is measured on, operator by operator.

Several continuations of one prompt (the beams of a search, the samples of one request) share the prompt's pages.  A step
of such a batch needs four things besides the model: attention that reads the shared keys and values once, the choice of
the next beams from the logits, the beams' caches moved to the rows that go on, and the block tables and slot maps of
the next step.  All four stay on the device, so that a step needs no answer from the host.

* ``attention``: ``CudaOps.paged_attention_shared``, single query tokens over the paged cache; groups of rows read their
  common first tokens once;
* ``select``: ``CudaOps.beam_select``, the best ``beams`` of ``in_beams * vocab`` continuations of every prompt; a beam
  that goes on stays in its row;
* ``reorder``: ``CudaOps.beam_reorder``, the rows that do not go on take over their parents' block tables, the tokens in
  the parents' last pages and the parents' fixed states;
* ``tables``: ``CudaOps.step_tables``, block tables, positions and slot maps from the requests' lengths.

With ``own`` false every operator runs in a plain form (elementary torch operations, 32 bits, rounded once at the end;
64 bits where the order of candidates hangs on the numbers).  Sizes are those of the 50M decoder (8 layers, 8 heads of
64, 50,304 ids), GPT-2 small (12 heads, 50,257 ids), grouped heads of 128, and generic ones.
"""

from __future__ import annotations

import math
import random

import torch

own = False
DEVICE = "cuda:0"


# ---- cases ----------------------------------------------------------------------------------------
def listed():
    return [
        # the smallest calls: a few continuations of a short prompt, where a launch is what counts
        dict(name="attention 1x4, 37 tokens, 8 heads of 64", op="attention", dtype="bfloat16", groups=1, beams=4, n_head=8,
             n_kv_head=8, head_dim=64, page=16, prefix=37, suffix=5),
        # an ordinary search: eight prompts of about a thousand tokens, eight beams each
        dict(name="attention 8x8, 1,021 tokens, 8 heads of 64", op="attention", dtype="bfloat16", groups=8, beams=8, n_head=8,
             n_kv_head=8, head_dim=64, page=16, prefix=1021, suffix=67),
        # the 32-bit mode, in which results are compared
        dict(name="attention 2x5, 509 tokens, 12 heads of 64, fp32", op="attention", dtype="float32", groups=2, beams=5,
             n_head=12, n_kv_head=12, head_dim=64, page=16, prefix=509, suffix=33),
        # many samples of one long prompt, grouped heads
        dict(name="attention 1x256, 16,384 tokens, 32/8 heads of 128", op="attention", dtype="bfloat16", groups=1, beams=256,
             n_head=32, n_kv_head=8, head_dim=128, page=64, prefix=16384, suffix=128),
        # the first choice after a prompt: one row of logits becomes four beams
        dict(name="select 1 row -> 4 beams of 50,304 ids", op="select", groups=1, in_beams=1, beams=4, vocab=50304, limit=50257,
             penalty=0.0, ends=False),
        # a step of eight searches, some beams of which have ended, with a length penalty
        dict(name="select 8x8 beams of 50,304 ids, ended ones", op="select", groups=8, in_beams=8, beams=8, vocab=50304,
             limit=50257, penalty=0.6, ends=True),
        # the largest: rows that start off the 16-byte boundaries
        dict(name="select 64x16 beams of 50,257 ids", op="select", groups=64, in_beams=16, beams=16, vocab=50257, limit=0,
             penalty=1.0, ends=True),
        # one search with the 50M decoder's cache
        dict(name="reorder 1x4 beams, 8 layers", op="reorder", dtype="bfloat16", groups=1, beams=4, layers=8, n_kv_head=8,
             head_dim=64, v_dim=64, page=16, prompt=37, made=22, states=0, state_words=0),
        # eight searches of eight beams with the 50M decoder's cache
        dict(name="reorder 8x8 beams, 8 layers", op="reorder", dtype="bfloat16", groups=8, beams=8, layers=8, n_kv_head=8,
             head_dim=64, v_dim=64, page=16, prompt=1021, made=71, states=0, state_words=0),
        # many searches with a model whose layers keep pages or a matrix memory (8 heads of 64 x 128 and an odd tail)
        dict(name="reorder 48x8 beams, 2 layers of pages and 4 of states", op="reorder", dtype="bfloat16", groups=48, beams=8,
             layers=2, n_kv_head=4, head_dim=128, v_dim=64, page=64, prompt=300, made=45, states=4, state_words=65545),
        # a step of one search
        dict(name="tables 4 rows", op="tables", requests=4, new=1, context=60, page=16, page2=0, spare=0),
        # a batch of prompts' portions and single tokens over two groups of layers with pages of their own size
        dict(name="tables 256 requests, 8,192 tokens, two groups", op="tables", requests=256, new=64, context=16000, page=16,
             page2=64, spare=77),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random):
    op = rng.choice(["attention", "attention", "select", "reorder", "tables"])
    if op == "attention":
        n_head, n_kv_head, head_dim = rng.choice([(8, 8, 64), (12, 12, 64), (16, 4, 64), (32, 8, 128), (25, 25, 64), (8, 2, 32)])
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        return dict(op=op, dtype=dtype, groups=_spread(rng, 1, 12), beams=_spread(rng, 1, 32), n_head=n_head,
                    n_kv_head=n_kv_head, head_dim=head_dim, page=rng.choice([8, 16, 32, 64]),
                    prefix=_spread(rng, 1, 1500 if dtype == "float32" else 6000), suffix=_spread(rng, 1, 120))
    if op == "select":
        beams = _spread(rng, 1, 16)
        vocab = _spread(rng, 40, 50304)
        return dict(op=op, groups=_spread(rng, 1, 60), in_beams=rng.choice([1, beams, beams]), beams=beams, vocab=vocab,
                    limit=rng.choice([0, max(beams, vocab - 7)]), penalty=rng.choice([0.0, 0.7, 1.0]), ends=rng.random() < 0.6)
    if op == "reorder":
        states = rng.choice([0, 1, 3])
        return dict(op=op, dtype=rng.choice(["bfloat16", "float32"]), groups=_spread(rng, 1, 24), beams=_spread(rng, 1, 16),
                    layers=rng.randint(1, 8), n_kv_head=rng.choice([1, 2, 8]), head_dim=rng.choice([24, 64, 128]),
                    v_dim=rng.choice([16, 64]), page=rng.choice([4, 16, 32]), prompt=_spread(rng, 1, 900),
                    made=_spread(rng, 1, 90), states=states, state_words=_spread(rng, 1, 30000) if states else 0)
    return dict(op=op, requests=_spread(rng, 1, 256), new=_spread(rng, 1, 64), context=_spread(rng, 1, 16000),
                page=rng.choice([1, 16, 32]), page2=rng.choice([0, 64]), spare=rng.choice([0, 13]))


# ---- inputs ---------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(77000 + seed)


def _rng(case, seed):
    """For what differs from seed to seed; the lengths of a case are those of seed "sizes"."""
    return random.Random(f"{seed} {sorted((k, v) for k, v in case.items() if k != 'name')}")


def _lengths(case):
    """The prompts' lengths, from three quarters of the case's longest to the longest, and the tokens that every row of their
    groups has made (attention: each row its own number; reorder: the rows of a group as many)."""
    rng, G, B = _rng(case, "sizes"), case["groups"], case["beams"]
    longest, made = (case["prefix"], case["suffix"]) if case["op"] == "attention" else (case["prompt"], case["made"])
    prompts = [max(1, round(longest * (1 - 0.25 * rng.random() * (g > 0)))) for g in range(G)]
    each = [rng.randint(max(1, made // 2), made) for _ in range(G * B)]
    if case["op"] == "reorder":
        each = [each[r // B * B] for r in range(G * B)]
    return prompts, each


def _requests(case):
    """Tokens that the requests bring, and those that they have in the cache already."""
    rng, R = _rng(case, "sizes"), case["requests"]
    new = [1 if rng.random() < 0.5 else rng.randint(1, case["new"]) for _ in range(R)]
    if R > 2 and case["new"] > 1:
        new[rng.randrange(R)] = 0                         # a row of the batch that holds no request
    return new, [_spread(rng, 1, case["context"]) - 1 for _ in range(R)]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    state = {"attention": _prepare_attention, "select": _prepare_select, "reorder": _prepare_reorder,
             "tables": _prepare_tables}[case["op"]](case, seed)
    if own:
        from mini_gpt_inference_b200.kernels.ops import default_ops

        state["ops"] = default_ops(DEVICE)
    return state


def _beam_pages(rng, prompts, rows_of, lengths, page):
    """Block tables of rows that share their prompt's full pages and hold pages of their own behind them (the prompt's
    part-filled last page is every row's own), in a pool whose pages lie in no order.  Returns (tables, pages)."""
    width = -(-max(lengths) // page)
    count, columns = 0, []
    for g, prompt in enumerate(prompts):
        columns.append(list(range(count, count + prompt // page)))
        count += prompt // page
    tables = []
    for r, g in enumerate(rows_of):
        shared, total = columns[g], -(-lengths[r] // page)
        tables.append(shared + list(range(count, count + total - len(shared))))
        count += total - len(shared)
    order = list(range(count + 3))                        # three pages that nobody has
    rng.shuffle(order)
    return [[order[p] for p in t] + [-1] * (width - len(t)) for t in tables], count + 3


def _prepare_attention(case, seed):
    rng, gen = _rng(case, seed), _gen(seed)
    dtype = getattr(torch, case["dtype"])
    G, B, H, KV, D, page = (case[k] for k in ("groups", "beams", "n_head", "n_kv_head", "head_dim", "page"))
    prompts, behind = _lengths(case)
    rows_of = [g for g in range(G) for _ in range(B)]
    lengths = [prompts[g] + n for g, n in zip(rows_of, behind)]
    tables, pages = _beam_pages(rng, prompts, rows_of, lengths, page)
    table = _i32(tables)
    k = torch.randn((pages, KV, page, D), generator=gen, device=DEVICE).to(dtype)
    v = torch.randn((pages, KV, page, D), generator=gen, device=DEVICE).to(dtype)
    for g, prompt in enumerate(prompts):                  # every row's copy of the prompt's part-filled last page
        column, used = prompt // page, prompt % page
        if used:
            first = tables[g * B][column]
            for r in range(g * B + 1, (g + 1) * B):
                k[tables[r][column], :, :used] = k[first, :, :used]
                v[tables[r][column], :, :used] = v[first, :, :used]
    qkv = torch.randn((G * B, (H + 2 * KV) * D), generator=gen, device=DEVICE)
    qkv[:, : H * D] *= 2.0                                # scores of this spread: some keys count, most do not
    state = dict(case=case, qkv=qkv.to(dtype), k=k, v=v, table=table, positions=_i32([n - 1 for n in lengths]),
                 requests=_i32(list(range(G * B))), prompts=prompts, lengths=lengths,
                 groups=_i32([[g * B, B, prompts[g]] for g in range(G)]))
    if own:
        from types import SimpleNamespace

        from mini_gpt_inference_b200.cache.storage import PagedKVView
        from mini_gpt_inference_b200.parts.context import SharedPrefix

        state["cache"] = PagedKVView(k, v, 0, page, None, False)
        state["ctx"] = SimpleNamespace(
            block_tables=[table], token_request=state["requests"], positions=state["positions"], decode_only=True,
            max_ctx_after=max(lengths), max_q_len=1, extra={},
            shared_prefix=SharedPrefix(state["groups"], max_rows=B, max_tokens=max(prompts), max_behind=case["suffix"]))
    return state


def _prepare_select(case, seed):
    rng, gen = _rng(case, seed), _gen(seed)
    G, I = case["groups"], case["in_beams"]
    rows = G * I
    # logits of this spread: a few hundred ids hold most of the probability
    logits = torch.randn((rows, case["vocab"]), generator=gen, device=DEVICE) * 2.5
    spare = torch.rand((rows, 3), generator=gen, device=DEVICE)
    made = rng.randint(1, 40)
    scores = -2.0 * made * (0.5 + spare[:, 0]).reshape(G, I)
    ended = (spare[:, 1] < 0.25).to(torch.int32) if case["ends"] else None
    lengths = None
    if case["ends"] or case["penalty"]:
        lengths = (made - (spare[:, 2] * made * 0.5).to(torch.int32) * (ended if ended is not None else 0)).to(torch.int32)
    return dict(case=case, logits=logits, scores=scores, ended=ended, lengths=lengths,
                end=min(case["vocab"], case["limit"] or case["vocab"]) - 1 if case["ends"] else None)


def _keeping_parents(rng, groups, beams):
    """Parents (row numbers) as a choice leaves them: a row that goes on stays where it is, the others take one of those over."""
    parents = []
    for g in range(groups):
        going_on = sorted(rng.sample(range(beams), max(1, round(beams * rng.uniform(0.4, 0.8)))))
        parents += [g * beams + (b if b in going_on else rng.choice(going_on)) for b in range(beams)]
    return parents


def _prepare_reorder(case, seed):
    rng, gen = _rng(case, seed), _gen(seed)
    dtype = getattr(torch, case["dtype"])
    G, B, L, page = (case[k] for k in ("groups", "beams", "layers", "page"))
    prompts, made = _lengths(case)
    rows_of = [g for g in range(G) for _ in range(B)]
    lengths = [prompts[g] + n for g, n in zip(rows_of, made)]
    tables, pages = _beam_pages(rng, prompts, rows_of, [n + 1 for n in lengths], page)
    k = torch.randn((L, pages, case["n_kv_head"], page, case["head_dim"]), generator=gen, device=DEVICE).to(dtype)
    v = torch.randn((L, pages, case["n_kv_head"], page, case["v_dim"]), generator=gen, device=DEVICE).to(dtype)
    slots = rng.sample(range(G * B + 5), G * B)
    states = [torch.randn((G * B + 5, case["state_words"]), generator=gen, device=DEVICE) for _ in range(case["states"])]
    return dict(case=case, parents=_i32(_keeping_parents(_rng(case, seed), G, B)), lengths=_i32(lengths), table=_i32(tables), k=k, v=v,
                slots=_i32(slots), states=states)


def _prepare_tables(case, seed):
    rng = _rng(case, seed)
    R = case["requests"]
    new, before = _requests(case)
    sizes = [case["page"]] + ([case["page2"]] if case["page2"] else [])
    rows = rng.sample(range(R + 3), R)
    pools = []
    for size in sizes:
        width = -(-max(b + n for b, n in zip(before, new)) // size)
        count = [0] * (R + 3)
        for r, b, n in zip(rows, before, new):
            count[r] = -(-(b + n) // size)
        pages = torch.randperm(sum(count) + 1, generator=torch.Generator().manual_seed(seed))
        pool, at = torch.full((R + 3, width), -1, dtype=torch.int32), 0
        for r in range(R + 3):
            pool[r, : count[r]] = pages[at: at + count[r]]
            at += count[r]
        pools.append(pool.to(DEVICE))
    return dict(case=case, pools=pools, sizes=sizes, rows=_i32(rows), before=_i32(before), new=_i32(new),
                tokens=sum(new) + case["spare"])


# ---- one pass -------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "select": _own_select, "reorder": _own_reorder, "tables": _own_tables}[op](state)
    return {"attention": _plain_attention, "select": _plain_select, "reorder": _plain_reorder, "tables": _plain_tables}[op](state)


def _own_attention(s):
    c = s["case"]
    return s["ops"].paged_attention_shared(s["qkv"], c["n_head"], c["n_kv_head"], c["head_dim"], c["head_dim"] ** -0.5,
                                           s["cache"], s["ctx"])


def _own_select(s):
    c = s["case"]
    got = s["ops"].beam_select(s["logits"], s["scores"], c["beams"], ended=s["ended"], lengths=s["lengths"], end_token=s["end"],
                               length_penalty=c["penalty"], vocab_limit=c["limit"] or None)
    return _choice(got.tokens, got.parents, got.scores, got.ranks, got.ended, got.lengths)


def _own_reorder(s):
    s["ops"].beam_reorder(s["parents"], s["lengths"], [s["table"]], [s["k"]], [s["v"]], s["slots"], s["states"])
    return [s["table"], s["k"], s["v"], *s["states"]]


def _own_tables(s):
    got = s["ops"].step_tables(s["pools"], s["sizes"], s["before"], s["new"], s["tokens"], rows=s["rows"])
    return [got.token_request, got.positions, got.req_q_start, *got.block_tables, *got.slot_mapping]


def _choice(tokens, parents, scores, ranks, ended, lengths):
    out = {"tokens": tokens, "parents": parents, "scores": scores, "ranks": ranks}
    if ended is not None:
        out["ended"] = ended
    if lengths is not None:
        out["lengths"] = lengths
    return out


def _softmax_rows(scores, seen):
    """Softmax over the last dimension of the scores where `seen`; a row that sees nothing gets zeros."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    return weights / torch.where(total == 0, torch.ones_like(total), total)


def _plain_attention(s):
    c = s["case"]
    H, KV, D, page, B = c["n_head"], c["n_kv_head"], c["head_dim"], c["page"], c["beams"]
    q = s["qkv"][:, : H * D].float().reshape(-1, KV, H // KV, D)
    out = torch.empty_like(q)
    for g, prompt in enumerate(s["prompts"]):
        rows = slice(g * B, (g + 1) * B)
        columns = -(-prompt // page)
        first = s["table"][g * B, :columns].long()
        # the prompt's keys and values once, [kv head, token, feature]
        k0 = s["k"][first].float().transpose(0, 1).reshape(KV, columns * page, D)[:, :prompt]
        v0 = s["v"][first].float().transpose(0, 1).reshape(KV, columns * page, D)[:, :prompt]
        begin = prompt // page                            # a row's own keys begin in this column
        own_pages = s["table"][rows, begin: -(-max(s["lengths"][rows]) // page)].long().clamp(min=0)
        k1 = s["k"][own_pages].float().transpose(1, 2).reshape(B, KV, -1, D)
        v1 = s["v"][own_pages].float().transpose(1, 2).reshape(B, KV, -1, D)
        at = begin * page + torch.arange(k1.shape[2], device=DEVICE)
        seen = (at >= prompt) & (at[None] <= s["positions"][rows, None])
        v1 = torch.where(seen[:, None, :, None], v1, 0.0)
        qg = q[rows] * D ** -0.5
        scores = torch.cat([torch.einsum("bkhd,ktd->bkht", qg, k0), torch.einsum("bkhd,bktd->bkht", qg, k1)], -1)
        shown = torch.cat([torch.ones((B, prompt), dtype=torch.bool, device=DEVICE), seen], -1)[:, None, None]
        weights = _softmax_rows(scores, shown)
        out[rows] = (torch.einsum("bkht,ktd->bkhd", weights[..., :prompt], v0)
                     + torch.einsum("bkht,bktd->bkhd", weights[..., prompt:], v1))
    return out.reshape(-1, H * D).to(s["qkv"].dtype)


def _plain_select(s):
    c = s["case"]
    G, I, B = c["groups"], c["in_beams"], c["beams"]
    limit = c["limit"] or c["vocab"]
    logits = s["logits"][:, :limit]
    # the best `beams` ids of every row; equal logits go to the lower id: 64-bit keys (logit, then id from above)
    bits = (logits + 0.0).contiguous().view(torch.int32).long()
    keys = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits)
    keys = keys * 2 ** 32 + (2 ** 32 - 1 - torch.arange(limit, device=DEVICE))
    ids = 2 ** 32 - 1 - (torch.topk(keys, B, dim=-1).values & (2 ** 32 - 1))
    wide = logits.double()
    top = wide.amax(-1, keepdim=True)
    total = top[:, 0] + torch.log(torch.exp(wide - top).sum(-1))
    before = s["scores"].double().reshape(-1, 1)
    value = before + (wide.gather(1, ids) - total[:, None])
    count = (s["lengths"].clamp(min=0)[:, None] + 1 if s["lengths"] is not None else torch.ones((G * I, 1), device=DEVICE)).expand(-1, B)
    if s["ended"] is not None:
        over = s["ended"][:, None] != 0
        first = torch.arange(B, device=DEVICE)[None] == 0
        value = torch.where(over, torch.where(first, before, -math.inf), value)
        ids = torch.where(over, s["end"], ids)
        count = torch.where(over, count - 1, count)
    value = torch.where(torch.isnan(value), -math.inf, value)
    weighed = value / count.double() ** c["penalty"]
    order = torch.sort(weighed.reshape(G, I * B), dim=-1, descending=True, stable=True).indices[:, :B]
    beam = order // B                                     # of the candidates chosen, best first
    again = (torch.tril((beam[:, :, None] == beam[:, None, :]).int(), -1).sum(-1) > 0)       # its row is taken by a better one
    taken = torch.zeros((G, B), dtype=torch.int64, device=DEVICE).scatter_(1, beam, 1)
    free = torch.sort(taken, dim=-1, stable=True).indices
    row = torch.where(again, free.gather(1, (torch.cumsum(again.int(), -1) - 1).clamp(min=0)), beam)
    place = torch.empty_like(row).scatter_(1, row, torch.arange(B, device=DEVICE).expand(G, B).contiguous())   # rank of each row
    order = order.gather(1, place)
    from_beam = order // B
    flat = (torch.arange(G, device=DEVICE)[:, None] * I * B + order).reshape(-1)
    tokens = ids.reshape(-1)[flat]
    parents = (torch.arange(G, device=DEVICE)[:, None] * B + from_beam).reshape(-1)
    ended = lengths = None
    in_row = (torch.arange(G, device=DEVICE)[:, None] * I + from_beam).reshape(-1)
    if s["ended"] is not None:
        ended = ((s["ended"][in_row] != 0) | (tokens == s["end"])).to(torch.int32)
    if s["lengths"] is not None:
        lengths = count.reshape(-1)[flat].to(torch.int32)
    return _choice(tokens.to(torch.int32), parents.to(torch.int32), value.reshape(-1)[flat].float().reshape(G, B),
                   place.reshape(-1).to(torch.int32), ended, lengths)


def _plain_reorder(s):
    page = s["case"]["page"]
    parents, length = s["parents"].long(), s["lengths"].long()[s["parents"].long()]
    rows = torch.arange(parents.numel(), device=DEVICE)
    moved = parents != rows
    full = (length // page)[:, None]                      # columns that the parent has filled: its pages are shared
    columns = torch.arange(s["table"].shape[1], device=DEVICE)[None]
    s["table"].copy_(torch.where(columns < full, s["table"][parents], s["table"]))
    # the tokens of the parent's part-filled page go to the row's own page of that column
    last = full.clamp(max=s["table"].shape[1] - 1)
    to, of = s["table"].gather(1, last)[:, 0].long(), s["table"][parents].gather(1, last)[:, 0].long()
    at = torch.arange(page, device=DEVICE)
    takes = (moved[:, None] & (at[None] < (length % page)[:, None])).nonzero()
    r, t = takes[:, 0], takes[:, 1]
    for x in (s["k"], s["v"]):
        x[:, to[r], :, t] = x[:, of[r], :, t]
    slots = s["slots"].long()
    for x in s["states"]:
        x[slots] = x[slots[parents]]
    return [s["table"], s["k"], s["v"], *s["states"]]


def _plain_tables(s):
    new, before = s["new"].long(), s["before"].long()
    start = torch.cumsum(new, 0) - new
    at = torch.arange(s["tokens"], device=DEVICE)
    request = (torch.searchsorted(torch.cumsum(new, 0), at, right=True)).clamp(max=new.numel() - 1)
    real = at < new.sum()
    positions = torch.where(real, before[request] + at - start[request], -1)
    request = torch.where(real, request, 0)
    tables, slots = [], []
    for pool, size in zip(s["pools"], s["sizes"]):
        held = pool[s["rows"].long()]
        columns = torch.arange(pool.shape[1], device=DEVICE)[None]
        table = torch.where(columns < ((before + new + size - 1) // size)[:, None], held, -1)
        tables.append(table)
        page = table[request, (positions // size).clamp(min=0)].long()
        slots.append(torch.where(real & (page >= 0), page * size + positions % size, -1).to(torch.int32))
    return [request.to(torch.int32), positions.to(torch.int32), start.to(torch.int32), *tables, *slots]


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        G, B, H, KV, D = (case[k] for k in ("groups", "beams", "n_head", "n_kv_head", "head_dim"))
        size = 2 if case["dtype"] == "bfloat16" else 4
        prompts, behind = _lengths(case)
        keys = sum(prompts) + sum(behind)                 # every key and value once
        pairs = B * sum(prompts) + sum(behind)            # of queries and keys
        return {"bytes": 2 * keys * KV * D * size + 2 * G * B * H * D * size, "flops": 4 * pairs * H * D}
    if case["op"] == "select":
        rows = case["groups"] * case["in_beams"]
        ids = case["limit"] or case["vocab"]
        return {"bytes": rows * ids * 4 + case["groups"] * case["beams"] * 24, "flops": 4 * rows * ids}
    if case["op"] == "reorder":
        G, B, page = case["groups"], case["beams"], case["page"]
        prompts, made = _lengths(case)
        parents = _keeping_parents(_rng(case, 0), G, B)   # (those of another seed differ in who goes on)
        size = 2 if case["dtype"] == "bfloat16" else 4
        token = case["layers"] * case["n_kv_head"] * (case["head_dim"] + case["v_dim"]) * size
        total = 0
        for r, p in enumerate(parents):
            length = prompts[r // B] + made[r]
            total += (p != r) * (length % page * token + length // page * 4 + case["states"] * case["state_words"] * 4)
        return {"bytes": 2 * total + 4 * len(parents), "flops": 0}
    new, before = _requests(case)
    total = 4 * (2 * (sum(new) + case["spare"]) + 4 * len(new))      # requests and positions; lengths, rows and starts
    for size in [case["page"]] + ([case["page2"]] if case["page2"] else []):
        width = -(-max(b + n for b, n in zip(before, new)) // size)
        total += 4 * (sum(-(-(b + n) // size) for b, n in zip(before, new)) + len(new) * width + sum(new) + case["spare"])
    return {"bytes": total, "flops": 0}


# ---- the definition in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    return {"attention": _exact_attention, "select": _exact_select, "reorder": _exact_reorder,
            "tables": _exact_tables}[case["op"]](case, seed)


def _exact_attention(case, seed):
    """Row by row: all of a row's keys through its own block table, one head group at a time."""
    s = _prepare_attention(case, seed)
    H, KV, D, page = case["n_head"], case["n_kv_head"], case["head_dim"], case["page"]
    share = H // KV
    out = torch.zeros((s["qkv"].shape[0], H * D), dtype=torch.float64, device=DEVICE)
    for r, n in enumerate(s["lengths"]):
        pages = s["table"][r, : -(-n // page)].long()
        k = s["k"][pages].double().permute(1, 0, 2, 3).reshape(KV, -1, D)[:, :n]
        v = s["v"][pages].double().permute(1, 0, 2, 3).reshape(KV, -1, D)[:, :n]
        q = s["qkv"][r, : H * D].double().reshape(KV, share, D)
        e = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(D)
        e = torch.exp(e - e.max(dim=-1, keepdim=True).values)
        out[r] = (torch.matmul(e, v) / e.sum(-1, keepdim=True)).reshape(-1)
    return out


def _exact_select(case, seed):
    """Prompt by prompt on the host: every candidate of every row, sorted once by value, row, logit and id."""
    s = _prepare_select(case, seed)
    G, I, B = case["groups"], case["in_beams"], case["beams"]
    limit = case["limit"] or case["vocab"]
    tokens, parents, scores, ranks, ended, lengths = [], [], [], [], [], []
    total = torch.logsumexp(s["logits"][:, :limit].double(), -1).tolist()
    best = torch.sort(s["logits"][:, :limit], dim=-1, descending=True, stable=True)
    best_v, best_i = best.values[:, :B].double().tolist(), best.indices[:, :B].tolist()
    before = s["scores"].double().reshape(-1).tolist()
    over = s["ended"].tolist() if s["ended"] is not None else None
    count = s["lengths"].tolist() if s["lengths"] is not None else None
    for g in range(G):
        candidates = []
        for b in range(I):
            r = g * I + b
            made = count[r] if count is not None else 0
            if over is not None and over[r]:
                listed_ones = [(before[r] if j == 0 else -math.inf, s["end"], made) for j in range(B)]
            else:
                listed_ones = [(before[r] + (v - total[r]), i, made + 1) for v, i in zip(best_v[r], best_i[r])]
            for j, (value, token, n) in enumerate(listed_ones):
                candidates.append((-value / float(n) ** case["penalty"] if case["penalty"] else -value, b, j, value, token, n))
        candidates.sort(key=lambda x: x[:3])
        chosen = candidates[:B]
        row_of, free = {}, []
        for rank, x in enumerate(chosen):
            if x[1] not in row_of:
                row_of[x[1]] = rank
            else:
                free.append(rank)
        for row in range(B):
            rank = row_of[row] if row in row_of else free.pop(0)
            _, b, _, value, token, n = chosen[rank]
            tokens.append(token)
            parents.append(g * B + b)
            scores.append(value)
            ranks.append(rank)
            ended.append(int(bool((over is not None and over[g * I + b]) or token == s["end"])))
            lengths.append(n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return _choice(i32(tokens), i32(parents), torch.tensor(scores, dtype=torch.float64).reshape(G, B), i32(ranks),
                   i32(ended) if over is not None else None, i32(lengths) if count is not None else None)


def _exact_reorder(case, seed):
    """Row by row; the values are moved, not computed."""
    s = _prepare_reorder(case, seed)
    page, parents, lengths, slots = case["page"], s["parents"].tolist(), s["lengths"].tolist(), s["slots"].tolist()
    tables = s["table"].tolist()
    for r, p in enumerate(parents):
        if p == r:
            continue
        full, used = lengths[p] // page, lengths[p] % page
        if used:
            for x in (s["k"], s["v"]):
                x[:, tables[r][full], :, :used] = x[:, tables[p][full], :, :used]
        s["table"][r, :full] = s["table"][p, :full]
        for x in s["states"]:
            x[slots[r]] = x[slots[p]]
    return [s["table"], *(x.double() for x in (s["k"], s["v"], *s["states"]))]


def _exact_tables(case, seed):
    """Token by token on the host."""
    s = _prepare_tables(case, seed)
    new, before, rows = s["new"].tolist(), s["before"].tolist(), s["rows"].tolist()
    request, positions, start, at = [], [], [], 0
    for r, (b, n) in enumerate(zip(before, new)):
        start.append(at)
        request += [r] * n
        positions += range(b, b + n)
        at += n
    tables, slots = [], []
    for pool, size in zip(s["pools"], s["sizes"]):
        held = pool.cpu().tolist()
        table = []
        for r, (b, n) in enumerate(zip(before, new)):
            pages = -(-(b + n) // size)
            table.append(held[rows[r]][:pages] + [-1] * (pool.shape[1] - pages))
        slot = [table[r][p // size] * size + p % size if table[r][p // size] >= 0 else -1 for r, p in zip(request, positions)]
        tables.append(torch.tensor(table, dtype=torch.int32))
        slots.append(torch.tensor(slot + [-1] * case["spare"], dtype=torch.int32))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return [i32(request + [0] * case["spare"]), i32(positions + [-1] * case["spare"]), i32(start), *tables, *slots]
