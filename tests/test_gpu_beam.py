"""What a beam search needs besides the model, each kernel against the plain forms in 64 bits: attention of rows that share
their first tokens, the choice of the next beams, caches handed over, and a step's integers on the device."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

import plain_beam
from mini_gpt_inference_b200.kernels.library import KernelLibraryError
from mini_gpt_inference_b200.parts.context import SharedPrefix

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from mini_gpt_inference_b200.kernels.ops import default_ops

    return default_ops("cuda:0")


def i32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


# ---- attention --------------------------------------------------------------------------------------
def shared_case(groups, loose, heads, page, dtype, seed, bounds=None, pad=0, spread=2.0, first_page=0, pool=None):
    """Rows of ``groups`` (list of (shared tokens, [keys behind them per row])), then ``loose`` rows of given lengths, then ``pad``
    rows of padding.  Pages lie in no order; what no row's context covers is NaN."""
    H, KV, D = heads
    gen = torch.Generator().manual_seed(seed)
    order, tables, lengths, spec, rows_k, rows_v = [], [], [], [], [], []
    count = 0
    for shared, behind in groups:
        spec.append([len(lengths), len(behind), shared])
        k0, v0 = (torch.randn(KV, shared, D, generator=gen).to(dtype) for _ in range(2))
        common = list(range(count, count + shared // page))
        count += len(common)
        for b in behind:
            own = -(-(shared + max(0, b)) // page) - len(common)
            tables.append(common + list(range(count, count + own)))
            count += own
            lengths.append(shared + b)
            rows_k.append(torch.cat([k0, torch.randn(KV, max(0, b), D, generator=gen).to(dtype)], 1))
            rows_v.append(torch.cat([v0, torch.randn(KV, max(0, b), D, generator=gen).to(dtype)], 1))
    for n in loose:
        tables.append(list(range(count, count + -(-n // page))))
        count += len(tables[-1])
        lengths.append(n)
        rows_k.append(torch.randn(KV, n, D, generator=gen).to(dtype))
        rows_v.append(torch.randn(KV, n, D, generator=gen).to(dtype))
    pages = pool or count + 2
    order = [first_page + p for p in torch.randperm(count + 2, generator=gen).tolist()]
    k_pages = torch.full((pages, KV, page, D), math.nan, dtype=dtype, device="cuda")
    v_pages = torch.full((pages, KV, page, D), math.nan, dtype=dtype, device="cuda")
    width = max(len(t) for t in tables) + 1
    for table, k, v in zip(tables, rows_k, rows_v):
        for c, p in enumerate(table):
            used = min(page, k.shape[1] - c * page)
            k_pages[order[p], :, :used] = k[:, c * page: c * page + used].cuda()
            v_pages[order[p], :, :used] = v[:, c * page: c * page + used].cuda()
    n = len(lengths) + pad
    q = (torch.randn(n, (H + 2 * KV) * D, generator=gen) * spread).to(dtype)
    rows = torch.randperm(n, generator=gen).tolist()                       # requests lie in another order than the rows
    block_table = torch.full((n, width), -1, dtype=torch.int32)
    for r, table in enumerate(tables):
        block_table[rows[r], : len(table)] = torch.tensor([order[p] for p in table], dtype=torch.int32)
    bounds = bounds or (max([len(b) for _, b in groups] or [1]), max([s for s, _ in groups] or [0]),
                        max([1] + [b for _, bs in groups for b in bs] + list(loose)))
    ctx = SimpleNamespace(block_tables=[block_table.cuda()], token_request=i32(rows), positions=i32([m - 1 for m in lengths] + [-1] * pad),
                          decode_only=True, extra={}, max_ctx_after=max(lengths),
                          shared_prefix=SharedPrefix(i32(spec).reshape(-1, 3), *bounds))
    cache = SimpleNamespace(k_pages=k_pages, v_pages=v_pages, group=0, page_tokens=page, window=None, writes=False,
                            values_in_keys=False, keep_first=0)
    return SimpleNamespace(q=q.cuda(), ctx=ctx, cache=cache, heads=heads, k=[k[:, :n] for k, n in zip(rows_k, lengths)],
                           v=[v[:, :n] for v, n in zip(rows_v, lengths)], pad=pad)


def check_attention(case, out, dtype):
    H, KV, D = case.heads
    for r, (k, v) in enumerate(zip(case.k, case.v)):
        want, size = plain_beam.attention_row(case.q[r, : H * D].cpu().reshape(H, D), k, v, D ** -0.5)
        got = out[r].double().cpu().reshape(H, D)
        # 32 bits: a score is a sum of D products, off by some sqrt(D) 2^-24 of its parts, and a weight by as much of itself;
        # twenty times that of the weighed values' sum.  bfloat16: half a step (2^-8) for the rounding of each weight, and
        # half a step of the result.
        tol = 20 * math.sqrt(D) * 2.0 ** -24 * size + 1e-6
        if dtype == BF16:
            tol = tol + 2.0 ** -8 * (size + want.abs())
        bad = (got - want).abs() > tol
        assert not bad.any() and torch.isfinite(got).all(), (r, float((got - want).abs().max()), float(tol.min()))
    if case.pad:
        assert (out[len(case.k):] == 0).all()


def run_attention(ops, case):
    H, KV, D = case.heads
    return ops.paged_attention_shared(case.q, H, KV, D, D ** -0.5, case.cache, case.ctx)


SHAPES = {
    "one group": ([(37, [5, 5, 1, 3])], [], 0),
    "one token": ([(1, [1])], [], 0),
    "ragged groups, loose rows, padding": ([(1, [1]), (130, [1, 2, 70]), (64, [64, 1]), (65, [0, 3])], [1, 200], 3),
    "nothing shared": ([(0, [7, 9])], [33], 1),
    "no groups": ([], [1, 65, 300], 0),
    "many rows": ([(200, [1 + i % 40 for i in range(70)])], [], 0),
    "long": ([(2500, [130, 1, 64])], [1700], 0),
}
HEADS = [(8, 8, 64), (4, 1, 48), (12, 4, 128), (5, 5, 16), (2, 2, 256), (3, 3, 40), (32, 8, 128), (20, 1, 32), (6, 2, 7)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("heads,page", [(h, (16, 5, 64, 1, 16, 8, 64, 16, 3)[i]) for i, h in enumerate(HEADS)])
def test_attention_shared(ops, dtype, shape, heads, page):
    groups, loose, pad = SHAPES[shape]
    case = shared_case(groups, loose, heads, page, dtype, seed=len(shape), pad=pad)
    check_attention(case, run_attention(ops, case), dtype)


@pytest.mark.parametrize("heads,page,shape", [
    ((8, 8, 64), 16, [(700, [3] * 70)]), ((32, 8, 128), 64, [(1300, [1 + i % 50 for i in range(100)]), (128, [5] * 3)]),
    ((16, 2, 128), 8, [(129, [2] * 9), (64, [1] * 20), (400, [-5, 7] * 20)]), ((64, 1, 64), 128, [(2049, [9] * 5), (0, [200] * 2)]),
    ((12, 4, 64), 32, [(300, [4] * 171)]), ((5, 1, 128), 256, [(513, [3] * 26)]), ((96, 1, 128), 16, [(1000, [70])])])
@pytest.mark.parametrize("spread", [2.0, 30.0])
def test_attention_shared_many_pairs(ops, heads, page, shape, spread):
    """Tiles of 128 (row, head) pairs on the 5th-generation tensor cores: odd numbers of pairs and keys, rows in front of the
    shared end, scores whose largest come late (the reference moves)."""
    case = shared_case(shape, [40], heads, page, BF16, seed=21, pad=1, spread=spread)
    H, KV, D = heads
    out = run_attention(ops, case)
    ops.check_status()
    for r, (k, v) in enumerate(zip(case.k, case.v)):
        want, size = plain_beam.attention_row(case.q[r, : H * D].cpu().reshape(H, D), k, v, D ** -0.5)
        # as in check_attention, the scores being `spread` / 2 times as large
        tol = (20 * spread * math.sqrt(D) * 2.0 ** -24 + 2.0 ** -8) * (size + want.abs()) + 1e-6
        assert ((out[r].double().cpu().reshape(H, D) - want).abs() <= tol).all(), r
    assert (out[len(case.k):] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bounds", [(1, 1, 1), (1, 0, 1), (3, 10000, 10000), (64, 64, 64)])
def test_attention_shared_bounds_are_hints(ops, dtype, bounds):
    case = shared_case([(300, [90, 1, 5, 17] * 9), (5, [1, 700])], [260], (8, 2, 64), 16, dtype, seed=3, bounds=bounds)
    check_attention(case, run_attention(ops, case), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_shared_rows_in_front_of_the_shared_end(ops, dtype):
    """Rows whose own position lies among the shared tokens see the keys up to their own."""
    case = shared_case([(140, [-139, 3, -1, -70, 1])], [], (8, 8, 64), 16, dtype, seed=5)
    check_attention(case, run_attention(ops, case), dtype)


@pytest.mark.parametrize("width", [1, 2, 8])
def test_attention_shared_rows_of_other_widths(ops, width):
    """Queries in rows that are wider by a few numbers: at 16-byte boundaries or not."""
    for heads, shape in (((8, 8, 64), [(300, [3] * 80)]), ((4, 2, 48), [(70, [1, 200])])):
        case = shared_case(shape, [], heads, 16, BF16, seed=31)
        case.q = torch.cat([case.q, torch.full((case.q.shape[0], width), math.nan, dtype=BF16, device="cuda")], 1)
        check_attention(case, run_attention(ops, case), BF16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_shared_groups_that_are_none(ops, dtype):
    """No rows, rows in front of the batch or behind it, tokens below zero or beyond any block table: the rows read all their keys."""
    case = shared_case([], [400, 30, 90, 260], (8, 2, 64), 16, dtype, seed=32, bounds=(4, 300, 400))
    case.ctx.shared_prefix.groups = i32([[-1, 2, 16], [0, 0, 16], [4, 3, 16], [0, 1, -5], [1, 1, 10 ** 9], [2, 2, 2 ** 31 - 1]])
    check_attention(case, run_attention(ops, case), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_shared_scores_of_large_range(ops, dtype):
    case = shared_case([(700, [30, 40, 1])], [], (4, 4, 64), 16, dtype, seed=6, spread=40.0)
    out = run_attention(ops, case)
    H, KV, D = case.heads
    for r, (k, v) in enumerate(zip(case.k, case.v)):
        want, size = plain_beam.attention_row(case.q[r, : H * D].cpu().reshape(H, D), k, v, D ** -0.5)
        # scores of some 300: their error, 2^-24 sqrt(D) of that, is the weights' relative one
        tol = (20 * 300 * 8 * 2.0 ** -24 + (2.0 ** -8 if dtype == BF16 else 0)) * (size + want.abs()) + 1e-6
        assert ((out[r].double().cpu().reshape(H, D) - want).abs() <= tol).all()


@pytest.mark.parametrize("behind", [13, 400])
def test_attention_shared_missing_pages(ops, behind):
    case = shared_case([(32, [13, behind])], [20], (8, 8, 64), 16, BF16, seed=7)
    table = case.ctx.block_tables[0]
    row = int(case.ctx.token_request[2])
    table[row] = -1                                                        # a row without any page: zeros
    table[int(case.ctx.token_request[1]), 2] = case.cache.k_pages.shape[0] + 5        # a page beyond the pool: its keys are not there
    out = run_attention(ops, case)
    assert (out[2] == 0).all()
    keep = [t for t in range(case.k[1].shape[1]) if not 32 <= t < 48]      # (the tokens of that page)
    case.k[1], case.v[1] = case.k[1][:, keep], case.v[1][:, keep]
    case.k, case.v, case.pad = case.k[:2], case.v[:2], 1
    check_attention(case, out, BF16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_shared_beyond_32_bit_offsets(ops, dtype):
    """A pool of more than 2^31 numbers, the rows' pages at its end."""
    heads, page = (2, 2, 256), 64
    pool = 2 ** 31 // (2 * 64 * 256) + 40
    case = shared_case([(150, [30, 1])], [70], heads, page, dtype, seed=8, first_page=pool - 30, pool=pool)
    check_attention(case, run_attention(ops, case), dtype)


def test_attention_shared_captured_with_other_lengths(ops):
    """One captured launch, replayed for two batches of other lengths, on another stream than the default one; two graphs
    replayed in turn."""
    cases = [shared_case([(377, [20, 3, 40]), (77, [9, 9, 1])], [], (8, 8, 64), 16, BF16, seed=s, bounds=(3, 400, 64)) for s in (1, 2)]
    other = shared_case([(30, [2, 60, 40]), (300, [1, 30, 8])], [], (8, 8, 64), 16, BF16, seed=3, bounds=(3, 400, 64))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for case in cases:
            run_attention(ops, case)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(run_attention(ops, case))
            graphs.append(graph)
        for _ in range(2):
            for graph in graphs:
                graph.replay()
        side.synchronize()
        for case, out in zip(cases, outs):
            check_attention(case, out, BF16)
        # the first graph's inputs become those of another batch
        a, b = cases[0], other
        width, pages = b.ctx.block_tables[0].shape[1], b.cache.k_pages.shape[0]
        assert a.ctx.block_tables[0].shape[1] >= width and a.cache.k_pages.shape[0] >= pages
        a.ctx.block_tables[0][:, :width] = b.ctx.block_tables[0]
        a.ctx.token_request.copy_(b.ctx.token_request)
        a.ctx.positions.copy_(b.ctx.positions)
        a.ctx.shared_prefix.groups.copy_(b.ctx.shared_prefix.groups)
        a.cache.k_pages[:pages] = b.cache.k_pages
        a.cache.v_pages[:pages] = b.cache.v_pages
        a.q.copy_(b.q)
        graphs[0].replay()
        side.synchronize()
        check_attention(b, outs[0], BF16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_shared_through_paged_attention(ops, dtype):
    """``paged_attention`` takes the form for shared tokens where the step says that rows share some, and gives the same."""
    case = shared_case([(130, [4, 9, 1]), (20, [30, 2])], [], (8, 2, 64), 16, dtype, seed=9)
    H, KV, D = case.heads
    before = ops.launches
    out = ops.paged_attention(case.q, H, KV, D, D ** -0.5, case.cache, case.ctx)
    assert ops.launches - before == 1                                       # (few keys: a range a row)
    check_attention(case, out, dtype)
    case.ctx.shared_prefix = None
    check_attention(case, ops.paged_attention(case.q, H, KV, D, D ** -0.5, case.cache, case.ctx), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bounds", [(2 ** 31 - 1,) * 3, (2 ** 40, 2 ** 33, 2 ** 32), (1, 0, 2 ** 31 - 1)])
def test_attention_shared_bounds_without_end(ops, dtype, bounds):
    """Bounds beyond all numbers (no bounds, that is) count as what the block tables can hold."""
    case = shared_case([(300, [90, 1, 5]), (40, [3, 1])], [200], (8, 2, 64), 16, dtype, seed=6, bounds=bounds, pad=1)
    check_attention(case, run_attention(ops, case), dtype)


@pytest.mark.parametrize("heads,rows,shared,page", [((8, 8, 96), 8, 300, 16), ((8, 8, 128), 5, 1000, 5), ((16, 8, 104), 4, 140, 64)])
def test_attention_shared_many_short_ranges(ops, heads, rows, shared, page):
    """So many CTAs of few keys that they take the smallest rings: ranges of no, one and some keys, features padded to 128."""
    groups = [(shared - 7 * i, [1 + (11 * i + 5 * j) % 90 for j in range(rows)]) for i in range(8)] + [(1, [1, 1, 129])]
    case = shared_case(groups, [1, 16, 17, 200] * 8, heads, page, BF16, seed=shared, pad=2)
    check_attention(case, run_attention(ops, case), BF16)


# ---- the choice of the next beams -----------------------------------------------------------------------
def check_choice(got, want, groups, beams):
    for name in ("tokens", "parents", "ranks", "ended", "lengths"):
        value = getattr(got, name)
        if value is not None:
            assert value.tolist() == want[name], name
    got_scores, scores = got.scores.double().cpu().reshape(-1), torch.tensor(want["scores"], dtype=torch.float64)
    finite = torch.isfinite(scores)
    assert torch.equal(torch.isfinite(got_scores), finite) and (got_scores[~finite] == scores[~finite]).all()
    # the sum of the exponentials in 32 bits, each off by some 2^-22 at arguments up to 16: 2^-18 of the logarithm's value at
    # the very most; and the result's own rounding
    assert ((got_scores - scores)[finite].abs() <= 2.0 ** -18 + 2.0 ** -24 * scores[finite].abs()).all()


@pytest.mark.parametrize("groups,in_beams,beams,vocab,limit", [
    (1, 1, 1, 1, 0), (1, 1, 4, 50304, 50257), (3, 4, 4, 97, 0), (2, 1, 32, 32, 0), (2, 32, 32, 1001, 999), (5, 3, 7, 5000, 4999),
    (40, 8, 8, 513, 0), (1, 2, 2, 50257, 0), (2, 16, 16, 33000, 0), (64, 16, 16, 1111, 0)])
@pytest.mark.parametrize("ends", [False, True])
def test_beam_select(ops, groups, in_beams, beams, vocab, limit, ends):
    gen = torch.Generator().manual_seed(vocab + beams)
    rows = groups * in_beams
    logits = torch.randn(rows, vocab, generator=gen) * 3
    scores = -10 * torch.rand(groups, in_beams, generator=gen)
    lengths = torch.randint(0, 9, (rows,), generator=gen, dtype=torch.int32)
    ended = (torch.rand(rows, generator=gen) < 0.3).to(torch.int32)
    end = (limit or vocab) // 2
    more = dict(ended=ended, end_token=end, lengths=lengths, length_penalty=0.7) if ends else {}
    got = ops.beam_select(logits.cuda(), scores.cuda(), beams, vocab_limit=limit or None,
                          **{k: v.cuda() if torch.is_tensor(v) else v for k, v in more.items()})
    check_choice(got, plain_beam.beam_select(logits, scores, beams, vocab_limit=limit or None, **more), groups, beams)
    parents = got.parents.long()
    assert torch.equal(parents[parents], parents)


@pytest.mark.parametrize("what", ["equal", "few values", "minus infinity", "nan", "one row nothing", "all nothing", "infinite", "rising",
                                  "zeros of both signs", "same rows"])
def test_beam_select_ties_and_odd_numbers(ops, what):
    gen = torch.Generator().manual_seed(5)
    groups, in_beams, beams, vocab = 2, 4, 4, 1500
    logits = torch.randn(groups * in_beams, vocab, generator=gen)
    scores = -3 * torch.rand(groups, in_beams, generator=gen)
    if what == "equal":
        logits[:] = 0.25
    elif what == "few values":
        logits = logits.round()
    elif what == "minus infinity":
        logits[:, 3:] = -math.inf
    elif what == "nan":
        logits[:, ::3] = math.nan
    elif what == "one row nothing":
        logits[1], logits[5] = -math.inf, math.nan
    elif what == "all nothing":
        logits[:], scores[0, 2] = -math.inf, -math.inf
    elif what == "infinite":
        logits[2, 700] = math.inf
        scores[1, 1] = math.nan
    elif what == "rising":
        logits = torch.arange(vocab).float().repeat(groups * in_beams, 1) * 0.01 + torch.rand(groups * in_beams, 1, generator=gen)
    elif what == "zeros of both signs":
        logits[:] = 0.0
        logits[:, ::2] = -0.0
    elif what == "same rows":
        logits[:], scores[:] = logits[0].clone(), -1.0
        scores[1] = torch.tensor([0.0, -math.inf, -math.inf, -math.inf])
    got = ops.beam_select(logits.cuda(), scores.cuda(), beams)
    check_choice(got, plain_beam.beam_select(logits, scores, beams), groups, beams)


@pytest.mark.parametrize("beams", [5, 32])
@pytest.mark.parametrize("what", ["equal", "few allowed", "few values", "last one", "two values"])
def test_beam_select_ties_over_a_long_row(ops, what, beams):
    """Ties over several pieces of a row: the lowest ids go on, wherever they lie."""
    gen = torch.Generator().manual_seed(beams)
    groups, in_beams, vocab = 2, 3, 50257
    logits = torch.randn(groups * in_beams, vocab, generator=gen)
    scores = -3 * torch.rand(groups, in_beams, generator=gen)
    if what == "equal":
        logits[:] = -1.5
    elif what == "few allowed":
        logits[:, torch.randperm(vocab, generator=gen)[3:]] = -math.inf
    elif what == "few values":
        logits = (logits * 2).round()
    elif what == "last one":
        logits[:] = 0.0
        logits[:, -1] = 1.0
    elif what == "two values":
        logits = (torch.rand(groups * in_beams, vocab, generator=gen) < 0.01).float()
    got = ops.beam_select(logits.cuda(), scores.cuda(), beams)
    check_choice(got, plain_beam.beam_select(logits, scores, beams), groups, beams)


def test_beam_select_all_ended_and_unaligned_rows(ops):
    logits = torch.randn(4 * 777 + 1, generator=torch.Generator().manual_seed(1))
    view = logits.cuda()[1:].view(4, 777)                                   # starts four bytes behind a boundary
    scores = torch.tensor([[-3.0, -1.0], [-2.0, -2.0]])
    ended = torch.tensor([1, 1, 0, 1], dtype=torch.int32)
    for limit in (777, 3):
        got = ops.beam_select(view, scores.cuda(), 2, ended=ended.cuda(), end_token=1, vocab_limit=limit)
        check_choice(got, plain_beam.beam_select(logits[1:].view(4, 777), scores, 2, ended=ended, end_token=1, vocab_limit=limit), 2, 2)


def test_beam_select_in_place_and_replayed(ops):
    """The outputs may be the inputs; a captured choice is replayed step after step."""
    gen = torch.Generator().manual_seed(11)
    groups, beams, vocab, end = 3, 4, 2000, 7
    steps = [torch.randn(groups * beams, vocab, generator=gen) * 2 for _ in range(4)]
    for x in steps:
        x[:, end] += 5
    logits = torch.empty(groups * beams, vocab, device="cuda")
    state = ops.beam_select(steps[0].cuda()[::beams].contiguous(), torch.zeros(groups, 1, device="cuda"), beams, end_token=end,
                            lengths=i32([0] * groups), length_penalty=1.0)
    want = plain_beam.beam_select(steps[0][::beams], torch.zeros(groups, 1), beams, end_token=end, lengths=i32([0] * groups), length_penalty=1.0)
    check_choice(state, want, groups, beams)
    start = [t.clone() for t in (state.tokens, state.parents, state.scores, state.ranks, state.ended, state.lengths)]

    def call():
        ops.beam_select(logits, state.scores, beams, ended=state.ended, lengths=state.lengths, end_token=end, length_penalty=1.0,
                        out=state)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for t, s in zip((state.tokens, state.parents, state.scores, state.ranks, state.ended, state.lengths), start):
        t.copy_(s)
    for x in steps[1:]:
        logits.copy_(x)
        scores = state.scores.cpu()
        graph.replay()
        want = plain_beam.beam_select(x, scores, beams, end_token=end,
                                      ended=torch.tensor(want["ended"]), lengths=torch.tensor(want["lengths"]), length_penalty=1.0)
        check_choice(state, want, groups, beams)


# ---- caches of rows that do not go on ---------------------------------------------------------------------
def reorder_case(parents, lengths, page, layers, heads, k_size, v_size, dtype, seed, states=(), one_layer=False, in_keys=False):
    gen = torch.Generator().manual_seed(seed)
    rows, width = len(parents), max(lengths) // page + 2
    pages = rows * width + 3
    table = torch.randperm(pages, generator=gen)[: rows * width].reshape(rows, width).to(torch.int32)
    lead = () if one_layer else (layers,)
    k = torch.randn(*lead, pages, heads, page, k_size, generator=gen).to(dtype)
    v = None if in_keys else torch.randn(*lead, pages, heads, page, v_size, generator=gen).to(dtype)
    slots = torch.randperm(rows + 4, generator=gen)[:rows].to(torch.int32)
    kept = [torch.randn(rows + 4, *shape, generator=gen).mul(100).to(kind) for shape, kind in states]
    return (torch.tensor(parents, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32), [table], [k], [v], slots, kept)


@pytest.mark.parametrize("parents,lengths", [([0], [5]), ([0, 0, 0, 3], [37] * 4), ([1, 1, 2, 2, 4, 4], [16, 16, 31, 31, 1, 1]),
                                             ([0] * 20 + [20] * 3, [130] * 20 + [7] * 3), ([0, 0], [0, 0])])
@pytest.mark.parametrize("page,layers,heads,k_size,v_size,dtype", [
    (16, 8, 8, 64, 64, BF16), (16, 1, 1, 24, 8, F32), (5, 3, 2, 3, 7, BF16), (1, 2, 2, 64, 64, BF16), (64, 2, 4, 128, 64, F32)])
def test_beam_reorder(ops, parents, lengths, page, layers, heads, k_size, v_size, dtype):
    states = [((3, 5), F32), ((1,), torch.int32), ((7,), BF16), ((1000, 33), F32), ((9,), torch.uint8)]
    for more in (dict(states=states), dict(one_layer=layers == 1, in_keys=True)):
        args = reorder_case(parents, lengths, page, layers, heads, k_size, v_size, dtype, seed=len(parents), **more)
        dev = [a.cuda() if torch.is_tensor(a) else [x.cuda() if x is not None else None for x in a] for a in args]
        ops.beam_reorder(*dev)
        plain_beam.beam_reorder(*args)
        for a, d in zip(args, dev):
            for x, y in zip([a] if torch.is_tensor(a) else a, [d] if torch.is_tensor(d) else d):
                assert x is None or torch.equal(x, y.cpu())


def test_beam_reorder_values_in_the_key_pages_and_two_groups(ops):
    a = reorder_case([0, 0, 2, 0], [20] * 4, 16, 2, 1, 64, 64, BF16, 1, in_keys=True)
    b = reorder_case([0, 0, 2, 0], [20] * 4, 4, 1, 2, 32, 16, BF16, 2)
    join = lambda x, y: [x[0], x[1], x[2] + y[2], x[3] + y[3], x[4] + y[4]]  # noqa: E731
    host = join(a, b)
    dev = [x.cuda() if torch.is_tensor(x) else [y.cuda() if y is not None else None for y in x] for x in host]
    dev[4][0] = dev[3][0]                                                    # as a cache of latents hands them over
    ops.beam_reorder(*dev)
    plain_beam.beam_reorder(*host)
    for x, y in zip(host[2] + host[3] + host[4][1:], dev[2] + dev[3] + dev[4][1:]):
        assert torch.equal(x, y.cpu())


def test_beam_reorder_leaves_bad_rows_alone(ops):
    """A parent out of range, one that is not its own, a missing page or slot: the row stays as it was."""
    args = reorder_case([9, -1, 3, 0, 4, 4, 4], [21] * 7, 16, 2, 2, 16, 16, F32, 3, states=[((4,), F32)])
    args[2][0][5, 1] = -1
    args[2][0][6, 1] = 10 ** 6
    args[5][5] = -1
    args[5][6] = 99
    dev = [a.cuda() if torch.is_tensor(a) else [x.cuda() for x in a] for a in args]
    ops.beam_reorder(*dev)
    want = args[2][0].clone()
    want[5, 0], want[6, 0] = want[4, 0], want[4, 0]                          # (their full pages are handed over)
    assert torch.equal(dev[2][0].cpu(), want)
    for a, d in zip(args[3] + args[4] + args[6], dev[3] + dev[4] + dev[6]):
        assert torch.equal(a, d.cpu())


# ---- a step's integers ------------------------------------------------------------------------------------
@pytest.mark.parametrize("fresh,before,spare,rows", [
    ([1], [0], 0, False), ([1, 1, 1, 1], [36, 15, 16, 17], 0, False), ([3, 0, 5, 1, 0], [10, 4, 0, 63, 0], 6, True),
    ([1 + i % 7 for i in range(300)], [i * 5 % 470 for i in range(300)], 9, True), ([2000, 1, 48], [0, 9, 300], 0, False),
    ([0, 0], [5, 9], 4, True), ([1] * 4096, [i % 500 for i in range(4096)], 0, False)])
@pytest.mark.parametrize("sizes", [[16], [1, 64, 5], [32] * 8, []])
def test_step_tables(ops, fresh, before, spare, rows, sizes):
    gen = torch.Generator().manual_seed(len(fresh))
    R, longest = len(fresh), max(b + n for b, n in zip(before, fresh))
    if R > 1000 and len(sizes) > 1:
        sizes = sizes[:2]
    pool_rows = R + 5 if rows else R
    pools = [torch.randint(0, 9999, (pool_rows, -(-longest // s) + 1), generator=gen, dtype=torch.int32) for s in sizes]
    for pool in pools:
        pool[:, 0] = torch.where(torch.rand(pool_rows, generator=gen) < 0.2, -1, pool[:, 0])        # pages that were given back
    at = torch.randperm(pool_rows, generator=gen)[:R].to(torch.int32) if rows else None
    f, b = torch.tensor(fresh, dtype=torch.int32), torch.tensor(before, dtype=torch.int32)
    n = sum(fresh) + spare
    got = ops.step_tables([p.cuda() for p in pools], sizes, b.cuda(), f.cuda(), n, rows=at.cuda() if rows else None)
    request, positions, start, tables, slots = plain_beam.step_tables(pools, sizes, b, f, n, at)
    assert got.token_request.tolist() == request and got.positions.tolist() == positions and got.req_q_start.tolist() == start
    for g in range(len(sizes)):
        assert got.block_tables[g].tolist() == tables[g] and got.slot_mapping[g].tolist() == slots[g]


def test_step_tables_short_of_rows_and_pages(ops):
    """Fewer token rows than tokens, positions behind the last column, rows of no pool: nothing is read or written outside."""
    pools = [torch.arange(12, dtype=torch.int32).reshape(3, 4)]
    fresh, before, rows = i32([5, 2, 2]), i32([14, 3, 0]), i32([2, 7, -1])
    got = ops.step_tables([p.cuda() for p in pools], [4], before, fresh, 8, rows=rows)
    assert got.positions.tolist() == [14, 15, 16, 17, 18, 3, 4, 0]
    assert got.slot_mapping[0].tolist() == [11 * 4 + 2, 11 * 4 + 3, -1, -1, -1, -1, -1, -1]
    assert got.block_tables[0].tolist() == [[8, 9, 10, 11], [-1] * 4, [-1] * 4]


# ---- refusals -----------------------------------------------------------------------------------------------
def test_refusals(ops):
    import beam_refusals

    for name, call in beam_refusals.calls(ops, "cuda"):
        with pytest.raises(KernelLibraryError):
            call()
            pytest.fail(f"not refused: {name}")
