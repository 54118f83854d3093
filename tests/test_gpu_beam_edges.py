"""The beam search's kernels on inputs at the edge of what a call allows: numbers that are none, groups whose first rows see
less than the others, scales below zero, large logits."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

import plain_beam
from test_gpu_beam import BF16, F32, check_attention, check_choice, i32, run_attention, shared_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from mini_gpt_inference_b200.kernels.ops import default_ops

    return default_ops("cuda:0")


# ---- attention: the kernels that a call may take, by type and shape ------------------------------------
JOINED, DIRECT = [(300, [90, 1, 70]), (5, [1])], [(70, [5, 20, 9]), (5, [1])]
KERNELS = {
    "32-bit": (F32, (4, 2, 64), JOINED), "32-bit, one launch": (F32, (4, 2, 64), DIRECT),
    "32-bit, many ranges": (F32, (4, 2, 64), [(700, [200, 1])]),
    "32-bit, odd heads": (F32, (3, 3, 7), JOINED),
    "bfloat16": (BF16, (4, 2, 64), JOINED), "bfloat16, one launch": (BF16, (4, 2, 64), DIRECT),
    "bfloat16, both halves of a weight": (BF16, (4, 2, 48), JOINED), "bfloat16, odd heads": (BF16, (3, 3, 7), JOINED),
    "tiles of 64": (BF16, (8, 8, 64), [(300, [90, 1, 70] * 14), (5, [1])]),
    "tiles of 128": (BF16, (32, 8, 128), [(300, [90, 1, 70] * 5), (5, [1])]),
}


def set_keys(case, rows, tokens, kv_head, feature, value):
    """Feature of the keys of some tokens of some rows, in the pages and in what the plain form sees."""
    page = case.cache.page_tokens
    for r in rows:
        table = case.ctx.block_tables[0][int(case.ctx.token_request[r])].tolist()
        for t in tokens:
            if t < case.k[r].shape[1]:
                case.cache.k_pages[table[t // page], kv_head, t % page, feature] = value
                case.k[r][kv_head, t, feature] = value


def check_numbers(case, out, dtype, scale=None):
    """No numbers exactly where the 64-bit softmax has none, the others as close as ever."""
    H, KV, D = case.heads
    some = False
    for r, (k, v) in enumerate(zip(case.k, case.v)):
        want, size = plain_beam.attention_row(case.q[r, : H * D].cpu().reshape(H, D), k, v, D ** -0.5 if scale is None else scale)
        got = out[r].double().cpu().reshape(H, D)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), r
        some = some or bool(torch.isnan(want).any())
        # (see test_gpu_beam.check_attention)
        tol = 20 * math.sqrt(D) * 2.0 ** -24 * size + 1e-6
        if dtype == BF16:
            tol = tol + 2.0 ** -8 * (size + want.abs())
        there = ~torch.isnan(want)
        assert ((got - want).abs() <= tol)[there].all(), (r, float((got - want)[there].abs().max()))
    return some


@pytest.mark.parametrize("what", ["query", "shared key", "shared keys", "own key", "low query", "high query", "low shared keys",
                                  "low first key"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_attention_shared_keeps_what_is_no_number(ops, kernel, what):
    """A query or a key that is none, one or a whole range of them; scores of minus infinity everywhere, or of a range alone (which then
    counts for nothing), and infinite ones."""
    dtype, heads, groups = KERNELS[kernel]
    case = shared_case(groups, [40], heads, 16, dtype, seed=51, pad=1)
    H, KV, D = heads
    n, first = len(case.k), len(groups[0][1])
    q = case.q.view(n + 1, -1)
    group, everyone = range(first), range(n)
    if what == "query":
        q[1, 3] = math.nan
    elif what == "shared key":
        set_keys(case, group, [33], KV - 1, 5, math.nan)
    elif what == "shared keys":
        set_keys(case, group, range(64), 0, 5, math.nan)
    elif what == "own key":
        set_keys(case, [first - 1], [case.k[first - 1].shape[1] - 1], 0, 5, math.nan)
    elif what in ("low query", "high query"):
        q[1, 0] = -math.inf if what == "low query" else math.inf
        case.cache.k_pages[:, 0, :, 0] = case.cache.k_pages[:, 0, :, 0].abs() + 1
        for k in case.k:
            k[0, :, 0] = k[0, :, 0].abs() + 1
    else:
        q[:n, : H * D: D] = q[:n, : H * D: D].abs() + 1                      # every head's first feature
        for head in range(KV):
            set_keys(case, group if what == "low shared keys" else everyone, range(64) if what == "low shared keys" else [0], head, 0, -math.inf)
    out = run_attention(ops, case)
    ops.check_status()
    some = check_numbers(case, out, dtype)
    assert some == (what not in ("low shared keys", "low first key"))
    assert (out[n:] == 0).all()


@pytest.mark.parametrize("how", ["short first rows", "padding first", "nobody sees all"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_attention_shared_takes_pages_of_a_row_that_sees_them(ops, kernel, how):
    """Groups whose first rows stand in front of the shared end, with block tables as ``step_tables`` leaves them (nothing behind the
    last page), or are padding, whose request is another one's."""
    dtype, heads, groups = KERNELS[kernel]
    shared, behind = groups[0]
    short = [-shared + 1, -shared + 20] if how != "padding first" else []
    behind = short + ([1 - shared // 2] * 5 if how == "nobody sees all" else behind)
    case = shared_case([(shared, behind), *groups[1:]], [40], heads, 16, dtype, seed=61)
    for r, k in enumerate(case.k):
        request = int(case.ctx.token_request[r])
        case.ctx.block_tables[0][request, -(-k.shape[1] // 16):] = -1
    padding = []
    if how == "padding first":
        padding = [0, 1] if len(behind) > 3 else [0]
        for r in padding:
            case.ctx.positions[r] = -1
            case.ctx.token_request[r] = int(case.ctx.token_request[len(case.k) - 1])
    out = run_attention(ops, case)
    ops.check_status()
    assert (out[padding] == 0).all()
    keep = [r for r in range(len(case.k)) if r not in padding]
    case.k, case.v, case.q, out = [case.k[r] for r in keep], [case.v[r] for r in keep], case.q[keep], out[keep]
    assert not check_numbers(case, out, dtype)


@pytest.mark.parametrize("scale", [-0.2, 0.0])
@pytest.mark.parametrize("kernel", KERNELS)
def test_attention_shared_scales_that_are_not_positive(ops, kernel, scale):
    dtype, heads, groups = KERNELS[kernel]
    case = shared_case(groups, [40], heads, 16, dtype, seed=62, pad=1)
    H, KV, D = heads
    out = ops.paged_attention_shared(case.q, H, KV, D, scale, case.cache, case.ctx)
    ops.check_status()
    assert not check_numbers(case, out, dtype, scale)
    assert (out[len(case.k):] == 0).all()


@pytest.mark.parametrize("heads,page", [((8, 2, 40), 16), ((4, 4, 8), 8), ((4, 2, 48), 5), ((12, 4, 104), 16), ((6, 1, 120), 64), ((3, 3, 136), 16), ((8, 2, 200), 32)])
@pytest.mark.parametrize("shape", [[(300, [90, 1, 70]), (5, [1])], [(70, [5, 20, 9])], [(1000, [3] * 24)]])
def test_attention_shared_holds_weights_as_paged_attention_does(ops, heads, page, shape):
    """Heads whose softmax weights ``paged_attention`` holds in more than bfloat16's 8 bits: so do these, and what a result is off by is
    its own rounding."""
    case = shared_case(shape, [40], heads, page, BF16, seed=63)
    H, KV, D = heads
    out = run_attention(ops, case)
    for r, (k, v) in enumerate(zip(case.k, case.v)):
        want, size = plain_beam.attention_row(case.q[r, : H * D].cpu().reshape(H, D), k, v, D ** -0.5)
        # a weight as two bfloat16 numbers: half a step of half a step, 2^-16 of it; 32-bit sums (see check_attention); half a step of
        # the result
        tol = (2.0 ** -16 + 20 * math.sqrt(D) * 2.0 ** -24) * size + 2.0 ** -8 * want.abs() + 1e-6
        bad = (out[r].double().cpu().reshape(H, D) - want).abs() / tol
        assert (bad <= 1).all(), (r, float(bad.max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("groups", [[(20, [1 + i % 3 for i in range(64)])] * 64, [(300, [1 + i % 5 for i in range(32)])] * 32])
def test_attention_shared_of_some_thousand_rows(ops, dtype, groups):
    case = shared_case(groups, [7], (4, 2, 16), 16, dtype, seed=64, pad=3)
    out = run_attention(ops, case)
    check_attention(case, out, dtype)


@pytest.mark.parametrize("kernel", KERNELS)
def test_attention_shared_of_one_request_in_several_rows(ops, kernel):
    """Rows of the same request, at the same position and at others: each sees the keys up to its own."""
    dtype, heads, groups = KERNELS[kernel]
    case = shared_case(groups, [40], heads, 16, dtype, seed=65)
    for r, of, n in ((1, 0, case.k[0].shape[1]), (2, 0, case.k[0].shape[1] - 4)):
        if r < len(groups[0][1]):
            case.ctx.token_request[r], case.ctx.positions[r] = int(case.ctx.token_request[of]), n - 1
            case.k[r], case.v[r] = case.k[of][:, :n], case.v[of][:, :n]
    assert not check_numbers(case, run_attention(ops, case), dtype)


def test_attention_and_choice_on_two_streams_at_once(ops):
    """Calls that overlap on the GPU share nothing."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = [shared_case([(900, [90, 1, 70] * 14)], [400], (8, 8, 64), 16, BF16, seed=66 + i) for i in range(2)]
    gen = torch.Generator().manual_seed(8)
    logits, scores = [torch.randn(32, 9000, generator=gen) for _ in range(2)], -3 * torch.rand(4, 8, generator=gen)
    on_device, first, outs = [x.cuda() for x in logits], scores.cuda(), [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append((run_attention(ops, cases[i]), ops.beam_select(on_device[i], first, 8)))
    torch.cuda.synchronize()
    ops.check_status()
    for case, mine, x in zip(cases, outs, logits):
        check_attention(case, mine[0][0], BF16)
        check_choice(mine[0][1], plain_beam.beam_select(x, scores, 8), 4, 8)
        for out, choice in mine[1:]:
            assert torch.equal(out, mine[0][0])
            for name in ("tokens", "parents", "scores", "ranks"):
                assert torch.equal(getattr(choice, name), getattr(mine[0][1], name))


# ---- the choice of the next beams ------------------------------------------------------------------------
@pytest.mark.parametrize("offset", [-10000.0, -1000.0, 100.0, 1000.0, 10000.0])
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("rows", [(2, 3), (8, 16)])
def test_beam_select_of_large_logits(ops, rows, offset, certain):
    """A number added to all logits of a row changes no score, and no log probability is above zero."""
    gen = torch.Generator().manual_seed(7)
    groups, beams = rows
    vocab = 5000
    logits = torch.randn(groups * beams, vocab, generator=gen) * 2 + offset + torch.rand(groups * beams, 1, generator=gen)
    if certain:
        logits[torch.arange(groups * beams), torch.randint(0, vocab, (groups * beams,), generator=gen)] += 40.0
    scores = -3 * torch.rand(groups, beams, generator=gen)
    got = ops.beam_select(logits.cuda(), scores.cuda(), beams)
    want = plain_beam.beam_select(logits, scores, beams)
    check_choice(got, want, groups, beams)                                 # (its tolerance knows nothing of the offset)
    parents = got.parents.long().cpu()
    assert (got.scores.cpu().reshape(-1) <= scores.reshape(-1)[parents]).all()


# ---- a step's integers, where kernels overlap -------------------------------------------------------------
@pytest.mark.parametrize("R", [3, 700])
def test_step_tables_are_whole_before_what_reads_them(ops, R):
    """Captured with overlapping launches, attention directly behind the step's integers (which it reads before it waits for what is in
    front of it): every replay sees those of its own lengths."""
    H, D, page, width = 4, 64, 16, 12
    gen = torch.Generator().manual_seed(R)
    pool = torch.randperm(R * width, generator=gen).to(torch.int32).reshape(R, width).cuda()
    k, v = (torch.randn(R * width, H, page, D, generator=gen).to(BF16).cuda() for _ in range(2))
    q = torch.randn(R, 3 * H * D, generator=gen).to(BF16).cuda()
    before, ones = i32([5] * R), torch.ones(R, dtype=torch.int32, device="cuda")
    cache = SimpleNamespace(k_pages=k, v_pages=v, group=0, page_tokens=page, window=None, writes=False, values_in_keys=False, keep_first=0)

    def step():
        t = ops.step_tables([pool], [page], before, ones, R)
        ctx = SimpleNamespace(block_tables=t.block_tables, token_request=t.token_request, positions=t.positions, decode_only=True,
                              extra={}, max_ctx_after=page * width)
        return ops.paged_attention(q, H, H, D, D ** -0.5, cache, ctx)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    ops.set_dependent_launch(True)
    try:
        with torch.cuda.graph(graph):
            out = step()
    finally:
        ops.set_dependent_launch(False)
    for seed in range(4):
        lengths = torch.randint(0, page * width - 1, (R,), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        before.copy_(lengths)
        graph.replay()
        torch.cuda.synchronize()
        for r in range(0, R, max(1, R // 40)):
            n = int(lengths[r]) + 1
            pages = pool[r, : -(-n // page)].long()
            mine = [x[pages].transpose(0, 1).reshape(H, -1, D)[:, :n].cpu() for x in (k, v)]
            want, size = plain_beam.attention_row(q[r, : H * D].cpu().reshape(H, D), *mine, D ** -0.5)
            # (see test_gpu_beam.check_attention)
            tol = 20 * math.sqrt(D) * 2.0 ** -24 * size + 1e-6 + 2.0 ** -8 * (size + want.abs())
            assert ((out[r].double().cpu().reshape(H, D) - want).abs() <= tol).all(), (seed, r)
