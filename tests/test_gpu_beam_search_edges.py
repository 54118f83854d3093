"""Beam search on the GPU beside other requests, over the architecture with a blending chain, and through the tensor-core tiles
inside a captured step."""

from __future__ import annotations

import pytest
import torch

import plain_beam
import plain_gpt
from harness import make_tensors
from test_beam_edges_cpu import fakilorn_engine
from test_gpu_beam import BF16, check_attention, i32, shared_case
from test_gpu_beam_search import engine_for

from mini_gpt_inference_b200 import BeamParams, EngineConfig, GPTConfig, LLMEngine, Request, SamplingParams
from mini_gpt_inference_b200.engine.build import load_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["A", "B", "D"])
def test_beam_search_of_the_architecture_with_a_blending_chain(which):
    engine, last, tokens = fakilorn_engine(which, "cuda:0")
    prompts = [tokens(n, 40 + n) for n in (6, 19)]
    found = engine.beam_search(prompts, BeamParams(beams=4, max_tokens=9))
    for prompt, mine in zip(prompts, found):
        want = plain_beam.search(last, prompt, 4, 9)
        assert len(mine) == 4 and len({tuple(h["token_ids"]) for h in mine}) == 4
        for h, (_, logprob, _) in zip(mine, want):
            # (as for the other architectures: 32-bit logits of some ten layers' parts)
            assert h["logprob"] == pytest.approx(logprob, abs=3e-3)
            x = [torch.log_softmax(last(prompt + h["token_ids"][:t]).double(), -1)[h["token_ids"][t]] for t in range(9)]
            assert h["logprob"] == pytest.approx(float(sum(x)), abs=3e-3)
    engine.runner.manager.check()


@pytest.mark.parametrize("made", [4, 12])
def test_requests_in_flight_keep_their_tokens(made):
    """A search between the steps of requests that decode from a graph, their next tokens still on the device: they go on as if
    alone, and the search finds what it finds alone."""
    engine, last, tokens, vocab = engine_for("A", "float32")
    greedy = lambda n: SamplingParams(max_tokens=n, temperature=0.0)  # noqa: E731
    prompts = [tokens(10, 8), tokens(7, 9)]
    alone = [engine.generate([p], greedy(30))[0]["token_ids"] for p in prompts]
    got = {"0": [], "1": []}
    for name, p in zip(got, prompts):
        engine.add_request(Request(name, p, greedy(30)))

    def steps(n):
        for _ in range(n):
            for out in engine.step():
                got[out.request_id] += out.new_token_ids

    for round_ in range(3):
        steps(4)
        assert engine.num_overlapped_steps > 0                             # (tokens are in flight)
        prompt = tokens(11, 60 + round_)
        found = engine.beam_search([prompt], BeamParams(beams=3, max_tokens=made))[0]
        assert [h["token_ids"] for h in found] == [ids for ids, _, _ in plain_beam.search(last, prompt, 3, made)]
    while engine.has_unfinished_requests():
        steps(1)
    assert [got["0"], got["1"]] == alone
    engine.runner.manager.check()
    assert engine.stats()["allocated_blocks"] == 0


def test_continuations_through_the_tiles_have_the_plain_models_log_probabilities():
    """32 beams a prompt over heads of 64: every continuation's log probability is what the plain model (same weights) gives it."""
    cfg = GPTConfig.from_dict(dict(vocab_size=600, n_positions=512, n_layer=2, n_head=4, n_embd=256, n_inner=512, bias=True,
                                   layer_norm_epsilon=1e-5))
    tensors = make_tensors(cfg, 9, "bfloat16", sharp=True)
    engine = LLMEngine(load_model(config=cfg, tensors=tensors, dtype="bfloat16", device="cuda:0"),
                       EngineConfig(block_size=16, num_blocks=2048, max_batch_size=128, dtype="bfloat16"))
    gen = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 600, (n,), generator=gen).tolist() for n in (300, 411)]
    ops, launched = engine.runner.ops, []
    shared = ops.paged_attention_shared

    def counted(*args):
        before = ops.launches
        out = shared(*args)
        launched.append(ops.launches - before)
        return out

    ops.paged_attention_shared = counted
    try:
        found = engine.beam_search(prompts, BeamParams(beams=32, max_tokens=12))
    finally:
        del ops.paged_attention_shared
    assert launched and set(launched) == {3}                               # tiles, own ranges, joined
    for prompt, mine in zip(prompts, found):
        assert len({tuple(h["token_ids"]) for h in mine}) == 32
        assert [h["logprob"] for h in mine] == sorted((h["logprob"] for h in mine), reverse=True)
        for h in mine:
            ids = h["token_ids"]
            logits = plain_gpt.forward_logits(prompt + ids, tensors, cfg.n_layer, cfg.n_head, cfg.layer_norm_epsilon)
            x = torch.log_softmax(logits[len(prompt) - 1: -1].double(), -1)
            # what bfloat16 activations move a logit, twice a token: the logit and the sum it is measured against
            assert h["logprob"] == pytest.approx(float(x[range(12), ids].sum()), abs=12 * 2 * 8e-3)


@pytest.mark.parametrize("heads,rows", [((8, 8, 64), 45), ((32, 8, 128), 9)])
def test_tiles_behind_a_projection_in_a_captured_step(heads, rows):
    """Projection, tiles, own ranges that start early, joined, projection: captured with overlapping launches and replayed with other
    lengths, groups and activations; every row against 64 bits."""
    from mini_gpt_inference_b200.kernels.ops import default_ops

    ops = default_ops("cuda:0")
    H, KV, D = heads
    bounds = (rows, 700, 200)
    cases = [shared_case([(s, [1 + (7 * i) % b for i in range(rows)])], [90], heads, 16, BF16, seed=s, bounds=bounds, pool=20 + 44 + 15 * rows)
             for s, b in ((650, 190), (130, 200), (700, 3), (301, 120))]
    width, gen = 1 + max(c.ctx.block_tables[0].shape[1] for c in cases), torch.Generator().manual_seed(3)
    n, K = rows + 1, 256
    x = torch.empty(n, K, dtype=BF16, device="cuda")
    w = (torch.randn((H + 2 * KV) * D, K, generator=gen) * 2 / K ** 0.5).to(BF16).cuda()
    w2 = (torch.randn(K, H * D, generator=gen) / (H * D) ** 0.5).to(BF16).cuda()
    live = cases[0]
    live.ctx.block_tables = [torch.full((n, width), -1, dtype=torch.int32, device="cuda")]

    def step():
        q = ops.linear(x, w, None, "none", BF16)
        before = ops.launches
        out = ops.paged_attention(q, H, KV, D, D ** -0.5, live.cache, live.ctx)
        assert ops.launches - before == 3
        return q, out, ops.linear(out, w2, None, "none", torch.float32)

    def load(case, table, seed):
        x.copy_(torch.randn(n, K, generator=torch.Generator().manual_seed(seed)))
        live.ctx.block_tables[0].fill_(-1)
        live.ctx.block_tables[0][:, : table.shape[1]] = table
        if case is not live:
            live.ctx.token_request.copy_(case.ctx.token_request)
            live.ctx.positions.copy_(case.ctx.positions)
            live.ctx.shared_prefix.groups.copy_(case.ctx.shared_prefix.groups)
            live.cache.k_pages.copy_(case.cache.k_pages)
            live.cache.v_pages.copy_(case.cache.v_pages)

    tables = [c.ctx.block_tables[0].clone() for c in cases]
    first = shared_case([(650, [1 + (7 * i) % 190 for i in range(rows)])], [90], heads, 16, BF16, seed=650, bounds=bounds, pool=20 + 44 + 15 * rows)
    tables[0], cases[0] = first.ctx.block_tables[0], first
    load(first, tables[0], 0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    ops.set_dependent_launch(True)
    try:
        with torch.cuda.graph(graph):
            q, out, after = step()
    finally:
        ops.set_dependent_launch(False)
    for seed, (case, table) in enumerate(zip(cases, tables)):
        load(case, table, seed)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        ops.check_status()
        case.q = q
        check_attention(case, out, BF16)
        want = out.double() @ w2.double().T
        # 32-bit sums of H * D products of some 1 / sqrt(H * D) each
        assert (after.double() - want).abs().max() <= 1e-4
