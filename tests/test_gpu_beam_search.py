"""Beam search on the GPU through the entry point: all of its kernels together, step after step, replayed from graphs."""

from __future__ import annotations

import math

import pytest
import torch

import beam_search_cases
import plain_beam

from mini_gpt_inference_b200 import BeamParams, EngineConfig, LLMEngine, Request, SamplingParams

pytestmark = pytest.mark.gpu


def engine_for(which, dtype, **more):
    cfg = dict(block_size=8, num_blocks=512, max_batch_size=40, max_num_batched_tokens=32, dtype=dtype, device="cuda:0")
    loaded, last, tokens, vocab = beam_search_cases.model(which, dtype, "cuda:0")
    return LLMEngine(loaded, EngineConfig(**{**cfg, **more})), last, tokens, vocab


def check(found, want, penalty=0.0):
    assert [h["token_ids"] for h in found] == [ids for ids, _, _ in want]
    for h, (ids, logprob, over) in zip(found, want):
        # a log probability a token: 32-bit logits, off by 2e-5 at most (see the harness)
        assert h["logprob"] == pytest.approx(logprob, abs=5e-5 * len(ids))
        assert h["finish_reason"] == ("eot" if over else "length")


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("which", ["A", "B"])
def test_beam_search_in_32_bits_matches_the_plain_one(which, graphs):
    engine, last, tokens, vocab = engine_for(which, "float32", use_cuda_graphs=graphs)
    for prompts, beams, made in (([tokens(n, 30 + n) for n in (5, 17, 8)], 4, 12), ([tokens(20, 3)], 7, 9), ([tokens(n, n) for n in (9, 16)], 4, 1)):
        found = engine.beam_search(prompts, BeamParams(beams=beams, max_tokens=made))
        for prompt, mine in zip(prompts, found):
            check(mine, plain_beam.search(last, prompt, beams, made))
    assert engine.stats()["allocated_blocks"] == 0
    engine.runner.manager.check()


def test_captured_steps_serve_later_searches():
    """The second search of a shape replays the first one's graph, with other prompts, lengths, pages and slots."""
    engine, last, tokens, vocab = engine_for("A", "float32")
    other = Request("held", tokens(9, 77), SamplingParams(max_tokens=4, temperature=0.0))
    params = BeamParams(beams=3, max_tokens=10)
    for round_ in range(3):
        prompts = [tokens(n, 100 * round_ + n) for n in (13 + round_, 9, 16)]
        found = engine.beam_search(prompts, params)
        for prompt, mine in zip(prompts, found):
            check(mine, plain_beam.search(last, prompt, 3, 10))
        if round_ == 0:
            engine.add_request(other)                                       # takes pages and a slot from now on
            engine.step()
    assert len(engine._beam_search._steps) == 1 and next(iter(engine._beam_search._steps.values())).graph is not None
    while engine.has_unfinished_requests():
        engine.step()
    engine.runner.manager.check()


def test_beam_search_ends():
    engine, last, tokens, vocab = engine_for("A", "float32")
    prompt = tokens(9, 3)
    end = plain_beam.search(last, prompt, 3, 2)[0][0][1]
    for penalty in (0.0, 1.0):
        found = engine.beam_search([prompt, tokens(5, 5)], BeamParams(beams=3, max_tokens=40, length_penalty=penalty), eot_token_id=end)
        check(found[0], plain_beam.search(last, prompt, 3, 40, penalty, end), penalty)


@pytest.mark.parametrize("which", beam_search_cases.OTHERS)
def test_beam_search_of_models_with_states_and_windows(which):
    """Matrix memories, convolutions, retention, windows, latents: in 32 bits the continuations of the plain search, or (where two are
    closer than rounding) ones whose log probabilities are as good."""
    engine, last, tokens, vocab = engine_for(which, "float32")
    prompts = [tokens(n, 40 + n) for n in (6, 19)]
    found = engine.beam_search(prompts, BeamParams(beams=4, max_tokens=9))
    for prompt, mine in zip(prompts, found):
        want = plain_beam.search(last, prompt, 4, 9)
        assert len(mine) == 4 and len({tuple(h["token_ids"]) for h in mine}) == 4
        for h, (ids, logprob, _) in zip(mine, want):
            assert h["logprob"] == pytest.approx(logprob, abs=3e-3)
            x = [torch.log_softmax(last(prompt + h["token_ids"][:t]).double(), -1)[h["token_ids"][t]] for t in range(9)]
            assert h["logprob"] == pytest.approx(float(sum(x)), abs=3e-3)
    engine.runner.manager.check()


@pytest.mark.parametrize("which", ["A", "B"])
def test_beam_search_in_bfloat16(which):
    """Every continuation has the log probability that the plain model (same weights) gives it, within what bfloat16 activations move
    a logit (the harness's tolerance, twice a token: the logit and the sum it is measured against); best first, all different."""
    engine, last, tokens, vocab = engine_for(which, "bfloat16")
    prompts = [tokens(n, 50 + n) for n in (21, 6)]
    found = engine.beam_search(prompts, BeamParams(beams=5, max_tokens=10))
    for prompt, mine in zip(prompts, found):
        assert len({tuple(h["token_ids"]) for h in mine}) == 5
        assert [h["logprob"] for h in mine] == sorted((h["logprob"] for h in mine), reverse=True)
        for h in mine:
            x = [torch.log_softmax(last(prompt + h["token_ids"][:t]).double(), -1)[h["token_ids"][t]] for t in range(10)]
            assert h["logprob"] == pytest.approx(float(sum(x)), abs=10 * 2 * 8e-3)


def test_beams_of_heads_and_rows_that_the_tiles_take():
    """Heads of 64, 32 beams a prompt of 300 tokens: the shared pages go through the tensor-core tiles; the result is that of rows that
    share nothing."""
    from mini_gpt_inference_b200 import GPTConfig
    from mini_gpt_inference_b200.engine.build import load_model
    from harness import make_tensors

    cfg = GPTConfig.from_dict(dict(vocab_size=600, n_positions=512, n_layer=2, n_head=4, n_embd=256, n_inner=512, bias=True,
                                   layer_norm_epsilon=1e-5))
    tensors = make_tensors(cfg, 9, "bfloat16", sharp=True)
    found = []
    for shared in (True, False):
        engine = LLMEngine(load_model(config=cfg, tensors=tensors, dtype="bfloat16", device="cuda:0"),
                           EngineConfig(block_size=16, num_blocks=2048, max_batch_size=128, dtype="bfloat16"))
        gen = torch.Generator().manual_seed(4)
        prompts = [torch.randint(0, 600, (n,), generator=gen).tolist() for n in (300, 411)]
        if not shared:
            from mini_gpt_inference_b200.engine import beam_search

            keep = beam_search.SharedPrefix
            beam_search.SharedPrefix = lambda *a: None
        try:
            found.append(engine.beam_search(prompts, BeamParams(beams=32, max_tokens=12)))
        finally:
            if not shared:
                beam_search.SharedPrefix = keep
    for with_tiles, without in zip(*found):
        # two roundings of the same numbers: the best ones' log probabilities agree to what bfloat16 moves them
        for a, b in zip(with_tiles, without):
            assert a["logprob"] == pytest.approx(b["logprob"], abs=12 * 2 * 8e-3)
        assert math.isfinite(with_tiles[-1]["logprob"])


def test_beam_search_by_the_command_line(tmp_path):
    import json
    import subprocess
    import sys
    from pathlib import Path

    from harness import make_model_dir, tokens_for
    import plain_gpt

    folder, cfg, tensors = make_model_dir(tmp_path, "A", 31, "float32")
    prompt = tokens_for(cfg, 9, 4)
    cmd = [sys.executable, str(Path(__file__).resolve().parent.parent / "bin" / "generate"), "--model", str(folder), "--prompt-ids",
           ",".join(map(str, prompt)), "--beams", "3", "--max-new-tokens", "6", "--dtype", "float32", "--kv-block-size", "8",
           "--num-kv-blocks", "64"]
    proc = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0, proc.stderr[-2000:]
    out = json.loads([line for line in proc.stdout.splitlines() if line.startswith("{")][0])
    last = lambda tokens: plain_gpt.forward_logits(tokens, tensors, cfg.n_layer, cfg.n_head, cfg.layer_norm_epsilon)[-1]  # noqa: E731
    check(out["beams"], plain_beam.search(last, prompt, 3, 6))


def test_a_search_of_few_tokens_keeps_the_captured_step():
    """Searches of too few tokens to be captured replay a step that is, and leave it to those that follow."""
    engine, last, tokens, vocab = engine_for("A", "float32")
    graphs = []
    for made in (8, 5, 8):
        prompt = tokens(14, 90 + made)
        check(engine.beam_search([prompt], BeamParams(beams=3, max_tokens=made))[0], plain_beam.search(last, prompt, 3, made))
        graphs.append([s.graph for s in engine._beam_search._steps.values()])
    assert len(graphs[0]) == 1 and graphs[0] == graphs[1] == graphs[2]
