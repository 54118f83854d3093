"""Beam search at the edge of what its parameters allow, on the plain-torch kernel set, and refusals made on the host."""

from __future__ import annotations

import math

import pytest
import torch

import fakilorn_cases
import plain_beam
from beam_torch_ops import BeamTorchOps
from test_beam_cpu import ops  # noqa: F401
from test_beam_search_cpu import engine_for

from mini_gpt_inference_b200 import BeamParams, EngineConfig, FakilornConfig, LLMEngine
from mini_gpt_inference_b200.engine.build import load_model
from mini_gpt_inference_b200.engine.runner import StepError
from mini_gpt_inference_b200.kernels.library import KernelLibraryError
from mini_gpt_inference_b200.kernels.ops import BeamChoice


def fakilorn_engine(which, device, ops=None):
    raw = fakilorn_cases.config(which)
    tensors = fakilorn_cases.random_weights(raw, 7, torch.float32)
    engine = LLMEngine(load_model(config=FakilornConfig.from_dict(raw), tensors=tensors, dtype="float32", device=device),
                       EngineConfig(block_size=8, num_blocks=256, max_batch_size=12, max_num_batched_tokens=16, dtype="float32", device=device),
                       ops=ops)
    return engine, lambda tokens: fakilorn_cases.plain_logits(raw, tensors, tokens)[-1], lambda n, seed: fakilorn_cases.tokens_for(raw, n, seed)


@pytest.mark.parametrize("penalty", [-16.0, -3.5, 16.0])
def test_length_penalties_up_to_the_bound(penalty):
    engine, last, tokens, vocab = engine_for("A")
    prompt = tokens(9, 3)
    found = engine.beam_search([prompt], BeamParams(beams=3, max_tokens=12, length_penalty=penalty))[0]
    want = plain_beam.search(last, prompt, 3, 12, penalty)
    assert [h["token_ids"] for h in found] == [ids for ids, _, _ in want]
    for h, (ids, logprob, _) in zip(found, want):
        assert h["score"] == pytest.approx(logprob / 12.0 ** penalty, rel=1e-4)
    # the longest continuation that there can be still has a value to be ranked by
    assert math.isfinite(1.0 / float(2 ** 31) ** penalty) and 1e-9 / float(2 ** 31) ** penalty != 0.0


@pytest.mark.parametrize("penalty", [16.01, -17.0, 700.0, -800.0, math.inf, math.nan])
def test_length_penalties_beyond_the_bound_are_refused(ops, penalty):  # noqa: F811
    with pytest.raises(ValueError, match="length_penalty"):
        BeamParams(length_penalty=penalty)
    logits, lengths = torch.zeros(6, 50), torch.zeros(6, dtype=torch.int32)
    with pytest.raises(KernelLibraryError, match="length penalty"):
        ops.beam_select(logits, torch.zeros(2, 3), 3, lengths=lengths, length_penalty=penalty)


@pytest.mark.parametrize("value", [math.nan, -math.inf, math.inf])
def test_a_model_without_log_probabilities_is_told(value, monkeypatch):
    """A prompt none of whose continuations has a log probability is an error, not a prompt without continuations; nothing stays
    behind, and the next search is as ever."""
    engine, last, tokens, vocab = engine_for("A")
    prompts = [tokens(9, 3), tokens(5, 4)]
    forward = engine.runner._forward

    def broken(ctx):
        logits = forward(ctx)
        if logits is not None:
            logits[-1] = value
        return logits

    monkeypatch.setattr(engine.runner, "_forward", broken)
    with pytest.raises(StepError, match="prompt 1"):
        engine.beam_search(prompts, BeamParams(beams=3, max_tokens=1))
    with pytest.raises(StepError, match="prompt 0"):
        engine.beam_search(prompts[:1], BeamParams(beams=1, max_tokens=4))
    assert engine.stats()["allocated_blocks"] == 0
    monkeypatch.setattr(engine.runner, "_forward", forward)
    found = engine.beam_search(prompts[:1], BeamParams(beams=3, max_tokens=4))[0]
    assert [h["token_ids"] for h in found] == [ids for ids, _, _ in plain_beam.search(last, prompts[0], 3, 4)]


def test_outputs_of_a_choice_that_lie_in_its_inputs_are_refused(ops):  # noqa: F811
    """In place only where rows stay rows: as many beams before as after, and the same tensor, not a part of it."""
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731

    def call(beams, in_beams, replace):
        scores, ended, lengths = torch.zeros(2, in_beams), i32(2 * in_beams), i32(2 * in_beams)
        logits, big = torch.zeros(2 * in_beams, 50), i32(100)
        given = dict(scores=scores, ended=ended, lengths=lengths, logits=logits.view(torch.int32).reshape(-1), big=big)
        n = 2 * beams
        out = dict(tokens=i32(n), parents=i32(n), scores=torch.zeros(2, beams), ranks=i32(n), ended=i32(n), lengths=i32(n))
        out.update(replace(given, n))
        ops.beam_select(logits, scores, beams, ended=ended, lengths=lengths, end_token=1, out=BeamChoice(**out))

    bad = [
        (4, 2, lambda g, n: dict(tokens=g["logits"][:n])),
        (3, 3, lambda g, n: dict(parents=g["logits"][4:4 + n])),
        (3, 3, lambda g, n: dict(tokens=g["big"][:n], parents=g["big"][2:2 + n])),
        (3, 3, lambda g, n: dict(tokens=g["big"][:n], ranks=g["big"][:n])),
        (3, 3, lambda g, n: dict(tokens=g["lengths"], parents=g["lengths"])),
    ]
    for beams, in_beams, replace in bad:
        with pytest.raises(KernelLibraryError, match="memory"):
            call(beams, in_beams, replace)
    # views that overlap an input by a part, and an input of other rows: one allocation for both
    for beams, in_beams, shift in ((3, 3, 1), (3, 3, -1), (4, 2, 0)):
        both = i32(64)
        ended, lengths = both[8: 8 + 2 * in_beams], i32(2 * in_beams)
        out = BeamChoice(i32(2 * beams), i32(2 * beams), torch.zeros(2, beams), i32(2 * beams), both[8 + shift: 8 + shift + 2 * beams], i32(2 * beams))
        with pytest.raises(KernelLibraryError, match="memory"):
            ops.beam_select(torch.zeros(2 * in_beams, 50), torch.zeros(2, in_beams), beams, ended=ended, lengths=lengths, end_token=1, out=out)
    with pytest.raises(AssertionError, match="mg_beam_select was reached"):      # in place: as the search calls it
        call(3, 3, lambda g, n: dict(scores=g["scores"], ended=g["ended"], lengths=g["lengths"]))


@pytest.mark.parametrize("which", ["A", "B", "C", "D"])
def test_beam_search_of_the_architecture_with_a_blending_chain(which):
    """Fakilorn: values blended from layer to layer, experts, a state of token pairs."""
    engine, last, tokens = fakilorn_engine(which, "cpu", BeamTorchOps())
    prompts = [tokens(n, 30 + n) for n in (5, 17)]
    found = engine.beam_search(prompts, BeamParams(beams=4, max_tokens=6))
    for prompt, mine in zip(prompts, found):
        want = plain_beam.search(last, prompt, 4, 6)
        assert [h["token_ids"] for h in mine] == [ids for ids, _, _ in want]
        for h, (_, logprob, _) in zip(mine, want):
            assert h["logprob"] == pytest.approx(logprob, abs=2e-4)
    engine.runner.manager.check()
