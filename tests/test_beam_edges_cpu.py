"""Beam search at the edge of what its parameters allow, on the plain-torch kernel set, and refusals made on the host."""

from __future__ import annotations

import math

import pytest
import torch

import plain_beam
from test_beam_cpu import ops  # noqa: F401
from test_beam_search_cpu import engine_for

from mini_gpt_inference_b200 import BeamParams
from mini_gpt_inference_b200.engine.runner import StepError
from mini_gpt_inference_b200.kernels.library import KernelLibraryError


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
