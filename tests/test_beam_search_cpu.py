"""Beam search through the entry point on the plain-torch kernel set, against a search one hypothesis at a time; and forks
of a request in the cache manager."""

from __future__ import annotations

import random

import pytest

import beam_search_cases
import plain_beam
from beam_torch_ops import BeamTorchOps

from mini_gpt_inference_b200 import BeamParams, EngineConfig, LLMEngine, SamplingParams
from mini_gpt_inference_b200.cache import CacheFullError, CacheManager, FixedStateSpec, PagedKVSpec, PoolError


def engine_for(which, **more):
    cfg = dict(block_size=8, num_blocks=128, max_batch_size=12, max_num_batched_tokens=16, dtype="float32", device="cpu")
    loaded, last, tokens, vocab = beam_search_cases.model(which, "float32", "cpu")
    return LLMEngine(loaded, EngineConfig(**{**cfg, **more}), ops=BeamTorchOps()), last, tokens, vocab


def check(found, want, penalty):
    assert [h["token_ids"] for h in found] == [ids for ids, _, _ in want]
    for h, (ids, logprob, over) in zip(found, want):
        assert h["logprob"] == pytest.approx(logprob, abs=2e-4)
        assert h["score"] == pytest.approx(logprob / len(ids) ** penalty, abs=2e-4)
        assert h["finish_reason"] == ("eot" if over else "length")


@pytest.mark.parametrize("which", ["A", "B", *beam_search_cases.OTHERS])
def test_beam_search_matches_the_plain_one(which):
    engine, last, tokens, vocab = engine_for(which)
    prompts = [tokens(n, 30 + n) for n in (5, 17, 8)]
    found = engine.beam_search(prompts, BeamParams(beams=4, max_tokens=6))
    for prompt, mine in zip(prompts, found):
        check(mine, plain_beam.search(last, prompt, 4, 6), 0.0)
    stats = engine.stats()
    assert stats["allocated_blocks"] == 0 and stats["free_state_slots"] == 12
    engine.runner.manager.check()


def test_beam_search_ends_with_a_penalty_and_a_limit():
    engine, last, tokens, vocab = engine_for("A")
    engine.sampler.vocab_limit = 200
    prompt = tokens(9, 3)
    # the second token of the best continuation ends one
    end = plain_beam.search(last, prompt, 3, 2, vocab_limit=200)[0][0][1]
    for penalty in (0.0, 1.0):
        found = engine.beam_search([prompt], BeamParams(beams=3, max_tokens=7, length_penalty=penalty), eot_token_id=end)[0]
        check(found, plain_beam.search(last, prompt, 3, 7, penalty, end, 200), penalty)
        if penalty == 0.0:                                                  # (per token a longer one may win)
            assert any(h["finish_reason"] == "eot" for h in found)


def test_one_beam_is_greedy_and_one_token_a_choice():
    engine, last, tokens, vocab = engine_for("B")
    prompt = tokens(11, 4)
    greedy = engine.generate([prompt], SamplingParams(max_tokens=5, temperature=0.0))[0]["token_ids"]
    assert engine.beam_search([prompt], BeamParams(beams=1, max_tokens=5))[0][0]["token_ids"] == greedy
    check(engine.beam_search([prompt], BeamParams(beams=4, max_tokens=1))[0], plain_beam.search(last, prompt, 4, 1), 0.0)


def test_refusals_leave_nothing_behind():
    engine, last, tokens, vocab = engine_for("A", num_blocks=6, max_batch_size=4)
    assert engine.beam_search([]) == []
    for prompts, params, end in (([[]], None, None), ([[vocab]], None, None), ([[1] * 60], BeamParams(max_tokens=9), None),
                                 ([[1]], BeamParams(max_tokens=2), vocab), ([[1]], BeamParams(max_tokens=2), -1)):
        with pytest.raises(ValueError):
            engine.beam_search(prompts, params, end)
    for bad in (dict(beams=0), dict(beams=33), dict(max_tokens=0), dict(length_penalty=float("inf"))):
        with pytest.raises(ValueError):
            BeamParams(**bad)
    with pytest.raises(CacheFullError):                                     # pages
        engine.beam_search([tokens(20, 1)], BeamParams(beams=4, max_tokens=30))
    with pytest.raises(CacheFullError):                                     # requests
        engine.beam_search([[1], [2]], BeamParams(beams=3, max_tokens=2))
    assert engine.stats()["allocated_blocks"] == 0 and engine.stats()["free_state_slots"] == 4
    engine.runner.manager.check()


def test_requests_that_run_keep_their_caches():
    from mini_gpt_inference_b200 import Request

    engine, last, tokens, vocab = engine_for("A")
    prompt = tokens(10, 8)
    alone = engine.generate([prompt], SamplingParams(max_tokens=8, temperature=0.0))[0]["token_ids"]
    engine.add_request(Request("r", prompt, SamplingParams(max_tokens=8, temperature=0.0)))
    got = [t for _ in range(3) for out in engine.step() for t in out.new_token_ids]
    engine.beam_search([tokens(5, 9)], BeamParams(beams=3, max_tokens=4))
    while engine.has_unfinished_requests():
        got += [t for out in engine.step() for t in out.new_token_ids]
    assert got == alone


# ---- forks in the cache manager ------------------------------------------------------------------------
def test_forks_share_full_pages_only():
    m = CacheManager([PagedKVSpec(2, 8), PagedKVSpec(1, 4, page_tokens=3), FixedStateSpec((4,))], 4, 20, 5)
    m.admit("p")
    assert m.reserve("p", 10)
    m.advance("p", 10)
    f = m.fork("f", "p")
    assert f.length == 10 and f.tables == [m.get("p").tables[0][:2], m.get("p").tables[1][:3]] and f.state_slot != m.get("p").state_slot
    assert f.capacity == 8
    used = m.groups[0].pool.num_used
    assert m.reserve("f", 13)
    assert m.groups[0].pool.num_used == used + 2 and len(f.tables[0]) == 4 and len(f.tables[1]) == 5
    assert not set(f.tables[0][2:]) & set(m.get("p").tables[0])
    m.check()
    m.stats()
    with pytest.raises(PoolError):
        m.release("p")                                                      # its pages are read by the fork
    with pytest.raises(PoolError):
        m.fork("g", "f")
    with pytest.raises(PoolError):
        m.fork("f", "p")
    m.release("f")
    m.release("p")
    m.check()
    assert m.stats()["allocated_blocks"] == 0


def test_a_window_gives_back_no_page_that_forks_read():
    m = CacheManager([PagedKVSpec(1, 4, window=4)], 2, 40, 4)
    m.admit("p")
    assert m.reserve("p", 9)
    m.advance("p", 9)
    f = m.fork("f", "p")
    assert m.reserve("f", 14) and m.reserve("p", 14)
    held = list(m.get("p").tables[0])
    m.advance("p", 14)
    assert m.get("p").tables[0] == held
    m.advance("f", 14)
    m.check()
    assert f.tables[0][: f.shared[0]] == held[: f.shared[0]]
    m.release("f")
    m.release("p")
    assert m.stats()["allocated_blocks"] == 0


@pytest.mark.parametrize("seed", range(4))
def test_random_forks_keep_the_pools_whole(seed):
    rng = random.Random(seed)
    m = CacheManager([PagedKVSpec(1, 4), PagedKVSpec(2, 4, page_tokens=5)], 3, 60, 9)
    free = m.stats()["free_blocks"]
    for step in range(200):
        ids = list(m.requests)
        act = rng.random()
        if act < 0.3 and m.slots.num_free:
            m.admit(f"r{step}")
        elif act < 0.5 and ids and m.slots.num_free:
            parent = rng.choice(ids)
            if m.get(parent).parent is None:
                m.fork(f"f{step}", parent)
        elif act < 0.8 and ids:
            name = rng.choice(ids)
            if m.get(name).forks == 0:
                n = m.get(name).length + rng.randint(1, 9)
                if m.reserve(name, n):
                    m.advance(name, n)
        elif ids:
            name = rng.choice(ids)
            if m.get(name).forks == 0:
                m.release(name)
        m.check()
    for name in sorted(m.requests, key=lambda n: m.get(n).parent is None):
        m.release(name)
    assert m.stats()["free_blocks"] == free
