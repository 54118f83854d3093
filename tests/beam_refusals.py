"""Calls of the beam search's kernels that have to be refused, on tensors of any device: none of them reaches a launch."""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

from mini_gpt_inference_b200.kernels.ops import BeamChoice
from mini_gpt_inference_b200.parts.context import SharedPrefix


def calls(ops, device):
    f32 = lambda *shape: torch.zeros(*shape, device=device)  # noqa: E731
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=device)  # noqa: E731
    logits, scores = f32(6, 50), f32(2, 3)

    def select(**more):
        args = dict(logits=logits, scores=scores, beams=3)
        args.update(more)
        return lambda: ops.beam_select(**args)

    yield "logits of 16 bits", select(logits=logits.to(torch.bfloat16))
    yield "rows that do not fit the scores", select(logits=f32(5, 50))
    yield "more beams before than after", select(beams=2)
    yield "too many beams", select(beams=33)
    yield "no beams", select(beams=0)
    yield "fewer ids than beams", select(vocab_limit=2)
    yield "strided logits", select(logits=f32(6, 100)[:, ::2])
    yield "a penalty without lengths", select(length_penalty=0.5)
    yield "a penalty that is no number", select(length_penalty=math.nan, lengths=i32(6))
    yield "ended beams without an end", select(ended=i32(6))
    yield "ended beams of another number", select(ended=i32(5), end_token=1)
    yield "lengths of 64 bits", select(lengths=i32(6).long())
    yield "an end outside the vocabulary", select(end_token=50)
    yield "an end at the limit", select(end_token=40, vocab_limit=40)
    yield "an end below zero", select(end_token=-1)
    choice = lambda **m: BeamChoice(**{**dict(tokens=i32(6), parents=i32(6), scores=f32(2, 3), ranks=i32(6)), **m})  # noqa: E731
    yield "no room for the ended", select(end_token=1, out=choice())
    yield "no room for the lengths", select(lengths=i32(6), out=choice())
    yield "room for too few tokens", select(out=choice(tokens=i32(5)))
    yield "scores of another shape", select(out=choice(scores=f32(3, 2)))

    def reorder(**more):
        args = dict(parents=i32(4), lengths=i32(4), block_tables=[i32(4, 3)], k_pages=[f32(2, 5, 1, 4, 8)], v_pages=[f32(2, 5, 1, 4, 8)])
        args.update(more)
        return lambda: ops.beam_reorder(**args)

    yield "lengths of another number", reorder(lengths=i32(3))
    yield "a table of another number of rows", reorder(block_tables=[i32(3, 3)])
    yield "keys without values", reorder(v_pages=[])
    yield "values of another type", reorder(v_pages=[f32(2, 5, 1, 4, 8).to(torch.bfloat16)])
    yield "values of other pages", reorder(v_pages=[f32(2, 6, 1, 4, 8)])
    yield "strided keys", reorder(k_pages=[f32(2, 5, 1, 4, 16)[..., ::2]])
    yield "parents of 64 bits", reorder(parents=i32(4).long())
    yield "states without slots", reorder(states=[f32(5, 3)])
    yield "too few slots", reorder(states=[f32(5, 3)], slots=i32(3))
    yield "a state of no slots", reorder(states=[f32(0, 3)], slots=i32(4))

    def tables(**more):
        args = dict(pages=[i32(4, 3)], page_tokens=[16], ctx_before=i32(4), q_len=i32(4), num_tokens=4)
        args.update(more)
        return lambda: ops.step_tables(**args)

    yield "no requests", tables(ctx_before=i32(0), q_len=i32(0))
    yield "lengths that do not match", tables(q_len=i32(3))
    yield "rows that do not match", tables(rows=i32(3))
    yield "too few rows of pages", tables(ctx_before=i32(5), q_len=i32(5))
    yield "a page of no tokens", tables(page_tokens=[0])
    yield "no page size", tables(page_tokens=[])
    yield "pools of other rows", tables(pages=[i32(4, 3), i32(5, 3)], page_tokens=[16, 16])
    yield "a pool of no columns", tables(pages=[i32(4, 0)])
    yield "fewer than no tokens", tables(num_tokens=-1)

    def attention(heads=(4, 2, 8), q=None, cache=None, ctx=None, **prefix):
        shared = dict(groups=i32(1, 3), max_rows=1, max_tokens=1, max_behind=1)
        shared.update(prefix)
        view = dict(k_pages=f32(5, 2, 4, 8), v_pages=f32(5, 2, 4, 8), group=0, page_tokens=4, window=None, values_in_keys=False)
        view.update(cache or {})
        more = dict(block_tables=[i32(3, 2)], token_request=i32(3), positions=i32(3), shared_prefix=SharedPrefix(**shared))
        more.update(ctx or {})
        return lambda: ops.paged_attention_shared(f32(3, 64) if q is None else q, *heads, 1.0, SimpleNamespace(**view), SimpleNamespace(**more))

    yield "queries of another type", attention(q=f32(3, 64).to(torch.bfloat16))
    yield "heads of half precision", attention(q=f32(3, 64).half(), cache=dict(k_pages=f32(5, 2, 4, 8).half(), v_pages=f32(5, 2, 4, 8).half()))
    yield "rows too narrow", attention(q=f32(3, 31))
    yield "heads that do not share evenly", attention(heads=(3, 2, 8))
    yield "pages of other heads", attention(heads=(4, 4, 8))
    yield "values of another size", attention(cache=dict(v_pages=f32(5, 2, 4, 4)))
    yield "a window", attention(cache=dict(window=8))
    yield "values in the keys", attention(cache=dict(values_in_keys=True))
    yield "too few positions", attention(ctx=dict(positions=i32(2)))
    yield "too few requests", attention(ctx=dict(token_request=i32(2)))
    yield "no groups at all", attention(ctx=dict(shared_prefix=None))
    yield "groups of two numbers", attention(groups=i32(1, 2))
    yield "no rows", attention(max_rows=0)
    yield "no keys behind", attention(max_behind=0)
    yield "tokens below zero", attention(max_tokens=-1)
