"""The plain-torch kernel set with a beam search's kernels, for tests without a GPU."""

from __future__ import annotations

import torch

import plain_beam
from torch_ops import TorchOps

from mini_gpt_inference_b200.kernels.ops import BeamChoice, StepTables


class BeamTorchOps(TorchOps):
    def beam_select(self, logits, scores, beams, ended=None, lengths=None, end_token=None, length_penalty=0.0, vocab_limit=None,
                    out=None):
        want = plain_beam.beam_select(logits, scores, beams, ended, lengths, end_token, length_penalty, vocab_limit)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
        got = BeamChoice(i32(want["tokens"]), i32(want["parents"]), torch.tensor(want["scores"]).reshape(-1, beams).float(),
                         i32(want["ranks"]), i32(want["ended"]) if end_token is not None else None,
                         i32(want["lengths"]) if lengths is not None else None)
        if out is None:
            return got
        for name in ("tokens", "parents", "scores", "ranks", "ended", "lengths"):
            if getattr(out, name) is not None:
                getattr(out, name).copy_(getattr(got, name))
        return out

    def beam_reorder(self, parents, lengths, block_tables, k_pages, v_pages, slots=None, states=()):
        plain_beam.beam_reorder(parents, lengths, block_tables, k_pages,
                                [None if v is not None and v.data_ptr() == k.data_ptr() else v for k, v in zip(k_pages, v_pages)],
                                slots, states)

    def step_tables(self, pages, page_tokens, ctx_before, q_len, num_tokens, rows=None):
        request, positions, start, tables, slots = plain_beam.step_tables(pages, page_tokens, ctx_before, q_len, num_tokens, rows)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
        return StepTables(i32(request), i32(positions), i32(start), [i32(t) for t in tables], [i32(s) for s in slots],
                          ctx_before + q_len.clamp(min=0))
