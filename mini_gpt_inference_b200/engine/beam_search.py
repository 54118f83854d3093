"""Beam search over the engine's cache: every step of it stays on the device.

The prompts run through the step function once.  Then every prompt has ``beams`` requests, forks of the one that ran it:
they share the pages that the prompt has filled, and hold a page of their own for each column behind (so many that no
step has to take one).  A step is

    step_tables     positions, cache rows and block tables from the rows' lengths
    model           one token a row; attention reads the shared pages once per prompt
    beam_select     the next beams; one that goes on stays in its row
    beam_reorder    the rows that do not go on take over block tables, the tokens of the part-filled page, and states

with nothing for the host to decide: it is captured as a graph and replayed, and the host looks every few steps whether all
beams have ended.  Tokens and parents of all steps are kept on the device and followed back at the end.

(The reference has no beam search; its sampler draws one token a request, src/minigpt_infer/sampling.py:97-137.)
"""

from __future__ import annotations

import math

import torch

from ..cache.manager import NO_PAGE, CacheFullError
from ..config.engine_config import BeamParams
from ..kernels.ops import BeamChoice
from ..parts.context import SharedPrefix, StepContext
from .runner import ModelRunner, StepEntry, StepError, _no_collection


def _bucket(n: int, most: int) -> int:
    return min(most, 1 << max(0, n - 1).bit_length())


class _Step:
    """A step of a search of ``groups`` prompts and ``beams`` beams each: its tensors, its launches and their graph."""

    def __init__(self, runner: ModelRunner, groups: int, beams: int, longest_prompt: int, longest: int, max_tokens: int,
                 penalty: float, end: int | None, vocab_limit: int | None) -> None:
        self.runner, self.ops, self.groups, self.beams = runner, runner.ops, groups, beams
        self.penalty, self.end, self.vocab_limit, self.longest = penalty, end, vocab_limit, longest
        rows, device = groups * beams, runner.device
        m, storage = runner.manager, runner.storage
        zeros = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
        self.page_tokens = [g.page_tokens for g in m.groups]
        self.tables = [zeros(rows, width) for width in runner.max_pages]
        self.slots, self.lengths = zeros(rows), zeros(rows)
        self.ones = torch.ones(rows, dtype=torch.int32, device=device)
        self.logit_rows = torch.arange(rows, dtype=torch.int32, device=device)
        self.shared_groups = zeros(groups, 3)
        self.shared = SharedPrefix(self.shared_groups, beams, longest_prompt, max_tokens)
        # tokens, parents, ranks, ended, lengths and scores of the last choice
        self.buffer = zeros(6, rows)
        tokens, parents, ranks, ended, made, scores = self.buffer.unbind(0)
        self.choice = BeamChoice(tokens, parents, scores.view(torch.float32).view(groups, beams), ranks,
                                 ended if end is not None else None, made)
        self.k = [storage.k[g] for g in range(len(m.groups))]
        self.v = [storage.v[g] for g in range(len(m.groups))]
        self.states = list(storage.state.values())
        self.graph = None
        self.kernels = 0

    def begin(self, requests, prompt_lengths, logits) -> None:
        """The beams of a new search, chosen from the logits behind the prompts.  ``requests``: their cache records, row by row."""
        device = self.runner.device
        put = lambda to, values: to.copy_(torch.tensor(values, dtype=torch.int32).to(device))  # noqa: E731
        for g, (table, width) in enumerate(zip(self.tables, self.runner.max_pages)):
            put(table, [r.tables[g] + [NO_PAGE] * (width - len(r.tables[g])) for r in requests])
        put(self.slots, [r.state_slot for r in requests])
        put(self.lengths, [n for n in prompt_lengths for _ in range(self.beams)])
        put(self.shared_groups, [[i * self.beams, self.beams, n] for i, n in enumerate(prompt_lengths)])
        none = torch.zeros((self.groups, 1), dtype=torch.float32, device=device)
        made = torch.zeros(self.groups, dtype=torch.int32, device=device)
        self.ops.beam_select(logits, none, self.beams, lengths=made, end_token=self.end, length_penalty=self.penalty,
                             vocab_limit=self.vocab_limit, out=self.choice)
        self._hand_over()

    def _hand_over(self) -> None:
        self.ops.beam_reorder(self.choice.parents, self.lengths, self.tables, self.k, self.v, self.slots, self.states)

    def _issue(self) -> None:
        runner, rows = self.runner, self.groups * self.beams
        t = self.ops.step_tables(self.tables, self.page_tokens, self.lengths, self.ones, rows)
        ctx = StepContext(
            ops=self.ops, act_dtype=runner.act_dtype, num_tokens=rows, num_requests=rows, token_ids=self.choice.tokens,
            positions=t.positions, token_request=t.token_request, req_q_start=t.req_q_start, req_q_len=self.ones,
            req_ctx_before=self.lengths, req_state_slot=self.slots, block_tables=t.block_tables, slot_mapping=t.slot_mapping,
            logit_rows=self.logit_rows, host_q_len=[1] * rows, host_ctx_before=[0] * rows, host_state_slot=[0] * rows,
            max_q_len=1, max_ctx_after=self.longest, decode_only=True, storage=runner.storage, shared_prefix=self.shared)
        logits = runner._forward(ctx)
        self.ops.beam_select(logits, self.choice.scores, self.beams, ended=self.choice.ended, lengths=self.choice.lengths,
                             end_token=self.end, length_penalty=self.penalty, vocab_limit=self.vocab_limit, out=self.choice)
        self.lengths.copy_(t.ctx_after)
        self._hand_over()

    def run(self, capture: bool) -> None:
        if self.graph is not None:
            self.graph.replay()
            if hasattr(self.ops, "launches"):
                self.ops.launches += self.kernels
            return
        self._issue()
        if capture:
            self._capture()

    def _capture(self) -> None:
        """Capture the launches that have just run, for the steps that follow."""
        runner, ops = self.runner, self.ops
        torch.cuda.synchronize(runner.device)
        graph, launches = torch.cuda.CUDAGraph(), getattr(ops, "launches", 0)
        dependent = getattr(ops, "set_dependent_launch", None)
        if dependent is not None:
            dependent(True)
        try:
            with _no_collection(), torch.cuda.graph(graph, pool=runner._graph_pool):
                self._issue()
        finally:
            if dependent is not None:
                dependent(False)
        self.kernels = getattr(ops, "launches", 0) - launches
        if hasattr(ops, "launches"):
            ops.launches = launches                        # captured, not run
        if runner._graph_pool is None:
            runner._graph_pool = graph.pool()
        self.graph = graph


class BeamSearch:
    GRAPHS = 4              # most captured steps kept
    GRAPH_TOKENS = 8        # searches of fewer tokens are not worth a capture
    LOOK_EVERY = 16         # steps between two looks whether all beams have ended

    def __init__(self, runner: ModelRunner, step_tokens: int) -> None:
        self.runner, self.step_tokens = runner, step_tokens
        self._steps: dict[tuple, _Step] = {}
        self._serial = 0

    def run(self, prompts: list[list[int]], params: BeamParams, end: int | None, vocab_limit: int | None) -> list[list[dict]]:
        m = self.runner.manager
        self._serial += 1
        names = [[f"beam search {self._serial}: {g}/{b}" for b in range(params.beams)] for g in range(len(prompts))]
        try:
            logits = self._prompts(names, prompts)
            requests = []
            for mine, prompt in zip(names, prompts):
                for name in mine[1:]:
                    m.fork(name, mine[0])
                for name in mine:
                    # (the last token of a continuation is chosen, not run)
                    if not m.reserve(name, len(prompt) + params.max_tokens - 1):
                        raise CacheFullError(f"the pools do not hold {params.beams} beams of {len(prompts)} prompts")
                    requests.append(m.get(name))
            return self._search(requests, [len(p) for p in prompts], params, end, vocab_limit, logits)
        finally:
            for mine in names:
                for name in reversed(mine):
                    if m.has(name):
                        m.release(name)

    def _prompts(self, names, prompts):
        """Run the prompts, at most ``step_tokens`` tokens a step; the logits behind their last tokens."""
        logits, entries, room = [], [], self.step_tokens

        def step():
            out = self.runner.step(entries)
            if out is not None:
                logits.append(out)
            entries.clear()

        for mine, prompt in zip(names, prompts):
            at = 0
            while at < len(prompt):
                n = min(room, len(prompt) - at)
                entries.append(StepEntry(mine[0], prompt[at: at + n], [n - 1] if at + n == len(prompt) else []))
                at += n
                room -= n
                if room == 0:
                    step()
                    room = self.step_tokens
        if entries:
            step()
        return torch.cat(logits)

    def _search(self, requests, prompt_lengths, params, end, vocab_limit, logits):
        runner, longest_prompt = self.runner, max(prompt_lengths)
        # sizes that kernels are launched with hold for searches of about this length
        longest = _bucket(longest_prompt + params.max_tokens, runner.max_context)
        key = (len(prompt_lengths), params.beams, _bucket(longest_prompt, runner.max_context), longest,
               _bucket(params.max_tokens, runner.max_context), params.length_penalty, end, vocab_limit)
        step = self._steps.pop(key, None)
        # (one that is captured already serves any search)
        capture = step is not None or (runner.use_cuda_graphs and params.max_tokens >= self.GRAPH_TOKENS)
        step = step or _Step(runner, *key)
        if capture:
            while len(self._steps) >= self.GRAPHS:
                self._steps.pop(next(iter(self._steps)))    # least recently used
            self._steps[key] = step
        rows = len(requests)
        history = torch.empty((params.max_tokens, 2, rows), dtype=torch.int32, device=runner.device)
        step.begin(requests, prompt_lengths, logits)
        history[0].copy_(step.buffer[:2])
        made = 1
        while made < params.max_tokens:
            if end is not None and made % self.LOOK_EVERY == 0 and all(step.choice.ended.tolist()):
                break
            step.run(capture)
            history[made].copy_(step.buffer[:2])
            made += 1
        tokens, parents = history[:made].cpu().unbind(1)
        scores, ranks = step.choice.scores.reshape(-1).tolist(), step.choice.ranks.tolist()
        lengths = step.choice.lengths.tolist()
        ended = step.choice.ended.tolist() if end is not None else [0] * rows
        check = getattr(runner.ops, "check_status", None)
        if check is not None:
            check()
        tokens, parents = tokens.tolist(), parents.tolist()
        found: list[list[dict]] = []
        for g in range(len(prompt_lengths)):
            mine = []
            for row in sorted(range(g * params.beams, (g + 1) * params.beams), key=lambda r: ranks[r]):
                if scores[row] == -math.inf:                # (fewer continuations than beams)
                    continue
                ids, at = [], row
                for t in range(made - 1, -1, -1):
                    ids.append(tokens[t][at])
                    at = parents[t][at]
                mine.append({"token_ids": ids[::-1][: lengths[row]], "logprob": scores[row],
                             "score": scores[row] / max(1, lengths[row]) ** params.length_penalty,
                             "finish_reason": "eot" if ended[row] else "length"})
            if not mine:
                raise StepError(f"prompt {g}: no continuation has a log probability (the model's logits are infinite or no numbers)")
            found.append(mine)
        return found
