"""Beam search: every prompt is continued in several ways at once, and the likeliest whole continuations come back.

Not in umarhassan-cloud/kvforge (its ``Sampler`` draws one token a request, src/tokenvault/sampling.py:69-88).  A prompt's
beams are requests of the same step function: they share the prompt's pages (``BlockManager.fork``), and a step's choice
among all of a prompt's continuations is one kernel over the step's logits (``ops.beam_select``).  What the choice moves is
little: a beam that goes on keeps its pages and its state slot for its first continuation; for each further one the full pages
are shared, and the partly filled page of every layer and the states are copied (``ops.copy_pages``, ``ops.copy_states``) into what
the beams that end give back.

The rules: of a prompt's best continuations, in order, one that ends in a stop token is a finished
hypothesis if it is among the first ``num_beams``, and the first ``num_beams`` of the others are the next beams.  (So many are looked at that all stop tokens
of all beams leave enough, as far as the kernel's 64 candidates go; where none of them goes on, the prompt ends.)  A hypothesis's score is the sum
of its tokens' log probabilities over its length to the power ``length_penalty``.  A prompt ends when it has ``num_beams`` finished
hypotheses and no beam could still beat the worst of them at its present length, or at ``max_tokens`` (then the beams are hypotheses too).
"""

from __future__ import annotations

import itertools
import math
from collections.abc import Sequence
from dataclasses import dataclass, field

import torch

from .. import ops
from .request import FinishReason
from .scheduler import RequestRejectedError
from .step import BatchItem


@dataclass
class BeamParams:
    num_beams: int = 4
    max_tokens: int = 64
    length_penalty: float = 1.0
    num_return: int = 1  # hypotheses reported, best first
    stop_token_ids: list[int] = field(default_factory=list)
    ignore_eos: bool = False

    def __post_init__(self) -> None:
        if not 1 <= self.num_beams <= ops.BEAM_MAX_K // 2:
            raise ValueError(f"num_beams must be between 1 and {ops.BEAM_MAX_K // 2}")
        if self.max_tokens < 1:
            raise ValueError("max_tokens must be >= 1")
        if not 1 <= self.num_return <= self.num_beams:
            raise ValueError("num_return must be between 1 and num_beams")
        if not abs(self.length_penalty) <= 64:
            raise ValueError("length_penalty must lie between -64 and 64")


@dataclass
class BeamHypothesis:
    token_ids: list[int]
    logprob: float  # sum over the tokens
    score: float
    finish_reason: FinishReason
    text: str | None = None


@dataclass
class BeamOutput:
    prompt_token_ids: list[int]
    hypotheses: list[BeamHypothesis]  # best first


@dataclass
class _Beam:
    seq: str | None  # the request that holds its pages; None: a place that no continuation is left for
    tokens: list[int]
    logprob: float


class BeamGroup:
    """The beams of one prompt and the rules of their choice; no tensors."""

    def __init__(self, prompt: list[int], params: BeamParams, stops: set[int], limit: int) -> None:
        self.prompt, self.params, self.stops = prompt, params, stops
        self.limit = limit  # tokens a hypothesis may have
        # scores are doubles above their smallest normal number, 2^-1022: sums of log probabilities lie between 2^-149 and 104 a token
        if abs(params.length_penalty) * math.log2(limit) > 870:
            raise RequestRejectedError(f"length_penalty = {params.length_penalty} has no scores for hypotheses of up to {limit} tokens")
        self.beams: list[_Beam] = []
        self.finished: list[BeamHypothesis] = []
        self.done = False

    @property
    def length(self) -> int:
        """Tokens of every beam."""
        return len(self.beams[0].tokens) if self.beams else 0

    def score(self, logprob: float, length: int) -> float:
        return logprob / length**self.params.length_penalty

    def _keep(self, tokens: list[int], logprob: float, reason: FinishReason) -> None:
        self.finished.append(BeamHypothesis(tokens, logprob, self.score(logprob, len(tokens)), reason))
        self.finished.sort(key=lambda h: -h.score)  # (stable: of equal ones the earlier)
        del self.finished[self.params.num_beams :]

    def choose(self, parents: Sequence[int], tokens: Sequence[int], logprobs: Sequence[float]) -> list[tuple[int, int, float]]:
        """The next beams as (parent, token, log probability) from a step's candidates, best first; ends the group if it is over."""
        w = self.params.num_beams
        following: list[tuple[int, int, float]] = []
        for rank, (parent, token, logprob) in enumerate(zip(parents, tokens, logprobs)):
            if parent < 0:
                break  # nothing is left
            if token in self.stops:
                if rank < w:
                    self._keep([*self.beams[parent].tokens, token], logprob, FinishReason.STOP)
            elif len(following) < w:
                following.append((parent, token, logprob))
        length = self.length + 1
        if not following:
            self.done = True
        elif length >= self.limit:
            for parent, token, logprob in following:
                self._keep([*self.beams[parent].tokens, token], logprob, FinishReason.LENGTH)
            self.done = True
        elif len(self.finished) == w and self.score(following[0][2], length) <= self.finished[-1].score:
            self.done = True
        return [] if self.done else following


class BeamSearch:
    """Runs prompts through an engine's step function; the engine must have nothing else under way."""

    def __init__(self, engine, params: BeamParams, adapter_slot: Sequence[int], stops: set[int]) -> None:
        self.engine, self.params, self.stops = engine, params, stops
        self.candidates = min(ops.BEAM_MAX_K, params.num_beams * (1 + max(1, len(stops))))  # a prompt
        self.core = engine.core
        self.bm, self.slots, self.pool = engine.block_manager, engine.core.state_slots, engine.kv_cache
        self.cfg = engine.config.scheduler
        self.adapters = adapter_slot
        self._count = itertools.count()
        self._issued: list[str] = []  # names of the requests that hold beams
        # a step takes so many beams: one request and one token each
        groups = max(1, min(self.cfg.max_num_seqs, self.cfg.max_num_batched_tokens) // params.num_beams)
        rows, k = groups * params.num_beams, self.candidates
        dev = self.core.device
        self.max_groups = groups
        self._workspace = ops.beam_workspace(rows, engine.vocab_size, k, dev)
        # scores in, and out: parents, tokens, scores (one buffer, one copy)
        self._scores = torch.empty(rows, dtype=torch.float32, device=dev)
        self._host_scores = torch.empty(rows, dtype=torch.float32, pin_memory=True)
        self._out = torch.empty(3 * groups * k, dtype=torch.int32, device=dev)

    def _name(self) -> str:
        self._issued.append(f"beam-{next(self._count)}")
        return self._issued[-1]

    # ------------------------------------------------------------------ pages
    def _reserve(self, prompt: list[int], limit: int) -> int:
        """Pages of a group that a prompt can take at the most: its own, and for every beam what lies behind its last full page."""
        bm, w = self.bm, self.params.num_beams
        total = len(prompt) + limit
        return bm.blocks_needed(len(prompt)) + w * (bm.blocks_needed(total) - len(prompt) // bm.block_size)

    # ------------------------------------------------------------------ the choice
    def _select(self, logits: torch.Tensor, scores: list[float], count: int) -> tuple[list, list, list]:
        """Per prompt of ``count``: parents, tokens and scores of its best continuations."""
        k, rows = self.candidates, len(scores)
        self._host_scores[:rows] = torch.tensor(scores)  # (the copy before this one has been waited for: its results were read)
        self._scores[:rows].copy_(self._host_scores[:rows], non_blocking=True)
        n = count * k
        views = [self._out[i * n : (i + 1) * n].view(count, k) for i in range(3)]
        ops.beam_select(logits[:rows], self._scores[:rows], views[0], views[1], views[2].view(torch.float32), self._workspace)
        host = self._out[: 3 * n].cpu()
        self.core.rt.check_error_flag()
        return host[:n].view(count, k).tolist(), host[n : 2 * n].view(count, k).tolist(), host[2 * n :].view(torch.float32).view(count, k).tolist()

    def _advance(self, group: BeamGroup, parents, tokens, logprobs) -> tuple[list, list]:
        """Apply one choice: returns the copies of pages and of states that it needs."""
        following = group.choose(parents, tokens, logprobs)
        before = group.beams
        pages: list = []
        states: list = []
        used = {p for p, _, _ in following}
        for i, beam in enumerate(before):  # what ends gives back first: its pages are taken again below
            if beam.seq is not None and i not in used:
                self.bm.free(beam.seq)
                self.slots.free(beam.seq)
        taken: set[int] = set()
        beams: list[_Beam] = []
        for parent, token, logprob in following:
            old = before[parent]
            seq = old.seq
            if parent in taken:
                seq = self._name()
                # the tokens whose keys are in the cache: all of the parent's but its next one
                computed = len(group.prompt) + len(old.tokens)
                pages += self.bm.fork(old.seq, seq, computed)
                states.append((self.slots.slot(old.seq), self.slots.allocate(seq, fresh=False)))
            taken.add(parent)
            beams.append(_Beam(seq, [*old.tokens, token], logprob))
        # (a vocabulary too small for all beams leaves places without one)
        while beams and len(beams) < self.params.num_beams:
            beams.append(_Beam(None, list(beams[0].tokens), -math.inf))
        group.beams = beams
        return pages, states

    # ------------------------------------------------------------------ steps
    def _prefill(self, fresh: list[tuple[BeamGroup, str, int]]) -> None:
        """Run new prompts to their ends, in portions that share steps, and choose their first beams."""
        rt, w = self.core.rt, self.params.num_beams
        done = {seq: 0 for _, seq, _ in fresh}
        waiting = list(fresh)
        while waiting:
            budget = self.cfg.max_num_batched_tokens
            items, ends = [], []
            for group, seq, adapter in waiting:
                start = done[seq]
                take = min(len(group.prompt) - start, budget)
                if self.cfg.enable_chunked_prefill:
                    take = min(take, self.cfg.max_prefill_chunk or take)
                elif take < len(group.prompt):
                    break
                if take < 1 or len(items) >= rt.max_seqs:
                    break
                self.bm.append_slots(seq, start + take, start)
                last = start + take == len(group.prompt)
                items.append(BatchItem(seq, group.prompt[start : start + take], start, "last" if last else "none", adapter=adapter))
                budget -= take
                done[seq] += take
                if last:
                    ends.append((group, seq))
            logits = self.engine.runner.step(items)
            waiting = [f for f in waiting if done[f[1]] < len(f[0].prompt)]
            if not ends:
                continue
            for at in range(0, len(ends), self.max_groups):
                part = ends[at : at + self.max_groups]
                results = self._select(logits[at : at + len(part)], [0.0] * len(part), len(part))
                moved: tuple[list, list] = ([], [])
                for (group, seq), *found in zip(part, *results):
                    group.beams = [_Beam(seq, [], 0.0)]
                    for copies, more in zip(moved, self._advance(group, *found)):
                        copies += more
                self._move(*moved)
        assert all(len(g.beams) in (0, w) for g, _, _ in fresh)

    def _move(self, pages: list, states: list) -> None:
        self.pool.copy_pages(pages)
        self.pool.copy_states(states)

    def _decode(self, live: list[tuple[BeamGroup, int]]) -> None:
        items, scores = [], []
        for group, adapter in live:
            at = len(group.prompt) + group.length - 1
            real = [b for b in group.beams if b.seq is not None]
            for beam in real:
                self.bm.append_slots(beam.seq, at + 1, at)
                items.append(BatchItem(beam.seq, [beam.tokens[-1]], at, "last", adapter=adapter))
            if len(real) < len(group.beams):  # places without a beam see the last one's logits, and nothing of them is chosen
                items[-1].logits = [0] * (1 + len(group.beams) - len(real))
            scores += [b.logprob for b in group.beams]
        results = self._select(self.engine.runner.step(items), scores, len(live))
        moved: tuple[list, list] = ([], [])
        for (group, _), *found in zip(live, *results):
            for copies, more in zip(moved, self._advance(group, *found)):
                copies += more
        self._move(*moved)

    # ------------------------------------------------------------------ all prompts
    def run(self, prompts: Sequence[list[int]]) -> list[BeamOutput]:
        p, cfg, bm = self.params, self.cfg, self.bm
        groups = []
        for prompt in prompts:
            if not prompt:
                raise RequestRejectedError("the prompt is empty")
            if len(prompt) >= cfg.max_model_len:
                raise RequestRejectedError(f"a prompt of {len(prompt)} tokens leaves no room under max_model_len = {cfg.max_model_len}")
            if not cfg.enable_chunked_prefill and len(prompt) > cfg.max_num_batched_tokens:
                raise RequestRejectedError(f"a prompt of {len(prompt)} tokens exceeds max_num_batched_tokens = {cfg.max_num_batched_tokens} and prompts are not cut")
            if p.num_beams > cfg.max_num_seqs:
                raise RequestRejectedError(f"{p.num_beams} beams are more than max_num_seqs = {cfg.max_num_seqs}")
            if p.num_beams > cfg.max_num_batched_tokens:
                raise RequestRejectedError(f"{p.num_beams} beams are more than max_num_batched_tokens = {cfg.max_num_batched_tokens}")
            group = BeamGroup(list(prompt), p, self.stops, min(p.max_tokens, cfg.max_model_len - len(prompt)))
            if self._reserve(group.prompt, group.limit) > bm.num_blocks:
                raise RequestRejectedError(f"{p.num_beams} beams of {len(prompt) + group.limit} tokens can never fit the pages of the cache")
            groups.append(group)
        waiting = list(zip(groups, self.adapters))
        live: list[tuple[BeamGroup, int]] = []
        try:
            while waiting or live:
                promised = sum(self._reserve(g.prompt, g.limit) for g, _ in live)
                fresh = []
                while waiting and len(live) + len(fresh) < self.max_groups:
                    group, adapter = waiting[0]
                    need = self._reserve(group.prompt, group.limit)
                    if promised + need > bm.num_blocks:
                        break
                    promised += need
                    seq = self._name()
                    bm.allocate(seq, len(group.prompt), min(len(group.prompt), cfg.max_num_batched_tokens))
                    self.slots.allocate(seq)
                    fresh.append((group, seq, adapter))
                    waiting.pop(0)
                if fresh:
                    self._prefill(fresh)
                    live += [(g, a) for g, _, a in fresh if not g.done]
                if live:
                    self._decode(live)
                    live = [(g, a) for g, a in live if not g.done]
        finally:  # (a step that failed leaves nothing behind)
            for seq in self._issued:
                bm.free(seq)
                self.slots.free(seq)
        return [BeamOutput(g.prompt, g.finished[: p.num_return]) for g in groups]
