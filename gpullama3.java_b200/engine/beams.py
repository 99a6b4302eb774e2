"""Beam search above the step function: of every request the ``beams`` most probable continuations go on side by side.

A request's prompt runs once.  From then on each step takes one token of every beam and, of all beams' continuations
together, selects the best (sum of log probabilities).  Those that end in a stop token and are among the ``beams`` best are
finished hypotheses; the best of the others are the new beams.  Beams that continue the same parent share its cache:
``SequenceCache.reorder`` hands pages on by reference and copies states, and a page is copied only when a beam
writes into one that others still hold.

Hypotheses are ranked by score / length ** length_penalty, the length being the tokens generated (the stop token
included).  A request is over when it has ``beams`` finished hypotheses and no beam could still come before the last of
them, when its beams are as long as they may get (they are hypotheses then, too), or when nothing can follow them.

The reference project samples one token per step of one sequence (inference/InferenceEngine.java:309-355); a search is
not part of it.  The loop around it (batches of requests, limits, stop tokens, metrics) is the generation loop's."""
from __future__ import annotations

import math
import time
from dataclasses import dataclass, field

from ..cache.pages import PAGE_TOKENS, pages_for
from ..kernels import ops
from ..sampling.sampler import BeamSelector
from .generate import FINISH_CONTEXT, FINISH_LENGTH, FINISH_STOP, GenerationError, RunMetrics
from .step import SequenceInput

FINISH_STUCK = "stuck"        # no token has a probability behind this hypothesis


@dataclass(frozen=True)
class BeamParams:
    beams: int = 4
    length_penalty: float = 1.0
    n_best: int = 1               # hypotheses returned per request, at most ``beams``

    def __post_init__(self):
        if self.beams < 1:
            raise ValueError(f"a beam search needs at least one beam, got {self.beams}")
        if not 1 <= self.n_best <= self.beams:
            raise ValueError(f"n_best {self.n_best} must be within [1, {self.beams}]")
        if not -32 <= self.length_penalty <= 32:        # (a length to that power is a number)
            raise ValueError(f"length_penalty must be within [-32, 32], got {self.length_penalty}")


@dataclass
class BeamHypothesis:
    tokens: list[int]             # the stop token included when one ended it
    log_prob: float               # sum of the tokens' log probabilities
    score: float                  # log_prob / len(tokens) ** length_penalty
    finish_reason: str


@dataclass
class BeamRequest:
    """One request's search: its beams and what has finished so far.  No device is involved."""
    params: BeamParams
    prompt_length: int
    max_new_tokens: int
    max_length: int
    stop: frozenset
    beams: list[tuple[list[int], float]] = field(default_factory=lambda: [([], 0.0)])     # (tokens, log probability), -inf: does not count
    finished: list[BeamHypothesis] = field(default_factory=list)                             # the best first
    done: bool = False

    def _finish(self, tokens: list[int], log_prob: float, reason: str) -> None:
        score = log_prob / max(1, len(tokens)) ** self.params.length_penalty
        self.finished.append(BeamHypothesis(list(tokens), log_prob, score, reason))
        self.finished.sort(key=lambda h: -h.score)       # (stable: of equal scores the earlier goes first)
        del self.finished[self.params.beams:]

    def _end(self, reason: str) -> None:
        for tokens, log_prob in self.beams:
            if log_prob > -math.inf:
                self._finish(tokens, log_prob, reason)
        self.done = True

    def advance(self, candidates: list[tuple[float, int, int]]) -> list[int]:
        """Takes a step's continuations (log probability, beam, token), the best first; returns the beam that each new one continues
        (always as many as there are beams; none when the request is over)."""
        k = self.params.beams
        new, parents = [], []
        for rank, (log_prob, beam, token) in enumerate(candidates):
            if token in self.stop:
                if rank < k:
                    self._finish(self.beams[beam][0] + [token], log_prob, FINISH_STOP)
            elif len(new) < k:
                new.append((self.beams[beam][0] + [token], log_prob))
                parents.append(beam)
        if not new:
            if candidates:
                self.done = True            # all that could follow has ended
            else:
                self._end(FINISH_STUCK)
            return []
        self.beams = new
        length = len(new[0][0])
        if length >= self.max_new_tokens:
            self._end(FINISH_LENGTH)
        elif self.prompt_length + length >= self.max_length:
            self._end(FINISH_CONTEXT)
        elif len(self.finished) == k and self._best_possible(length) <= self.finished[-1].score:
            self.done = True
        if self.done:
            return []
        # places for which there is no continuation stay in the batch and do not count
        while len(self.beams) < k:
            self.beams.append((new[0][0], -math.inf))
            parents.append(parents[0])
        return parents

    def _best_possible(self, length: int) -> float:
        """The highest score a beam may end with: log probabilities only fall, and are divided by the longest or the next length."""
        best, p = max(lp for _, lp in self.beams), self.params.length_penalty
        longest = min(self.max_new_tokens, self.max_length - self.prompt_length)
        return best / (longest if p > 0 else length + 1) ** p

    def best(self) -> list[BeamHypothesis]:
        return self.finished[:self.params.n_best]


def plan_beam_batches(prompt_lengths: list[int], max_new_tokens: int, beams: int, max_slots: int, n_pages: int,
                      max_length: int) -> list[list[int]]:
    """Cut the requests, in order, into batches whose beams have slots and, each at its longest, pages: the full pages of a prompt are one
    set for all beams of a request, every page behind them may be each beam's own."""
    if beams > max_slots:
        raise GenerationError(f"{beams} beams need as many sequence slots, there are {max_slots}")
    batches, cur, cur_pages = [], [], 0
    for i, n in enumerate(prompt_lengths):
        if n < 1:
            raise GenerationError(f"request {i}: empty prompt")
        if n > max_length:
            raise GenerationError(f"request {i}: prompt of {n} tokens exceeds the longest sequence allowed ({max_length})")
        shared = n // PAGE_TOKENS
        need = shared + beams * (pages_for(min(n + max_new_tokens, max_length)) - shared)
        if need > n_pages:
            raise GenerationError(f"request {i}: {beams} beams need {need} cache pages, the cache has {n_pages}")
        if cur and ((len(cur) + 1) * beams > max_slots or cur_pages + need > n_pages):
            batches.append(cur)
            cur, cur_pages = [], 0
        cur.append(i)
        cur_pages += need
    if cur:
        batches.append(cur)
    return batches


class BeamSearcher:
    """``step_fn`` is the step function: called for prompts, its ``decode_beams`` for the steps behind them and its ``select_beams``
    for the first selection.  ``cache`` gives slots, forks them and takes them back."""

    def __init__(self, step_fn, cache, *, max_batch: int, max_length: int):
        self.step_fn, self.cache = step_fn, cache
        self.max_batch, self.max_length = max_batch, max_length
        self.last_metrics = RunMetrics()

    def search(self, prompts: list[list[int]], max_new_tokens: int, params: BeamParams, stop_ids=()) -> list[list[BeamHypothesis]]:
        """The best hypotheses of every prompt, in the order of the prompts."""
        stop = frozenset(stop_ids)
        metrics = RunMetrics()
        if max_new_tokens <= 0:
            self.last_metrics = metrics
            return [[BeamHypothesis([], 0.0, 0.0, FINISH_LENGTH)] for _ in prompts]
        # every beam may have all its stop tokens among the best, and as many others are needed
        keep = params.beams * (1 + len(stop))
        if not ops.beam_select_takes(params.beams, keep):
            raise GenerationError(f"{params.beams} beams and {len(stop)} stop tokens need {keep} continuations a step, at most "
                                  f"{ops.BEAM_MAX_KEEP} are selected")
        t0 = time.perf_counter()
        requests = [BeamRequest(params, len(p), max_new_tokens, self.max_length, stop) for p in prompts]
        for batch in plan_beam_batches([len(p) for p in prompts], max_new_tokens, params.beams, min(self.max_batch, self.cache.max_slots),
                                       self.cache.pages_for_planning(), self.max_length):
            slots: dict[int, list[int]] = {}
            try:
                for i in batch:
                    slots[i] = [self.cache.acquire()]
                self._run_batch(batch, slots, prompts, requests, params.beams, keep, metrics)
            finally:
                for taken in slots.values():
                    for s in taken:
                        self.cache.release(s)
        metrics.seconds = time.perf_counter() - t0
        self.last_metrics = metrics
        return [r.best() for r in requests]

    def _run_batch(self, batch, slots, prompts, requests, beams, keep, metrics):
        t0 = time.perf_counter()
        logits = self.step_fn([SequenceInput(slots[i][0], list(prompts[i]), [len(prompts[i]) - 1]) for i in batch])
        metrics.prompt_tokens += sum(len(prompts[i]) for i in batch)
        found = self.step_fn.select_beams(logits, BeamSelector(1, keep), [0.0] * len(batch))
        metrics.prefill_seconds += time.perf_counter() - t0
        t0 = time.perf_counter()

        def take(live, found):
            """Advances the requests of ``live``; returns those that go on, their slots in the order of their beams."""
            going = []
            for i, candidates in zip(live, found):
                metrics.generated_tokens += 1
                parents = requests[i].advance(candidates)
                if requests[i].done:
                    for s in slots.pop(i):
                        self.cache.release(s)
                    continue
                if len(slots[i]) == 1 and beams > 1:      # behind the prompt: one sequence becomes all beams
                    slots[i] = slots[i] + self.cache.fork(slots[i] * (beams - 1))
                else:
                    slots[i] = self.cache.reorder(slots[i], parents)
                going.append(i)
            return going

        selector = BeamSelector(beams, keep)
        live = take(batch, found)
        while live:
            inputs = [SequenceInput(s, [tokens[-1]], [0]) for i in live for s, (tokens, _) in zip(slots[i], requests[i].beams)]
            scores = [log_prob for i in live for _, log_prob in requests[i].beams]
            metrics.decode_steps += 1
            live = take(live, self.step_fn.decode_beams(inputs, selector, scores))
        metrics.decode_seconds += time.perf_counter() - t0
