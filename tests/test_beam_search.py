"""Beam search without a GPU: forks of cached sequences (pages shared, copied when written, states copied), and the search itself
over a scripted step function that reads its history back from the cache."""
import math
import random

import pytest
import torch

from gpullama3.java_b200.cache import (CacheError, CacheFull, KVCacheNeed, PagedGroup, PagePool, SequenceCache, StateNeed, pages_for,
                                       register_cache_group, unregister_cache_group)
from gpullama3.java_b200.engine.beams import FINISH_STUCK, BeamParams, BeamRequest, BeamSearcher, plan_beam_batches
from gpullama3.java_b200.engine.generate import FINISH_CONTEXT, FINISH_LENGTH, FINISH_STOP, GenerationError
from gpullama3.java_b200.kernels import ops
from gpullama3.java_b200.sampling.sampler import BeamSelector


# ---- pages with several holders


def test_a_shared_page_is_free_after_its_last_holder():
    pool = PagePool(3)
    a, b = pool.alloc(2)
    pool.share([a])
    pool.share([a, b])
    assert pool.holders(a) == 3 and pool.holders(b) == 2 and pool.n_held == 2 and pool.n_shared == 2
    pool.free([a, b])
    assert pool.n_shared == 1
    pool.free([a])
    assert pool.n_shared == 0 and pool.n_free == 1 and pool.n_held == 2
    pool.free([b, a])
    assert pool.n_free == 3
    with pytest.raises(CacheError, match="twice"):
        pool.free([a])
    for bad in (a, 7, -1):
        with pytest.raises(CacheError, match="cannot be shared"):
            pool.share([bad])


def _cache(max_tokens=64 * 40, max_slots=12, **more):
    needs = {0: KVCacheNeed(1, 16), 1: StateNeed((3,), torch.float64), 2: KVCacheNeed(2, 16, window=70), 3: KVCacheNeed(1, 16, chunk=100)}
    needs.update(more)
    return SequenceCache(needs, max_tokens=max_tokens, max_slots=max_slots, dtype=torch.float32, device="cpu", window_slack=64)


class Told:
    """What a sequence has been told, kept beside the cache: its tokens, and which positions a query may still read."""

    def __init__(self, cache):
        self.cache, self.tokens = cache, {}

    def start(self):
        s = self.cache.acquire()
        self.tokens[s] = []
        return s

    def write(self, requests):
        self.cache.reserve([(s, len(t)) for s, t in requests])
        for s, toks in requests:
            for t in toks:
                pos = len(self.tokens[s])
                for g in self.cache.paged_groups:
                    page = g.rows[s][pos // 64]
                    g.k[:, page, :, pos % 64] = float(t)
                    g.v[:, page, :, :, pos % 64] = -float(t)
                for g in self.cache.slot_groups:
                    g.data[:, s] += float(t) * (pos + 1)
                self.tokens[s].append(t)
            self.cache.commit(s, len(toks))

    def check(self):
        self.cache.check_invariants()
        for s, toks in self.tokens.items():
            n = len(toks)
            assert self.cache.length(s) == n
            for g in self.cache.paged_groups:
                lo = max(0, n - g.window + 1) if g.window else n - n % g.chunk if g.chunk else 0
                for pos in range(lo, n):
                    page = g.rows[s][pos // 64]
                    assert float(g.k[0, page, 0, pos % 64, 5]) == toks[pos] and float(g.v[-1, page, -1, 3, pos % 64]) == -toks[pos]
            for g in self.cache.slot_groups:
                assert bool((g.data[:, s] == sum(t * (i + 1) for i, t in enumerate(toks))).all())


def test_forks_share_pages_until_one_of_them_writes():
    c = _cache()
    told = Told(c)
    a = told.start()
    told.write([(a, list(range(100)))])
    held = c.paged_groups[0].pool.n_held
    b, d = c.fork([a, a])
    told.tokens[b], told.tokens[d] = list(told.tokens[a]), list(told.tokens[a])
    assert c.paged_groups[0].pool.n_held == held and c.shared_pages([a, b, d])[0] == 1
    told.check()
    told.write([(a, [7]), (b, [8]), (d, [9])])            # all three write: two copies, the last holder keeps the page
    assert c.paged_groups[0].pool.n_held == held + 2
    told.check()
    e = c.fork([b])[0]
    told.tokens[e] = list(told.tokens[b])
    told.write([(b, [1])])                                # the one that writes gets the copy
    told.write([(e, [2])])                                # the other is the last holder now
    assert c.paged_groups[0].pool.n_held == held + 3
    told.check()
    for s in (a, b, d, e):
        c.release(s)
    assert all(g.pool.n_free == g.pool.n_pages for g in c.paged_groups) and c.slots.n_free == c.max_slots


def test_a_fork_at_a_page_border_copies_nothing_and_keeps_no_pages_reserved_ahead():
    c = _cache()
    told = Told(c)
    a = told.start()
    told.write([(a, list(range(64)))])
    c.reserve([(a, 100)])                                 # room that nothing has been written to
    n = len(c.page_rows(0, [a])[0])
    b = c.fork([a])[0]
    told.tokens[b] = list(told.tokens[a])
    assert n == 3 and len(c.page_rows(0, [b])[0]) == 1
    moves = []
    c.paged_groups[0].copy = moves.extend
    told.write([(b, [5]), (a, [6])])
    assert moves == []
    told.check()


def test_reorder_keeps_slots_where_it_can():
    c = _cache()
    told = Told(c)
    slots = [told.start() for _ in range(4)]
    told.write([(s, [10 * i + 1, 3, i]) for i, s in enumerate(slots)])
    old = {s: list(told.tokens[s]) for s in slots}
    new = c.reorder(slots, [2, 1, 2, 2])                  # beams 0 and 3 end; 2 has three children, one of them itself
    assert new[1] == slots[1] and new[2] == slots[2] and {new[0], new[3]} == {slots[0], slots[3]}
    told.tokens = {n: list(old[slots[p]]) for n, p in zip(new, [2, 1, 2, 2])}
    told.check()
    assert c.reorder(new, [0, 1, 2, 3]) == new
    assert c.reorder(new, [3, 2, 1, 0]) == new[::-1]      # everyone goes on, in another order
    fewer = c.reorder(new, [1, 1])
    assert len(c.live_slots()) == 2 and fewer[1] == new[1]
    assert c.reorder(fewer, []) == [] and c.live_slots() == []


def test_forks_refuse_and_change_nothing():
    c = _cache(max_tokens=64 * 6, max_slots=3)
    told = Told(c)
    a = told.start()
    told.write([(a, [1] * 70)])
    with pytest.raises(CacheFull, match="3 sequence slot"):
        c.fork([a, a, a])
    with pytest.raises(CacheError, match="not live"):
        c.fork([a, 2])
    with pytest.raises(CacheError, match="not live"):
        c.reorder([a, 2], [0, 1])
    for slots, parents in (([a], [0, 0]), ([a, a], [0])):
        with pytest.raises(CacheError, match="children"):
            c.reorder(slots, parents)
    with pytest.raises(CacheError, match="parents"):
        c.reorder([a], [1])
    assert c.live_slots() == [a]
    b, d = c.fork([a, a])
    told.tokens[b], told.tokens[d] = list(told.tokens[a]), list(told.tokens[a])
    changes = c.ownership_changes
    told.write([(a, [2]), (b, [3]), (d, [4])])            # 4 of 6 pages; the slot numbers mean what they meant, but for a page
    assert c.ownership_changes > changes
    with pytest.raises(CacheFull):
        c.reserve([(a, 64), (b, 64), (d, 64)])
    e = c.page_rows(0, [a, b, d])
    c.release(d)
    del told.tokens[d]
    f = c.fork([b])[0]
    told.tokens[f] = list(told.tokens[b])
    with pytest.raises(CacheFull):                        # three pages are left, the copy is a fourth
        c.reserve([(a, 64 * 3), (b, 1)])
    assert c.page_rows(0, [a, b]) == e[:2]
    told.check()


def test_a_group_that_cannot_copy_refuses_forks():
    class Need:
        pass

    class Group(PagedGroup):
        def view(self, entry):
            return None

    need = Need()
    register_cache_group(Need, Group)
    try:
        c = SequenceCache({0: KVCacheNeed(1, 16), 1: need}, max_tokens=640, dtype=torch.float32, device="cpu")
        a, b = c.acquire(), c.acquire()
        with pytest.raises(CacheError, match="cannot fork"):
            c.fork([a])
        with pytest.raises(CacheError, match="cannot fork"):
            c.reorder([a, b], [0, 0])
        assert c.reorder([a, b], [1, 0]) == [b, a] and c.live_slots() == [a, b]      # no copy, no refusal
    finally:
        unregister_cache_group(Need)


def test_random_forks_reorders_and_writes_keep_every_sequence():
    rng = random.Random(3)
    c = _cache(max_tokens=64 * 60, max_slots=9)
    told = Told(c)
    for step in range(600):
        live = list(told.tokens)
        op = rng.random()
        try:
            if op < 0.12 and len(live) < 9:
                told.start()
            elif op < 0.25 and live:
                parents = [rng.choice(live) for _ in range(rng.randint(1, 3))]
                for n, p in zip(c.fork(parents), parents):
                    told.tokens[n] = list(told.tokens[p])
            elif op < 0.35 and live:
                s = rng.choice(live)
                c.release(s)
                del told.tokens[s]
            elif op < 0.5 and live:
                slots = rng.sample(live, rng.randint(1, len(live)))
                parents = [rng.randrange(len(slots)) for _ in range(rng.randint(0, len(slots)))]
                old = {s: told.tokens.pop(s) for s in slots}
                for n, p in zip(c.reorder(slots, parents), parents):
                    told.tokens[n] = list(old[slots[p]])
            elif live:
                some = rng.sample(live, rng.randint(1, len(live)))
                told.write([(s, [rng.randrange(1000) for _ in range(rng.choice([1, 1, 1, 5, 40]))]) for s in some])
        except CacheFull:
            pass
        if step % 10 == 0:
            told.check()
        if sum(len(t) for t in told.tokens.values()) > 1500:
            for s in list(told.tokens):
                c.release(s)
            told.tokens = {}
    told.check()


def test_shared_pages_with_unequal_lengths():
    c = SequenceCache({0: KVCacheNeed(1, 16, window=64)}, max_tokens=64 * 20, max_slots=4, dtype=torch.float32, device="cpu", window_slack=64)
    a = c.acquire()
    c.reserve([(a, 100)])
    c.commit(a, 100)
    b = c.fork([a])[0]
    assert c.shared_pages([a, b]) == [1]
    c.reserve([(a, 64)])
    c.commit(a, 64)            # lets go of its first page, which the other still reads
    assert c.shared_pages([a, b]) == [0]


# ---- the search


VOCAB = 24


def _row(history):
    """Log probabilities behind a history: a function of all of its tokens."""
    g = torch.Generator().manual_seed(hash(tuple(int(t) for t in history)) & 0x7FFFFFFF)
    return torch.log_softmax(torch.randn(VOCAB, generator=g) * 2, dim=0)


class ScriptedBeams:
    """Stands in for the step function.  What a sequence was told is read back from the cache's pages, so a wrong fork shows."""

    def __init__(self, cache, forbid=()):
        self.cache, self.told, self.forbid, self.steps = cache, Told(cache), set(forbid), []

    def _logits(self, slots):
        out = []
        for s in slots:
            g = self.cache.paged_groups[0]
            history = [float(g.k[0, g.rows[s][p // 64], 0, p % 64, 0]) for p in range(self.cache.length(s))]
            assert float(self.cache.slot_groups[0].data[0, s, 0]) == sum(t * (i + 1) for i, t in enumerate(history))
            row = _row(history)
            row[list(self.forbid)] = -math.inf
            out.append(row)
        return torch.stack(out)

    def _write(self, inputs):
        for s in inputs:
            self.told.tokens[s.slot] = [None] * self.cache.length(s.slot)
        self.told.write([(s.slot, s.tokens) for s in inputs])

    def __call__(self, inputs):
        self._write(inputs)
        self.steps.append(len(inputs))
        return self._logits([s.slot for s in inputs])

    def decode_beams(self, inputs, selector, scores):
        self._write(inputs)
        self.steps.append(len(inputs))
        return self.select_beams(self._logits([s.slot for s in inputs]), selector, scores)

    def select_beams(self, logits, selector, scores):
        G = len(scores) // selector.beams
        total = torch.tensor(scores).view(G, selector.beams, 1) + logits.view(G, selector.beams, -1)
        out = []
        for g in range(G):
            order = torch.argsort(total[g].flatten(), descending=True, stable=True)[:selector.keep].tolist()
            out.append([(float(total[g].flatten()[i]), *divmod(i, VOCAB)) for i in order if total[g].flatten()[i] > -math.inf])
        return out


def _plain_search(prompt, k, n_new, stop, alpha, max_length, forbid=()):
    """The search by its definition, over token lists."""
    beams, finished = [([], 0.0)], []
    rank = lambda h: -(h[1] / max(1, len(h[0])) ** alpha)
    while True:
        found = []
        for b, (toks, lp) in enumerate(beams):
            row = _row(prompt + toks)
            found += [(toks + [t], float(torch.tensor(lp) + row[t]), t in stop) for t in range(VOCAB) if t not in forbid]
        found.sort(key=lambda c: -c[1])
        finished += [(t, lp, FINISH_STOP) for t, lp, ends in found[:k] if ends]
        finished = sorted(finished, key=rank)[:k]
        going = [(t, lp) for t, lp, ends in found[:k * (1 + len(stop))] if not ends][:k]
        if not going:
            if not found:
                finished = sorted(finished + [(t, lp, FINISH_STUCK) for t, lp in beams], key=rank)[:k]
            return finished
        beams = going
        n = len(beams[0][0])
        reason = FINISH_LENGTH if n >= n_new else FINISH_CONTEXT if len(prompt) + n >= max_length else None
        if reason:
            return sorted(finished + [(t, lp, reason) for t, lp in beams], key=rank)[:k]
        if len(finished) == k:
            longest = min(n_new, max_length - len(prompt))
            if beams[0][1] / (longest if alpha > 0 else n + 1) ** alpha <= finished[-1][1] / len(finished[-1][0]) ** alpha:
                return finished


@pytest.mark.parametrize("k, n_new, stop, alpha, lengths, max_length", [
    (1, 5, (), 1.0, [3], 999), (3, 6, (), 1.0, [3, 1, 5], 999), (4, 8, (2,), 1.0, [62, 63, 64, 65], 999), (5, 7, (1, 4, 9), 0.5, [60, 3], 999),
    (4, 9, (0, 3, 7, 11, 15), 0.0, [5, 6], 999), (3, 10, (5, 6, 8), -0.7, [2, 9], 999), (2, 70, (3,), 1.3, [60], 999),
    (3, 20, (), 1.0, [60, 64], 66), (30, 3, (), 1.0, [4], 999), (40, 2, (1,), 1.0, [4], 999),
])
def test_search_matches_its_definition(k, n_new, stop, alpha, lengths, max_length):
    cache = SequenceCache({0: KVCacheNeed(1, 16), 1: StateNeed((1,))}, max_tokens=64 * 100, max_slots=48, dtype=torch.float32, device="cpu")
    step = ScriptedBeams(cache)
    searcher = BeamSearcher(step, cache, max_batch=48, max_length=max_length)
    prompts = [[(7 * i + j) % VOCAB for j in range(n)] for i, n in enumerate(lengths)]
    got = searcher.search(prompts, n_new, BeamParams(k, alpha, k), stop)
    for p, hyps in zip(prompts, got):
        want = _plain_search(p, k, n_new, set(stop), alpha, max_length)
        assert [(h.tokens, h.finish_reason) for h in hyps] == [(t, r) for t, _, r in want]
        for h, (t, lp, _) in zip(hyps, want):
            assert h.log_prob == pytest.approx(lp, abs=1e-5) and h.score == pytest.approx(lp / len(t) ** alpha, abs=1e-5)
    assert cache.live_slots() == [] and cache.paged_groups[0].pool.n_held == 0
    m = searcher.last_metrics
    assert m.prompt_tokens == sum(lengths) and m.decode_steps == len(step.steps) - 1


def test_requests_go_in_batches_and_an_ended_one_leaves():
    cache = SequenceCache({0: KVCacheNeed(1, 16), 1: StateNeed((1,))}, max_tokens=64 * 20, max_slots=7, dtype=torch.float32, device="cpu")
    step = ScriptedBeams(cache)
    searcher = BeamSearcher(step, cache, max_batch=7, max_length=999)
    prompts = [[1, 2], [3], [4, 5, 6], [9]]
    stop = (2, 5, 7, 11, 12, 20)
    got = searcher.search(prompts, 12, BeamParams(3), stop)
    for p, hyps in zip(prompts, got):
        want = _plain_search(p, 3, 12, set(stop), 1.0, 999)[0]
        assert len(hyps) == 1 and hyps[0].tokens == want[0]
    assert step.steps[0] == 2 and step.steps[1] == 6 and 3 in step.steps      # two requests of three beams at a time, then one alone
    assert cache.live_slots() == []


def test_too_few_continuations_and_none_at_all():
    cache = SequenceCache({0: KVCacheNeed(1, 16), 1: StateNeed((1,))}, max_tokens=64 * 40, max_slots=8, dtype=torch.float32, device="cpu")
    for allowed in ([3], [3, 4], [], [5]):
        forbid = [t for t in range(VOCAB) if t not in allowed]
        searcher = BeamSearcher(ScriptedBeams(cache, forbid), cache, max_batch=8, max_length=999)
        stop = (5,)
        got = searcher.search([[1, 2, 3]], 4, BeamParams(4, 1.0, 4), stop)[0]
        want = _plain_search([1, 2, 3], 4, 4, set(stop), 1.0, 999, forbid)
        assert [(h.tokens, h.finish_reason) for h in got] == [(t, r) for t, _, r in want]
        assert cache.live_slots() == []


def test_limits_and_refusals():
    cache = SequenceCache({0: KVCacheNeed(1, 16)}, max_tokens=64 * 10, max_slots=8, dtype=torch.float32, device="cpu")
    searcher = BeamSearcher(None, cache, max_batch=8, max_length=600)
    assert [[h.tokens for h in hyps] for hyps in searcher.search([[1], [2]], 0, BeamParams(2))] == [[[]], [[]]]
    with pytest.raises(GenerationError, match="9 beams"):
        searcher.search([[1]], 4, BeamParams(9))
    with pytest.raises(GenerationError, match="empty prompt"):
        searcher.search([[]], 4, BeamParams(2))
    with pytest.raises(GenerationError, match="cache pages"):
        searcher.search([[1] * 300], 200, BeamParams(4))
    with pytest.raises(GenerationError, match="exceeds"):
        searcher.search([[1] * 700], 4, BeamParams(2))
    with pytest.raises(GenerationError, match="continuations"):
        searcher.search([[1]], 4, BeamParams(8), stop_ids=range(40))
    for bad in (dict(beams=0), dict(beams=2, n_best=3), dict(n_best=0), dict(length_penalty=math.inf)):
        with pytest.raises(ValueError):
            BeamParams(**bad)
    with pytest.raises(ValueError):
        BeamSelector(4, 300)
    # prompts of 100 tokens: a full page for all beams, two more for each
    assert plan_beam_batches([100, 100, 100], 60, 2, 8, 10, 600) == [[0, 1], [2]]
    assert plan_beam_batches([100, 100, 100], 60, 2, 3, 100, 600) == [[0], [1], [2]]
    assert cache.live_slots() == []


def test_a_request_without_beams_that_count_is_over():
    r = BeamRequest(BeamParams(2), 3, 5, 100, frozenset({9}))
    assert r.advance([(-1.0, 0, 4), (-2.0, 0, 9)]) == [0, 0] and r.beams[1][1] == -math.inf      # (one continuation, one ending)
    assert [h.finish_reason for h in r.finished] == [FINISH_STOP]
    assert r.advance([]) == [] and r.done and [h.tokens for h in r.best()] == [[4]] and r.finished[0].finish_reason == FINISH_STUCK
    assert pages_for(65) == 2


def test_moves_are_grouped_by_source():
    sources, firsts, destinations = ops.copy_groups([(3, 1, 5), (0, 2, 7), (3, 4, 5)], 6)
    assert list(sources) == [3, 0] and list(firsts) == [0, 2, 3] and list(destinations) == [1, 4, 2]
    assert [list(a) for a in ops.copy_groups([], 6)] == [[], [0], []]
    for moves, what in [([(6, 0)], "there are 6"), ([(0, -1)], "there are 6"), ([(0, 1), (2, 1)], "two moves"), ([(0, 1), (1, 2)], "source and")]:
        with pytest.raises(ops.KernelError, match=what):
            ops.copy_groups(moves, 6)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.copy_slots(torch.zeros(1, 2, 3), [(0, 1)])
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.beam_select(*[torch.zeros(1, 4)] * 5)


def test_attention_parts_follow_the_gpu_and_the_pages():
    import unittest.mock as mock

    with mock.patch.object(ops, "sm_count", lambda device: 148):
        parts = ops.attention_beams_parts
        assert parts(1, 4, 32, 8, 64, 1024, torch.bfloat16, "cuda") == 16 + 4            # no more than pages
        assert parts(8, 8, 32, 8, 64, 4352, torch.bfloat16, "cuda") <= 3 * 148 // 8
        assert parts(1, 1, 1, 1, 32, 1, torch.float32, "cuda") == 2
        assert parts(4, 2, 256, 256, 128, 100000, torch.bfloat16, "cuda") >= 1


@pytest.mark.parametrize("penalty", [400.0, -400.0, 33.0, float("inf"), float("nan")])
def test_length_penalties_without_a_score_are_refused(penalty):
    """A length to such a power is no number, or 0."""
    with pytest.raises(ValueError, match="length_penalty"):
        BeamParams(2, penalty)


@pytest.mark.parametrize("penalty", [32.0, -32.0])
def test_the_largest_length_penalties_have_scores(penalty):
    request = BeamRequest(BeamParams(2, penalty), 5, 1 << 20, 1 << 21, frozenset({7}))
    request.beams = [([1] * ((1 << 20) - 2), -3.0), ([2] * ((1 << 20) - 2), -4.0)]
    request.advance([(-3.5, 0, 7), (-4.5, 1, 7), (-5.0, 0, 1), (-6.0, 1, 1)])
    assert all(math.isfinite(h.score) for h in request.finished) and len(request.finished) == 2


@pytest.mark.parametrize("seed", range(4))
def test_reordered_rows_are_the_parents_with_windows_too(seed):
    """A child in the place of a sequence that is over keeps the pages they have in common: rows, holders and lengths come out as its parent's."""
    rng = random.Random(seed)
    c = SequenceCache({0: KVCacheNeed(1, 16), 1: KVCacheNeed(1, 16, window=100), 2: StateNeed((3,), torch.float32)}, max_tokens=64 * 80, max_slots=6,
                      dtype=torch.float32, device="cpu", window_slack=64)
    slots = [c.acquire()]
    c.reserve([(slots[0], 70)])
    c.commit(slots[0], 70)
    slots += c.fork([slots[0]] * 5)
    state, = c.slot_groups
    for step in range(300):
        new = [1] * len(slots) if rng.random() < 0.8 else [rng.randint(1, 40) for _ in slots]      # equally long, and not
        try:
            c.reserve(list(zip(slots, new)))
        except CacheFull:
            for s in slots:
                c.release(s)
            slots = [c.acquire()]
            slots += c.fork([slots[0]] * 5)
            continue
        for s, n in zip(slots, new):
            c.commit(s, n)
            state.data[:, s] = float(step * 10 + s)
        parents = [rng.randrange(len(slots)) for _ in slots]
        want = [([g.rows[slots[p]][:pages_for(c.length(slots[p]))] for g in c.paged_groups], c.length(slots[p]), state.data[:, slots[p]].clone())
                for p in parents]
        slots = c.reorder(slots, parents)
        for s, (rows, length, kept) in zip(slots, want):
            assert [g.rows[s][:pages_for(length)] for g in c.paged_groups] == rows and c.length(s) == length and torch.equal(state.data[:, s], kept)
        c.check_invariants()
