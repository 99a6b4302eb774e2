"""Beam search through the engine's entry point and the command line: against a plain search over the plain implementation's
logits, and for every decoder of the library against the log probabilities that a fresh pass over each hypothesis gives."""
import importlib
import json
import subprocess

import pytest
import torch

import plain_llama as P
from conftest import BF16_EPS, ROOT, TINY, make_model_dir, plain_inputs, random_prompts

pytestmark = pytest.mark.gpu
SCALE = {"embed_tokens": 8.0, "lm_head": 8.0}


def _plain_beams(cfg, w, prompt, k, n_new, stop, alpha):
    """The search by its definition on the plain implementation's float32 logits, log probabilities in 64 bits."""
    beams, finished = [([], 0.0)], []
    rank = lambda h: -(h[1] / len(h[0]) ** alpha)
    while True:
        found = []
        for toks, lp in beams:
            row = torch.log_softmax(P.forward(cfg, w, prompt + toks)[-1].double(), dim=0)
            best = torch.topk(row, min(len(row), k * (1 + len(stop)))).indices.tolist()
            found += [(toks + [t], lp + float(row[t])) for t in best]
        found.sort(key=lambda c: -c[1])
        finished = sorted(finished + [h for h in found[:k] if h[0][-1] in stop], key=rank)[:k]
        beams = [h for h in found if h[0][-1] not in stop][:k]
        n = len(beams[0][0])
        if n >= n_new:
            return sorted(finished + beams, key=rank)[:k]
        if len(finished) == k and beams[0][1] / n_new ** alpha <= finished[-1][1] / len(finished[-1][0]) ** alpha:
            return finished


@pytest.mark.parametrize("name, k, n_new, lengths", [("A", 3, 8, [5, 11, 17]), ("B", 4, 10, [1, 7, 30, 64]), ("B", 6, 6, [60])])
@pytest.mark.parametrize("stops", [0, 2])
def test_float32_search_matches_plain(session_tmp, name, k, n_new, lengths, stops):
    from gpullama3.java_b200.engine.api import Engine

    cfg_json, norm_std = TINY[name]
    d = make_model_dir(session_tmp, cfg_json, seed=21, norm_std=norm_std, scale=SCALE)
    cfg, w = plain_inputs(d)
    prompts = random_prompts(cfg["vocab_size"], lengths, seed=2)
    engine = Engine.from_folder(d, dtype="float32", max_tokens=64 * 32, max_batch=12)
    free = [_plain_beams(cfg, w, p, k, n_new, set(), 1.0) for p in prompts]
    stop = {free[0][0][0][1], free[-1][0][0][2]} if stops else set()
    got = engine.beam_search(prompts, k, n_new, n_best=k, stop_ids=stop, return_hypotheses=True)
    for p, hyps, plain in zip(prompts, got, free):
        want = _plain_beams(cfg, w, p, k, n_new, stop, 1.0) if stop else plain
        assert [h.tokens for h in hyps] == [t for t, _ in want]
        for h, (t, lp) in zip(hyps, want):
            assert abs(h.log_prob - lp) <= 1e-4 * len(t) and h.finish_reason == ("stop" if t[-1] in stop else "length")
    assert engine.cache.live_slots() == []
    engine.cache.check_invariants()
    assert all(g.pool.n_free == g.pool.n_pages for g in engine.cache.paged_groups)
    # again, by recorded steps from the first on: the same
    again = engine.beam_search(prompts, k, n_new, n_best=k, stop_ids=stop, return_hypotheses=True)
    assert [[(h.tokens, h.log_prob) for h in hyps] for hyps in again] == [[(h.tokens, h.log_prob) for h in hyps] for hyps in got]
    assert engine.beam_search(prompts, k, n_new, stop_ids=stop) == [hyps[0].tokens for hyps in got]
    m = engine.last_metrics
    assert m.prompt_tokens == sum(lengths) and m.decode_steps > 0
    assert engine.generate(prompts, max_new_tokens=4, stop_ids=()) and engine.last_metrics.generated_tokens == 4 * len(prompts)


def test_one_beam_is_the_greedy_continuation(session_tmp):
    from gpullama3.java_b200.engine.api import Engine

    d = make_model_dir(session_tmp, TINY["B"][0], seed=21, norm_std=0.1, scale=SCALE)
    prompts = random_prompts(384, [7, 63, 100], seed=5)
    engine = Engine.from_folder(d, dtype="float32", max_tokens=64 * 12, max_batch=4)
    assert engine.beam_search(prompts, 1, 9, stop_ids=()) == engine.generate(prompts, max_new_tokens=9, stop_ids=())


def _rescore(engine, prompt, hyp):
    """The log probabilities of a hypothesis' tokens in a fresh pass of the prompt with them behind it; the largest logit."""
    from gpullama3.java_b200.engine.api import SequenceInput

    slot = engine.cache.acquire()
    try:
        tokens = prompt + hyp.tokens[:-1]
        logits = engine.step([SequenceInput(slot, tokens, list(range(len(prompt) - 1, len(tokens))))]).double()
    finally:
        engine.cache.release(slot)
    lp = torch.log_softmax(logits, dim=1)
    return float(lp[torch.arange(len(hyp.tokens)), torch.tensor(hyp.tokens)].sum()), float(logits.abs().max())


# Two float32 passes are each within 2e-5 of the largest logit from the plain implementation (conftest), so their log probabilities
# within 2 * 2 * 2e-5 of it a token.  bfloat16 passes: 4 * 2^-8 in place of 2e-5.
def _check_hypotheses(engine, prompts, got, step_error):
    for p, hyps in zip(prompts, got):
        assert [h.score for h in hyps] == sorted((h.score for h in hyps), reverse=True)
        assert len({tuple(h.tokens) for h in hyps}) == len(hyps)
        for h in hyps:
            lp, scale = _rescore(engine, p, h)
            assert abs(lp - h.log_prob) <= 4 * step_error * scale * len(h.tokens), (h, lp, scale)


FAMILIES = [("guduzen", "A"), ("guduzen", "B"), ("pekerax", "A"), ("pekerax", "B"), ("gatuzen", "A"), ("gatuzen", "D"), ("bisudra", "A"), ("bisudra", "C"),
            ("fazezen", "A"), ("fazezen", "C"), ("zanezen", "A"), ("zanezen", "B")]


@pytest.mark.parametrize("family, name", FAMILIES)
def test_every_decoders_caches_and_states_follow_the_beams(session_tmp, family, name):
    from gpullama3.java_b200.engine.api import Engine

    helpers = importlib.import_module(f"{family}_helpers")
    d = getattr(helpers, f"make_{family}_dir")(session_tmp, helpers.CONFIGS[name], seed=11)
    engine = Engine.from_folder(d, dtype="float32", max_tokens=64 * 40, max_batch=10)
    cfg = json.loads((d / "config.json").read_text())
    prompts = random_prompts(cfg.get("vocab") or cfg["vocab_size"], [62, 9, 130], seed=3)
    got = engine.beam_search(prompts, 5, 7, n_best=5, stop_ids=(), return_hypotheses=True)
    assert all(len(h.tokens) == 7 and h.finish_reason == "length" for hyps in got for h in hyps)
    _check_hypotheses(engine, prompts, got, 2e-5)
    assert engine.cache.live_slots() == []
    engine.cache.check_invariants()


WIDE = {"architectures": ["LlamaForCausalLM"], "num_hidden_layers": 2, "hidden_size": 256, "num_attention_heads": 8, "num_key_value_heads": 2,
        "head_dim": 64, "intermediate_size": 512, "vocab_size": 3000, "rope_theta": 10000.0, "rope_scaling": None, "rms_norm_eps": 1e-5,
        "tie_word_embeddings": False, "max_position_embeddings": 4096}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [True, False])
def test_search_over_long_shared_prompts(session_tmp, dtype, graphs):
    """Many full pages shared by the beams, in recorded steps and in steps launched one by one: the attention of groups runs."""
    from gpullama3.java_b200.engine.api import Engine
    from gpullama3.java_b200.kernels import ops

    d = make_model_dir(session_tmp, WIDE, seed=4, scale={"embed_tokens": 8.0, "lm_head": 4.0, "q_proj": 3.0, "k_proj": 3.0})
    engine = Engine.from_folder(d, dtype=dtype, max_tokens=64 * 200, max_batch=20)
    engine.step_fn.use_graphs = graphs
    prompts = random_prompts(3000, [1100, 64, 333, 190, 961], seed=6)
    launches = lambda: sum(n for name, n in ops.launches_by_kernel().items() if name.startswith("attention_decode_beams"))
    before = launches()
    got = engine.beam_search(prompts, 4, 70, n_best=4, stop_ids=(), return_hypotheses=True)      # (beams fill pages of their own)
    assert launches() > before
    _check_hypotheses(engine, prompts, got, 2e-5 if dtype == "float32" else 4 * BF16_EPS)
    if not graphs:
        return
    plain = Engine.from_folder(d, dtype=dtype, max_tokens=64 * 200, max_batch=20)
    plain.step_fn.use_graphs = False
    other = plain.beam_search(prompts, 4, 70, n_best=4, stop_ids=(), return_hypotheses=True)
    assert [h.tokens for hyps in other for h in hyps[:1]] == [h.tokens for hyps in got for h in hyps[:1]] or dtype == "bfloat16"


def test_searches_and_generations_take_turns_in_one_cache(session_tmp):
    """Slots and pages go from one to the other, recorded steps of both stay right."""
    from gpullama3.java_b200.engine.api import Engine

    d = make_model_dir(session_tmp, TINY["B"][0], seed=21, norm_std=0.1, scale=SCALE)
    prompts = random_prompts(384, [40, 63, 100, 12, 70], seed=8)
    fresh = lambda: Engine.from_folder(d, dtype="float32", max_tokens=64 * 24, max_batch=6)
    want_g = fresh().generate(prompts, max_new_tokens=20, stop_ids=())
    want_b = fresh().beam_search(prompts, 3, 20, n_best=3, stop_ids=())
    engine = fresh()
    for _ in range(2):
        assert engine.generate(prompts, max_new_tokens=20, stop_ids=()) == want_g
        assert engine.beam_search(prompts, 3, 20, n_best=3, stop_ids=()) == want_b
    assert engine.beam_search(prompts, 3, 20, length_penalty=0.0, stop_ids=()) == [hyps[0] for hyps in want_b]


def test_steps_of_beams_refuse(session_tmp):
    from gpullama3.java_b200.engine.api import Engine, SequenceInput
    from gpullama3.java_b200.engine.step import StepError
    from gpullama3.java_b200.sampling.sampler import BeamSelector

    d = make_model_dir(session_tmp, TINY["B"][0], seed=21, norm_std=0.1, scale=SCALE)
    engine = Engine.from_folder(d, dtype="float32", max_tokens=64 * 6, max_batch=4)
    a = engine.cache.acquire()
    engine.step([SequenceInput(a, [1, 2, 3], [2])])
    b = engine.cache.fork([a])[0]
    c = engine.cache.acquire()
    engine.step([SequenceInput(c, [1, 2], [1])])
    one = lambda s: SequenceInput(s, [5], [0])
    step, selector = engine.step_fn.decode_beams, BeamSelector(2, 4)
    with pytest.raises(StepError, match="groups of 2"):
        step([one(a)], selector, [0.0])
    with pytest.raises(StepError, match="groups of 2"):
        step([one(a), one(b)], selector, [0.0])
    with pytest.raises(StepError, match="one token"):
        step([one(a), SequenceInput(b, [5, 6], [0])], selector, [0.0, 0.0])
    with pytest.raises(StepError, match="equally long"):
        step([one(a), one(c)], selector, [0.0, 0.0])
    with pytest.raises(StepError, match="twice"):
        step([one(a), one(a)], selector, [0.0, 0.0])
    found = step([one(a), one(b)], selector, [0.0, -1.0])
    assert len(found) == 1 and len(found[0]) == 4 and found[0][0][1] == 0


def test_command_line_searches(session_tmp):
    d = make_model_dir(session_tmp, TINY["B"][0], seed=21, norm_std=0.1, scale=SCALE)
    from gpullama3.java_b200.engine.api import Engine

    want = Engine.from_folder(d, dtype="float32", max_tokens=64 * 12, max_batch=8).beam_search([[5, 17, 3], [9] * 70], 4, 6, length_penalty=0.5)
    r = subprocess.run([str(ROOT / "bin" / "llama-b200"), "--model", str(d), "--dtype", "float32", "--prompt", "5 17 3",
                        "--prompt", " ".join(["9"] * 70), "-n", "6", "--beams", "4", "--length-penalty", "0.5"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    assert [[int(t) for t in line.split()] for line in r.stdout.strip().splitlines()] == want
    assert "achieved tok/s" in r.stderr


@pytest.mark.parametrize("family, name", [("llama", "B"), ("guduzen", "A"), ("gatuzen", "A")])
def test_forked_sequences_go_on_by_ordinary_steps(session_tmp, family, name):
    """Forks of one sequence, continued by single tokens (recorded steps), by chunks and by chunks of unequal length in one step, give
    the logits of sequences that were told the same from their beginning."""
    from conftest import assert_close_logits
    from gpullama3.java_b200.engine.api import Engine, SequenceInput

    if family == "llama":
        d = make_model_dir(session_tmp, TINY[name][0], seed=21, norm_std=0.1, scale=SCALE)
    else:
        helpers = importlib.import_module(f"{family}_helpers")
        d = getattr(helpers, f"make_{family}_dir")(session_tmp, helpers.CONFIGS[name], seed=11)
    engine = Engine.from_folder(d, dtype="float32", max_tokens=64 * 40, max_batch=8)
    vocab = engine.config.vocab_size
    prompt, *more = random_prompts(vocab, [70, 5, 64, 1, 130], seed=4)
    cache, step = engine.cache, engine.step
    first = cache.acquire()
    step([SequenceInput(first, prompt, [])])
    slots = [first] + cache.fork([first] * (len(more) - 1))
    told = [list(prompt) for _ in more]
    for turn in range(3):                             # single tokens of all, twice the recorded step
        tokens = random_prompts(vocab, [1] * len(more), seed=50 + turn)
        got = step([SequenceInput(s, t, [0]) for s, t in zip(slots, tokens)])
        for i, t in enumerate(tokens):
            told[i] += t
    chunks = step([SequenceInput(s, t, [len(t) - 1]) for s, t in zip(slots, more)])
    again = cache.fork([slots[3]])[0]                 # a fork of a fork, behind a page border or not
    tail = random_prompts(vocab, [2], seed=9)[0]
    last = step([SequenceInput(again, tail, [0, 1])])
    for rows, histories in ((got, told), (chunks, [a + b for a, b in zip(told, more)])):
        for i, history in enumerate(histories):
            s = cache.acquire()
            want = step([SequenceInput(s, history, [len(history) - 1])])
            cache.release(s)
            assert_close_logits(rows[i:i + 1], want, torch.float32, f"sequence {i}")
    s = cache.acquire()
    history = told[3] + more[3] + tail
    want = step([SequenceInput(s, history, [len(history) - 2, len(history) - 1])])
    assert_close_logits(last, want, torch.float32, "fork of a fork")
    cache.check_invariants()
    for s in cache.live_slots():
        cache.release(s)


def test_more_groups_than_one_attention_call_takes(session_tmp):
    """Such a step reads every sequence for itself: the same as in smaller batches."""
    from gpullama3.java_b200.engine.api import Engine
    from gpullama3.java_b200.kernels import ops

    cfg_json, norm_std = TINY["B"]
    d = make_model_dir(session_tmp, cfg_json, seed=21, norm_std=norm_std, scale=SCALE)
    prompts = random_prompts(cfg_json["vocab_size"], [1 + i % 3 for i in range(260)], seed=9)
    H, KVH = cfg_json["num_attention_heads"], cfg_json["num_key_value_heads"]
    assert not ops.attention_beams_takes(260, 8, H, KVH) and ops.attention_beams_takes(32, 8, H, KVH)
    found = [Engine.from_folder(d, dtype="float32", max_tokens=64 * 2100, max_batch=n).beam_search(prompts, 8, 3, stop_ids=(), return_hypotheses=True)
             for n in (8 * 260, 8 * 32)]
    # (other kernels for other numbers of rows: the same tokens but where two scores are as near as float32 is)
    for a, b in zip(*found):
        assert a.tokens == b.tokens or abs(a.log_prob - b.log_prob) <= 1e-4 * len(a.tokens)
