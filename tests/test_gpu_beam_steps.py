"""Steps of a beam search whose attention reads shared pages once, against the same steps with every sequence read by itself: forks, children
and their pages in two caches that go through the same, logits compared step by step."""
import importlib
import json
import random

import pytest
import torch

from conftest import BF16_EPS, make_model_dir, random_prompts
from gpullama3.java_b200.engine import step as steps
from gpullama3.java_b200.kernels import fast, ops
from gpullama3.java_b200.sampling.sampler import BeamSelector

pytestmark = pytest.mark.gpu

LLAMA = {"architectures": ["LlamaForCausalLM"], "num_hidden_layers": 2, "hidden_size": 256, "num_attention_heads": 8, "num_key_value_heads": 2,
         "head_dim": 64, "intermediate_size": 512, "vocab_size": 2000, "rope_theta": 10000.0, "rope_scaling": None, "rms_norm_eps": 1e-5,
         "tie_word_embeddings": False, "max_position_embeddings": 4096}
# (in bfloat16 a rounding may choose another expert of a routed layer, and such a row's logits are others: those decoders in float32 alone)
CASES = [(*who, dtype) for who in [("llama", None), ("guduzen", "A"), ("guduzen", "B")] for dtype in ("bfloat16", "float32")]
CASES += [(*who, "float32") for who in [("gatuzen", "A"), ("gatuzen", "D"), ("bisudra", "A"), ("bisudra", "C")]]


def _wherever_it_can(ctx, mixer, dtype, capacity):
    """``beams_share_attention`` without what it says about speed."""
    beams = getattr(ctx, "beams", 1)
    if beams == 1 or not ctx.all_decode or mixer.keep_first or getattr(mixer, "has_terms", False) or getattr(mixer, "chunk", None):
        return False
    return (ops.attention_beams_supported(dtype, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim)
            and ops.attention_beams_takes(ctx.n_seqs // beams, beams, mixer.n_heads, mixer.n_kv_heads))


def _logits_of_steps(monkeypatch, folder, dtype, shared, graphs, prompts, beams, n_steps):
    """The logits [groups * beams, vocab] of every step, and how often the attention of groups was launched."""
    from gpullama3.java_b200.engine.api import Engine, SequenceInput

    monkeypatch.setattr(fast, "beams_share_attention", _wherever_it_can if shared else lambda *args: False)
    engine = Engine.from_folder(folder, dtype=dtype, max_tokens=64 * 120, max_batch=beams * len(prompts))
    step, cache, vocab = engine.step_fn, engine.cache, engine.config.vocab_size
    step.use_graphs = graphs
    seen = []
    run, select = steps.DecodeGraph.run, step.select_beams

    def recorded(self, *args, **kwargs):
        logits = run(self, *args, **kwargs)
        torch.cuda.synchronize()
        seen.append(logits.float().cpu())
        return logits

    def launched(logits, *args):
        seen.append(logits.float().cpu())
        return select(logits, *args)

    if graphs:
        monkeypatch.setattr(steps.DecodeGraph, "run", recorded)
    else:
        monkeypatch.setattr(step, "select_beams", launched)
    launches = lambda: sum(n for name, n in ops.launches_by_kernel().items() if name.startswith("attention_decode_beams"))
    before = launches()
    slots = [[cache.acquire()] for _ in prompts]
    step([SequenceInput(s[0], p, [len(p) - 1]) for s, p in zip(slots, prompts)])
    slots = [s + cache.fork(s * (beams - 1)) for s in slots]
    rng, selector = random.Random(5), BeamSelector(beams, beams)
    for i in range(n_steps):
        # at the end all beams are told the same: they differ by what they have behind the pages that they share
        tokens = [rng.randrange(vocab) for _ in range(len(prompts) * beams)]
        tokens = [tokens[j - j % beams] for j in range(len(tokens))] if i == n_steps - 1 else tokens
        flat = [s for group in slots for s in group]
        step.decode_beams([SequenceInput(s, [t], [0]) for s, t in zip(flat, tokens)], selector, [-0.1] * len(flat))
        if i < n_steps - 14:
            slots = [cache.reorder(group, [rng.randrange(beams) for _ in group]) for group in slots]
        cache.check_invariants()
    monkeypatch.undo()
    return seen, launches() - before


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("family, name, dtype", CASES)
def test_shared_and_separate_attention_give_the_same_logits(monkeypatch, session_tmp, family, name, dtype, graphs):
    """Both ways are as far from the definition as two passes of the engine are: float32 2e-5 of the largest logit each, bfloat16 4 half steps of
    it, 0.5 on average.  What a beam's own pages make of its logits is at least eight times the error seen, so another beam's could not pass."""
    if family == "llama":
        folder = make_model_dir(session_tmp, LLAMA, seed=4, scale={n: 4.0 for n in ("q_proj", "k_proj", "v_proj", "o_proj")})
    else:
        helpers = importlib.import_module(f"{family}_helpers")
        folder = getattr(helpers, f"make_{family}_dir")(session_tmp, helpers.CONFIGS[name], seed=11)
    cfg = json.loads((folder / "config.json").read_text())
    prompts, beams, n_steps = random_prompts(cfg.get("vocab") or cfg["vocab_size"], [62, 9, 130, 200] + [1000] * (family == "llama"), seed=3), 5, 24
    shared, n = _logits_of_steps(monkeypatch, folder, dtype, True, graphs, prompts, beams, n_steps)
    separate, none = _logits_of_steps(monkeypatch, folder, dtype, False, graphs, prompts, beams, n_steps)
    assert n > 0 and none == 0 and len(shared) == len(separate) == n_steps
    most, mean = (2 * 2e-5, 2 * 2e-5) if dtype == "float32" else (2 * 4 * BF16_EPS, 2 * 0.5 * BF16_EPS)
    worst = 0.0
    for a, b in zip(shared, separate):
        scale, err = float(b.abs().max()), (a - b).abs()
        assert torch.isfinite(a).all() and float(err.max()) <= most * scale and float(err.mean()) <= mean * scale
        worst = max(worst, float(err.mean()))
    last = separate[-1].view(len(prompts), beams, -1)[:4]       # (behind 1,000 positions the beams' own 14 weigh too little)
    apart = min(float((g[i] - g[j]).abs().mean()) for g in last for i in range(beams) for j in range(i))
    assert apart >= 8 * worst
