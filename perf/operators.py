"""What a beam search asks of the GPU beside the model's own layers, as cases that can be timed and checked:

* ``select``: the best continuations of every request's beams, over beams and vocabulary together (``ops.beam_select``);
* ``pages``: cache pages that two beams share and one of them is about to write, copied for it (``ops.copy_pages``);
* ``slots``: recurrent states of fixed size, copied to the beams that continue the same parent (``ops.copy_slots``);
* ``attend``: one decode step's attention of beams over the pages that all beams of a request share and the pages that each
  has for itself (``ops.attention_decode_beams``).

Sizes are those of the library's models: the shapes of Llama 3.2 1B and 3B and of Llama 3.1 8B, and the delta rule's state of
the Guduzen decoder of the 1B shape's width."""
import math
import random

import numpy as np
import torch

own = False             # False: the plain forms, elementary torch operations; True: the library's kernels

DEVICE = "cuda"
PAGE = 64               # positions of a cache page
F64 = torch.float64


def listed():
    return [
        # one chat at 4 beams: a step's selection is a matter of latency
        {"name": "select chat", "kind": "select", "groups": 1, "beams": 4, "vocab": 128256, "keep": 8, "pad": 0, "masked": 0.0,
         "first": False},
        # the first step of some requests, whose prompts have one beam each so far, over an odd vocabulary in wider rows, a
        # part of it forbidden
        {"name": "select first step", "kind": "select", "groups": 3, "beams": 5, "vocab": 32003, "keep": 10, "pad": 13,
         "masked": 0.6, "first": True},
        # a served batch: 8 requests of 8 beams
        {"name": "select batch", "kind": "select", "groups": 8, "beams": 8, "vocab": 128256, "keep": 16, "pad": 0, "masked": 0.0,
         "first": False},
        # many beams, as for a list of the best answers
        {"name": "select wide", "kind": "select", "groups": 8, "beams": 32, "vocab": 128256, "keep": 64, "pad": 0, "masked": 0.0,
         "first": False},
        # one chat at 4 beams, all of which continue the same parent: its last page, not full, for three more
        {"name": "pages chat 1b", "kind": "pages", "layers": 16, "heads": 8, "dim": 64, "dtype": "bfloat16", "pool": 24,
         "copies": 3, "sources": 1},
        # 8 requests of 8 beams on the 8B shape
        {"name": "pages batch 8b", "kind": "pages", "layers": 32, "heads": 8, "dim": 128, "dtype": "bfloat16", "pool": 64,
         "copies": 40, "sources": 22},
        # the same in true 32 bits on a smaller scale, with the 3B shape's layers
        {"name": "pages float32 3b", "kind": "pages", "layers": 28, "heads": 8, "dim": 128, "dtype": "float32", "pool": 24,
         "copies": 13, "sources": 7},
        # the delta rule's states of 4 layers with the inputs of their convolutions (32 heads of 64 x 64, 3 inputs of 3 x 2,048)
        {"name": "slots guduzen", "kind": "slots", "layers": 4, "floats": 32 * 64 * 64 + 3 * 3 * 2048, "pool": 64, "copies": 37,
         "sources": 19},
        # one chat at 4 beams
        {"name": "attend chat 1b", "kind": "attend", "groups": "14:25", "beams": 4, "heads": 32, "kv_heads": 8, "dim": 64,
         "dtype": "bfloat16", "window": 0},
        # the benchmark's context at a served batch
        {"name": "attend batch 1b", "kind": "attend", "groups": "8*63:70", "beams": 8, "heads": 32, "kv_heads": 8, "dim": 64,
         "dtype": "bfloat16", "window": 0},
        # unequal long documents on the 8B shape
        {"name": "attend documents 8b", "kind": "attend", "groups": "251:133,97:64,181:1,30:300", "beams": 4, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "window": 0},
        # true 32 bits
        {"name": "attend float32 1b", "kind": "attend", "groups": "23:40,9:121", "beams": 5, "heads": 32, "kv_heads": 8, "dim": 64,
         "dtype": "float32", "window": 0},
    ]


def _log_uniform(rng, lo, hi):
    return lo if hi <= lo else min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["select", "select", "pages", "slots", "attend", "attend", "attend"])
    if kind == "select":
        beams = _log_uniform(rng, 1, 32)
        vocab = rng.choice([128256, 32000, 50257, _log_uniform(rng, 256, 200000)])
        groups = max(1, min(_log_uniform(rng, 1, 32), 32_000_000 // (beams * vocab)))
        return {"kind": kind, "groups": groups, "beams": beams, "vocab": vocab,
                "keep": beams * rng.choice([1, 2, 3]), "pad": rng.choice([0, 0, 3, 64]),
                "masked": rng.choice([0.0, 0.0, 0.5, 0.97]), "first": rng.random() < 0.25}
    if kind == "pages":
        layers, heads, dim = rng.choice([(16, 8, 64), (28, 8, 128), (32, 8, 128), (2, 2, 16), (3, 1, 32), (6, 3, 96)])
        copies = _log_uniform(rng, 1, 30)
        sources = rng.randint(1, copies)
        return {"kind": kind, "layers": layers, "heads": heads, "dim": dim, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])
                if dim < 128 or copies < 16 else "bfloat16", "pool": copies + sources + rng.randint(0, 16), "copies": copies,
                "sources": sources}
    if kind == "slots":
        layers, floats = rng.randint(1, 8), rng.choice([131072 + 18432, 6144, _log_uniform(rng, 3, 200000)])
        copies = min(_log_uniform(rng, 1, 64), 28_000_000 // (layers * floats))
        sources = rng.randint(1, copies)
        return {"kind": kind, "layers": layers, "floats": floats,
                "pool": copies + sources + rng.randint(0, 8), "copies": copies, "sources": sources}
    heads, kv_heads, dim, most = rng.choice([(32, 8, 64, 24000), (24, 8, 128, 16000), (32, 8, 128, 16000), (8, 8, 96, 8000), (12, 1, 32, 8000)])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    most = most // 4 if dtype == "float32" else most
    beams = _log_uniform(rng, 2, 16)
    groups = _log_uniform(rng, 1, 64 // beams)
    pages = _log_uniform(rng, 1, max(1, 4 * most // (PAGE * groups * max(4, beams))))
    lens = [f"{rng.randint(pages // 3, pages)}:{rng.choice([1, 17, 64, 65, rng.randint(1, 250)])}" for _ in range(groups)]
    return {"kind": kind, "groups": ",".join(lens), "beams": beams, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "window": rng.choice([0, 0, 0, 1000])}


# ---- inputs


def _group_lengths(case):
    """Per group: the pages that its beams share, and the positions that each beam has behind them."""
    out = []
    for part in case["groups"].split(","):
        count, _, rest = part.rpartition("*")
        pages, own_positions = rest.split(":")
        out += [(int(pages), int(own_positions))] * int(count or 1)
    return out


def _generator(seed):
    return torch.Generator(DEVICE).manual_seed(int(seed) * 7919 + 101)


def _fan_out(case, seed):
    """(source, destination) pairs: every source at least once, no number among sources and destinations twice."""
    rng = random.Random(int(seed) * 104729 + 7)
    numbers = rng.sample(range(case["pool"]), case["sources"] + case["copies"])
    sources, rest = numbers[:case["sources"]], numbers[case["sources"]:]
    chosen = sources + [rng.choice(sources) for _ in range(case["copies"] - case["sources"])]
    return sorted(zip(chosen, rest))


def _fills(case, seed):
    """How many positions of each source page are in use."""
    rng = random.Random(int(seed) * 31337 + 3)
    return {s: rng.randint(1, PAGE - 1) for s in sorted({s for s, _ in _fan_out(case, seed)})}


def prepare(case, seed):
    state = dict(case)
    g = _generator(seed)
    if case["kind"] == "select":
        G, B, V = case["groups"], case["beams"], case["vocab"]
        wide = torch.randn((G * B, V + case["pad"]), generator=g, device=DEVICE).mul_(2.5)
        logits = wide[:, :V]
        if case["masked"]:      # tokens that a grammar does not allow here
            logits[torch.rand((G * B, V), generator=g, device=DEVICE) < case["masked"]] = -math.inf
        scores = torch.rand((G, B), generator=g, device=DEVICE).mul_(-4.0).sub_(20.0)
        if case["first"]:       # only the prompt's own row counts
            scores.fill_(-math.inf)
            scores[:, 0] = 0.0
        state.update(logits=logits, scores=scores)
    elif case["kind"] == "pages":
        E, P, H, D = case["layers"], case["pool"], case["heads"], case["dim"]
        dtype = getattr(torch, case["dtype"])
        state.update(k=torch.randn((E, P, H, PAGE, D), generator=g, device=DEVICE).to(dtype),
                     v=torch.randn((E, P, H, D, PAGE), generator=g, device=DEVICE).to(dtype))
        fills = _fills(case, seed)
        state["moves"] = [(s, d, fills[s]) for s, d in _fan_out(case, seed)]
    elif case["kind"] == "slots":
        state["data"] = torch.randn((case["layers"], case["pool"], case["floats"]), generator=g, device=DEVICE)
        state["moves"] = _fan_out(case, seed)
    else:
        _prepare_attend(case, seed, g, state)
    return state


def _prepare_attend(case, seed, g, state):
    B, H, G, D = case["beams"], case["heads"], case["kv_heads"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    lengths = _group_lengths(case)
    own_pages = [-(-tail // PAGE) for _, tail in lengths]
    n_pages = sum(pages + B * o for (pages, _), o in zip(lengths, own_pages))
    numbers = list(range(n_pages))
    random.Random(int(seed) * 65537 + 11).shuffle(numbers)
    rows, kv_lens = [], []
    for (pages, tail), o in zip(lengths, own_pages):
        shared = [numbers.pop() for _ in range(pages)]
        for _ in range(B):
            rows.append(shared + [numbers.pop() for _ in range(o)])
            kv_lens.append(PAGE * pages + tail)
    width = max(len(r) for r in rows)
    table = torch.zeros((len(rows), width), dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
    # queries and keys whose scores spread by about two, as trained heads have it
    q = torch.randn((len(rows), H * D), generator=g, device=DEVICE).mul_(1.4)
    k = torch.randn((n_pages, G, PAGE, D), generator=g, device=DEVICE).mul_(1.4)
    state.update(q=q.to(dtype), k=k.to(dtype), v=torch.randn((n_pages, G, D, PAGE), generator=g, device=DEVICE).to(dtype),
                 table=table.to(DEVICE), kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device=DEVICE),
                 shared=torch.tensor([p for p, _ in lengths], dtype=torch.int32, device=DEVICE),
                 lengths=lengths, kv_host=kv_lens)
    if own:
        from gpullama3.java_b200.kernels import ops
        state["parts"] = ops.attention_beams_parts(len(lengths), B, H, G, D, width * PAGE, dtype, q.device)


# ---- the calls


def run(state):
    return (_own if own else _plain)[state["kind"]](state)


def _own_select(state):
    from gpullama3.java_b200.kernels import ops
    shape, device = (state["groups"], state["keep"]), state["logits"].device
    scores = torch.empty(shape, dtype=torch.float32, device=device)
    beams, tokens = (torch.empty(shape, dtype=torch.int32, device=device) for _ in range(2))
    ops.beam_select(state["logits"], state["scores"], scores, beams, tokens)
    return scores, beams, tokens


def _own_pages(state):
    from gpullama3.java_b200.kernels import ops
    ops.copy_pages(state["k"], state["v"], state["moves"])
    return state["k"], state["v"]


def _own_slots(state):
    from gpullama3.java_b200.kernels import ops
    ops.copy_slots(state["data"], state["moves"])
    return state["data"]


def _own_attend(state):
    from gpullama3.java_b200.kernels import ops
    q, out = state["q"], torch.empty_like(state["q"])
    ops.attention_decode_beams(q, q.shape[1], out, state["kv_lens"], state["table"], state["shared"], state["k"], state["v"],
                               state["heads"], state["kv_heads"], state["dim"], state["window"], state["parts"])
    return out


_own = {"select": _own_select, "pages": _own_pages, "slots": _own_slots, "attend": _own_attend}


def _plain_select(state):
    """Every row's best tokens by logit (ties: the lower token), their totals score + log softmax in 64 bits, and of all beams'
    together the best (ties: the lower beam, then the row's order).  A row whose softmax does not exist gives none."""
    G, B, keep = state["groups"], state["beams"], state["keep"]
    x = state["logits"] + 0.0                                                # (-0 counts as 0)
    V = x.shape[1]
    top = x.amax(dim=1, keepdim=True)
    lse = top.to(F64) + torch.log(torch.exp(x.to(F64) - top.to(F64)).sum(dim=1, keepdim=True))
    bits = x.view(torch.int32).to(torch.int64)
    rising = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF)                 # rises with the number
    places = torch.arange(V, device=x.device)
    order = rising * 4294967296 + (4294967295 - places)                      # unique: ties go to the lower token
    chosen = torch.topk(order, min(keep, V), dim=1, sorted=True).values
    tokens = 4294967295 - (chosen & 4294967295)
    totals = state["scores"].reshape(G * B, 1).to(F64) + (torch.gather(x, 1, tokens).to(F64) - lse)
    totals = torch.where(torch.isfinite(totals), totals, -math.inf)
    n = tokens.shape[1]
    best, place = torch.sort(totals.view(G, B * n), dim=1, descending=True, stable=True)
    best, place = best[:, :keep], place[:, :keep]
    if best.shape[1] < keep:
        fill = keep - best.shape[1]
        best = torch.cat([best, best.new_full((G, fill), -math.inf)], dim=1)
        place = torch.cat([place, place.new_zeros((G, fill))], dim=1)
    none = best == -math.inf
    token = torch.gather(tokens.reshape(G, B * n), 1, place)
    return (best.to(torch.float32), torch.where(none, -1, place // n).to(torch.int32), torch.where(none, -1, token).to(torch.int32))


def _plain_pages(state):
    k, v = state["k"], state["v"]
    for s, d, n in state["moves"]:
        k[:, d, :, :n] = k[:, s, :, :n]
        v[:, d, :, :, :n] = v[:, s, :, :, :n]
    return k, v


def _plain_slots(state):
    data, moves = state["data"], state["moves"]
    data[:, [d for _, d in moves]] = data[:, [s for s, _ in moves]]
    return data


def _plain_attend(state):
    B, H, G, D, window = state["beams"], state["heads"], state["kv_heads"], state["dim"], state["window"]
    rep, out = H // G, torch.empty_like(state["q"])
    for i, (pages, tail) in enumerate(state["lengths"]):
        rows = slice(i * B, (i + 1) * B)
        kv_len = PAGE * pages + tail
        q = state["q"][rows].view(B, G, rep, D).to(torch.float32) / math.sqrt(D)
        table = state["table"][rows].long()
        n_own = -(-tail // PAGE)
        ks = state["k"][table[0, :pages]].to(torch.float32).permute(1, 0, 2, 3).reshape(G, PAGE * pages, D)
        vs = state["v"][table[0, :pages]].to(torch.float32).permute(1, 0, 3, 2).reshape(G, PAGE * pages, D)
        mine = table[:, pages:pages + n_own]
        ko = state["k"][mine].to(torch.float32).permute(0, 2, 1, 3, 4).reshape(B, G, PAGE * n_own, D)[:, :, :tail]
        vo = state["v"][mine].to(torch.float32).permute(0, 2, 1, 4, 3).reshape(B, G, PAGE * n_own, D)[:, :, :tail]
        s = torch.cat([torch.einsum("bgrd,gkd->bgrk", q, ks), torch.einsum("bgrd,bgkd->bgrk", q, ko)], dim=3)
        if window and kv_len > window:
            s[..., :kv_len - window] = -math.inf
        p = torch.exp(s - s.amax(dim=3, keepdim=True))
        total = p.sum(dim=3, keepdim=True)
        o = torch.einsum("bgrk,gkd->bgrd", p[..., :PAGE * pages], vs) + torch.einsum("bgrk,bgkd->bgrd", p[..., PAGE * pages:], vo)
        out[rows] = (o / total).reshape(B, H * D).to(out.dtype)
    return out


_plain = {"select": _plain_select, "pages": _plain_pages, "slots": _plain_slots, "attend": _plain_attend}


# ---- what a pass cannot do without


def work(case):
    if case["kind"] == "select":
        rows = case["groups"] * case["beams"]
        read = case["groups"] if case["first"] else rows      # a beam that does not count need not be read
        return {"bytes": 4 * read * case["vocab"] + 4 * rows + 12 * case["groups"] * case["keep"], "flops": 4 * read * case["vocab"]}
    if case["kind"] == "pages":
        position = 2 * case["layers"] * case["heads"] * case["dim"] * (2 if case["dtype"] == "bfloat16" else 4)
        return {"bytes": position * 32 * (case["sources"] + case["copies"]), "flops": 0}   # (half a page on average)
    if case["kind"] == "slots":
        return {"bytes": 4 * case["layers"] * case["floats"] * (case["sources"] + case["copies"]), "flops": 0}
    B, H, G, D, window = case["beams"], case["heads"], case["kv_heads"], case["dim"], case["window"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    n_bytes = flops = 0
    for pages, tail in _group_lengths(case):
        seen = PAGE * pages + tail if not window else min(window, PAGE * pages + tail)
        shared = max(0, seen - tail)
        n_bytes += 2 * G * D * size * (shared + B * min(tail, seen)) + 2 * B * H * D * size
        flops += 4 * B * H * D * seen
    return {"bytes": n_bytes, "flops": flops}


# ---- the definitions in 64 bits


def exact(case, seed):
    if case["kind"] in ("pages", "slots"):
        return None         # copies: nothing is computed
    state = prepare(case, seed)
    if case["kind"] == "select":
        return _exact_select(state)
    return _exact_attend(state)


def _exact_select(state):
    G, B, keep = state["groups"], state["beams"], state["keep"]
    scores = state["scores"].cpu().numpy().astype(np.float64)
    out = np.full((G, keep), -np.inf), np.full((G, keep), -1, np.int32), np.full((G, keep), -1, np.int32)
    for g in range(G):
        found = []
        for b in range(B):
            row = state["logits"][g * B + b].cpu().numpy().astype(np.float64)
            if not np.isfinite(scores[g, b]) or not np.isfinite(row.max()):
                continue
            lse = row.max() + math.log(np.sum(np.exp(row - row.max())))
            if len(row) > keep:
                border = np.partition(row, len(row) - keep)[len(row) - keep]
                at = np.nonzero(row >= border)[0]
            else:
                at = np.arange(len(row))
            found += [(-(scores[g, b] + (row[t] - lse)), b, -row[t], int(t)) for t in at if row[t] > -np.inf]
        for i, (total, b, _, t) in enumerate(sorted(found)[:keep]):
            out[0][g, i], out[1][g, i], out[2][g, i] = -total, b, t
    return tuple(torch.from_numpy(o) for o in out)


def _exact_attend(state):
    H, G, D, window = state["heads"], state["kv_heads"], state["dim"], state["window"]
    q = state["q"].to(F64)
    out = torch.empty_like(q)
    for r, kv_len in enumerate(state["kv_host"]):
        pages = state["table"][r, :-(-kv_len // PAGE)].long()
        first = max(0, kv_len - window) if window else 0
        for h in range(G):
            keys = state["k"][pages, h].to(F64).reshape(-1, D)[first:kv_len]
            values = state["v"][pages, h].to(F64).transpose(1, 2).reshape(-1, D)[first:kv_len]
            heads = slice(h * (H // G) * D, (h + 1) * (H // G) * D)
            weights = torch.softmax(q[r, heads].view(H // G, D) @ keys.T / math.sqrt(D), dim=1)
            out[r, heads] = (weights @ values).reshape(-1)
    return out
