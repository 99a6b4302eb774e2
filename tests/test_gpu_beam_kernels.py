"""The kernels of a beam search against plain implementations in 64 bits: selection over beams and vocabulary, copies of cache pages
and of states, attention of groups of sequences that share their first pages."""
import math

import pytest
import torch

from gpullama3.java_b200.kernels import ops

pytestmark = pytest.mark.gpu
HALF_STEP = 2.0 ** -24      # of float32
INF = math.inf


# ---- selection
#
# The kernel's log sum is off by at most 55 half steps: an exponential by 4 (2 units in the last place), its argument by up to 30 (the
# rounding of x - m where that is below 30; what lies lower weighs nothing), the 32-bit additions of a thread's 16 and a warp's
# lanes by 21.  The score is rounded once more.
LSE_ERROR = 55 * HALF_STEP


def _reference(logits, scores, n):
    """Totals [G, B, V] in 64 bits (-inf: no candidate) and the order of all of a request's candidates."""
    G, B = scores.shape
    x = logits.double().cpu().view(G, B, -1)
    m = x.amax(-1, keepdim=True)
    log_sum = torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    s = scores.double().cpu().unsqueeze(-1)
    total = s + ((x - m) - log_sum)         # (not x - (m + log_sum): at the type's lowest value that loses the second)
    total[~(torch.isfinite(s) & torch.isfinite(m + log_sum)).expand_as(total)] = -INF
    total[x == -INF] = -INF
    order = []
    for g in range(G):
        flat = total[g].flatten()
        best = torch.argsort(flat, descending=True, stable=True)[:n].tolist()
        order.append([divmod(i, x.shape[-1]) for i in best if flat[i] > -INF])
    return total, order


def _select(logits, scores, n, scratch=None):
    G = scores.shape[0]
    outs = (torch.full((G, n), 7.0, device="cuda"), torch.full((G, n), 7, dtype=torch.int32, device="cuda"),
            torch.full((G, n), 7, dtype=torch.int32, device="cuda"))
    ops.beam_select(logits, scores, *outs, scratch)
    return outs


def _check_selection(logits, scores, n, outs=None):
    got_s, got_b, got_t = (o.cpu() for o in (outs or _select(logits, scores, n)))
    total, order = _reference(logits, scores, n)
    for g, want in enumerate(order):
        found = list(zip(got_b[g].tolist(), got_t[g].tolist()))
        k = len(want)
        assert found[k:] == [(-1, -1)] * (n - k) and bool((got_s[g, k:] == -INF).all())
        assert len(set(found[:k])) == k
        for i, (f, w) in enumerate(zip(found, want)):
            tf, tw = float(total[g][f]), float(total[g][w])
            # another candidate only where two beams' totals are nearer than their two rows' errors
            assert f == w or (f[0] != w[0] and abs(tf - tw) <= 2 * LSE_ERROR) or \
                any(abs(tf - float(total[g][o])) <= 2 * LSE_ERROR and o[0] != f[0] for o in want), (g, i, f, w, tf, tw)
            assert abs(float(got_s[g, i]) - tf) <= HALF_STEP * abs(tf) + LSE_ERROR, (g, i, float(got_s[g, i]), tf)


def _logits(rows, V, pad=0, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(rows, V + pad, generator=g) * spread
    return wide.cuda()[:, :V]


def _scores(G, B, seed=0):
    return (-20 - 4 * torch.rand(G, B, generator=torch.Generator().manual_seed(seed + 99))).cuda()


@pytest.mark.parametrize("G, B, V, n, pad", [
    (1, 1, 1, 1, 0), (1, 1, 1, 5, 0), (2, 3, 2, 6, 0), (3, 4, 7, 8, 1), (1, 4, 383, 8, 0), (2, 5, 384, 10, 0), (3, 2, 4095, 4, 1),
    (1, 3, 4096, 6, 0), (2, 3, 4097, 6, 0), (1, 2, 8191, 33, 5), (2, 8, 32003, 16, 13), (1, 4, 128256, 8, 0), (4, 6, 50257, 12, 0),
    (1, 32, 20000, 64, 0), (2, 2, 9000, 256, 0), (1, 1, 30000, 200, 2), (1, 100, 500, 3, 0), (16, 1, 1000, 2, 0),
])
def test_selection_matches_64_bits(G, B, V, n, pad):
    _check_selection(_logits(G * B, V, pad, seed=V + n), _scores(G, B, seed=V), n)


def test_equal_logits_go_by_token_and_equal_beams_by_beam():
    for V, n in [(10, 4), (4100, 40), (20000, 16), (9000, 256)]:
        logits = torch.zeros(6, V, device="cuda")
        s, b, t = _select(logits, torch.zeros(2, 3, device="cuda"), n)
        assert b.tolist() == [[i // V for i in range(n)]] * 2 and t.tolist() == [[i % V for i in range(n)]] * 2
        assert float((s.double() + math.log(V)).abs().max()) <= HALF_STEP * math.log(V) + LSE_ERROR
    # a row repeated: every token of beam 0 stands right before the same token of beams 1 and 2
    row = _logits(1, 5000, seed=3)
    s, b, t = _select(row.expand(3, -1).contiguous(), torch.full((1, 3), -2.5, device="cuda"), 9)
    best = torch.argsort(row[0], descending=True)[:3].tolist()
    assert b[0].tolist() == [0, 1, 2] * 3 and t[0].tolist() == [x for x in best for _ in range(3)]


def test_minus_zero_is_zero():
    logits = torch.full((1, 5000), -50.0, device="cuda")
    logits[0, 4900] = 0.0
    logits[0, 77] = -0.0
    logits[0, 200] = -0.0
    assert _select(logits, torch.zeros(1, 1, device="cuda"), 3)[2].tolist() == [[77, 200, 4900]]


@pytest.mark.parametrize("V", [40, 4500, 32003])
def test_masked_tokens_and_rows_without_a_distribution(V):
    B, n = 7, 12
    logits = _logits(2 * B, V, seed=V)
    gen = torch.Generator().manual_seed(5)
    logits[torch.rand(2 * B, V, generator=gen).cuda() < 0.6] = -INF
    logits[1] = -INF                                  # nothing left
    logits[2, V // 2] = math.nan
    logits[3, 1] = INF
    logits[4] = -INF
    logits[4, V - 1] = 0.25                           # one token: its probability is 1
    logits[B] = torch.finfo(torch.float32).min        # masked by the type's lowest value: still a distribution, if no other is
    logits[B + 1, : V // 2] = torch.finfo(torch.float32).min
    scores = _scores(2, B)
    scores[0, 5], scores[1, 3], scores[1, 4] = -INF, math.nan, INF
    _check_selection(logits, scores, n)
    s, b, t = _select(logits, scores, n)
    assert not {1, 2, 3, 5} & set(b[0].tolist()) and not {3, 4} & set(b[1].tolist())
    # no beam counts: nothing to choose
    s, b, t = _select(logits, torch.full((2, B), -INF, device="cuda"), n)
    assert bool((s == -INF).all()) and bool((b == -1).all()) and bool((t == -1).all())


def test_long_masked_stretches_and_rising_rows():
    V = 20000
    logits = torch.full((4, V), -INF, device="cuda")
    logits[0, 100:700] = _logits(1, 600, seed=1)[0]              # a stretch inside one chunk
    logits[1] = torch.arange(V, device="cuda") * 1e-3            # rising: every chunk's best are its last
    logits[2] = -torch.arange(V, device="cuda") * 1e-3
    logits[3, ::3] = 1.5                                         # many equal numbers between masked ones
    _check_selection(logits, torch.tensor([[-1.0, -3.0, -3.5, -2.0]], device="cuda"), 40)
    _check_selection(logits[3:], torch.zeros(1, 1, device="cuda"), 250)
    _check_selection(torch.zeros(8, V, device="cuda"), torch.zeros(1, 8, device="cuda"), 200)    # more equal heads than the list holds


def test_selection_is_repeatable_on_a_stream_of_its_own_and_replayed():
    logits, scores = _logits(24, 30000, seed=8), _scores(3, 8, seed=8)
    want = _select(logits, scores, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _select(logits, scores, 16)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    outs = tuple(torch.empty_like(o) for o in want)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):      # two recordings of the same call, replayed in turn with new inputs
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.beam_select(logits, scores, *outs)
        graphs.append(g)
    for i, g in enumerate(graphs * 2):
        logits.copy_(_logits(24, 30000, seed=20 + i))
        g.replay()
        fresh = _select(logits, scores, 16)
        assert all(torch.equal(a, b) for a, b in zip(outs, fresh))
    _check_selection(logits, scores, 16, outs)


def test_selection_refuses():
    logits, scores = _logits(4, 100), _scores(2, 2)
    with pytest.raises(ops.KernelError, match="257 continuations"):
        _select(logits, scores, 257)
    with pytest.raises(AssertionError):
        _select(logits[:3], scores, 4)
    with pytest.raises(AssertionError):
        _select(logits.double(), scores, 4)
    with pytest.raises(AssertionError):
        _select(logits.t().contiguous().t(), scores, 4)
    with pytest.raises(ops.KernelError, match="CUDA"):
        _select(logits.cpu(), scores, 4)


# ---- copies


def _moves(n, n_sources, n_copies, seed):
    g = torch.Generator().manual_seed(seed)
    at = torch.randperm(n, generator=g).tolist()
    sources, rest = at[:n_sources], at[n_sources:n_sources + n_copies]
    chosen = sources + [sources[i] for i in torch.randint(0, n_sources, (n_copies - n_sources,), generator=g).tolist()]
    order = torch.randperm(n_copies, generator=g).tolist()
    return [(chosen[i], rest[i]) for i in order]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E, P, H, D, n_sources, n_copies", [
    (1, 2, 1, 16, 1, 1), (3, 9, 2, 16, 2, 5), (2, 40, 3, 96, 9, 30), (1, 700, 1, 32, 101, 500), (2, 600, 1, 16, 1, 599), (16, 12, 8, 64, 3, 7),
    (2, 8, 8, 128, 4, 4),
])
def test_page_copies(dtype, E, P, H, D, n_sources, n_copies):
    g = torch.Generator().manual_seed(P + D)
    k = torch.randn(E, P, H, 64, D, generator=g).to(dtype).cuda()
    v = torch.randn(E, P, H, D, 64, generator=g).to(dtype).cuda()
    fills = torch.randint(0, 65, (P,), generator=g).tolist()
    for i, n in enumerate((0, 1, 7, 8, 63, 64)):
        fills[i % P] = n
    moves = [(s, d, fills[s]) for s, d in _moves(P, n_sources, n_copies, D)]
    want_k, want_v = k.clone(), v.clone()
    for s, d, n in moves:
        want_k[:, d, :, :n] = k[:, s, :, :n]
        want_v[:, d, :, :, :n] = v[:, s, :, :, :n]
    ops.copy_pages(k, v, moves)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_page_copies_of_one_entry_and_of_every_other():
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(4, 6, 2, 64, 32, generator=g).cuda(), torch.randn(4, 6, 2, 32, 64, generator=g).cuda()
    want_k, want_v = k.clone(), v.clone()
    ops.copy_pages(k[1], v[1], [(0, 3, 11)])
    want_k[1, 3, :, :11], want_v[1, 3, :, :, :11] = want_k[1, 0, :, :11], want_v[1, 0, :, :, :11]
    ops.copy_pages(k[::2], v[::2], [(5, 1, 64), (5, 2, 64)])
    for d in (1, 2):
        want_k[::2, d], want_v[::2, d] = want_k[::2, 5], want_v[::2, 5]
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    ops.copy_pages(k, v, [])
    assert torch.equal(k, want_k)
    ops.copy_pages(k, v, (m for m in [(5, 4, 64)]))       # any iterable
    want_k[:, 4], want_v[:, 4] = want_k[:, 5], want_v[:, 5]
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


@pytest.mark.parametrize("dtype, shape", [(torch.float32, (149504,)), (torch.float32, (3,)), (torch.float32, (4097,)), (torch.bfloat16, (5, 7)),
                                          (torch.int8, (13,)), (torch.float64, (2, 3)), (torch.int32, (8, 16, 33)), (torch.float32, ())])
def test_state_copies(dtype, shape):
    E, S = 3, 40
    data = (torch.randn(E, S, *shape, generator=torch.Generator().manual_seed(1)) * 50).to(dtype).cuda()
    moves = _moves(S, 9, 25, 4)
    want = data.clone()
    for s, d in moves:
        want[:, d] = data[:, s]
    ops.copy_slots(data, moves)
    assert torch.equal(data, want)
    ops.copy_slots(data[1:2, 3:], [(0, 5)])           # a part of the states, at an address of its own
    want[1, 8] = want[1, 3]
    assert torch.equal(data, want)


def test_copies_refuse():
    k, v = torch.zeros(1, 4, 1, 64, 16, device="cuda"), torch.zeros(1, 4, 1, 16, 64, device="cuda")
    for moves, what in [([(0, 4, 1)], "there are 4"), ([(-1, 2, 1)], "there are 4"), ([(0, 1, 65)], "65. positions"), ([(0, 1, -1)], "-1. positions"),
                        ([(0, 1, 3), (2, 1, 3)], "two moves"), ([(0, 1, 3), (1, 2, 3)], "source and a destination"), ([(2, 2, 3)], "source and a destination"),
                        ([(0, 1, 3), (0, 2, 4)], "two numbers")]:
        with pytest.raises(ops.KernelError, match=what):
            ops.copy_pages(k, v, moves)
    with pytest.raises(AssertionError):
        ops.copy_pages(k, v.transpose(3, 4), [(0, 1, 3)])
    with pytest.raises(AssertionError):
        ops.copy_slots(torch.zeros(1, 1, 8, device="cuda").expand(2, 4, 8), [(0, 1)])
    with pytest.raises(ops.KernelError, match="entries, slots"):
        ops.copy_slots(torch.zeros(4, device="cuda"), [(0, 1)])


# ---- attention


class Groups:
    """Groups of sequences with pages of their own behind shared ones, in shuffled pages; what no position has claimed holds NaN."""

    def __init__(self, shared, kv_lens, H, KVH, D, dtype, seed=0, spread=1.4):
        g = torch.Generator().manual_seed(seed)
        self.G, self.B = len(shared), len(kv_lens) // len(shared)
        self.H, self.KVH, self.D, self.dtype, self.kv_lens = H, KVH, D, dtype, kv_lens
        rows = []
        count = 0
        for i in range(self.G):
            common = list(range(count, count + shared[i]))
            count += shared[i]
            for b in range(self.B):
                n = max(0, -(-kv_lens[i * self.B + b] // 64) - shared[i])
                rows.append(common[:-(-kv_lens[i * self.B + b] // 64)] + list(range(count, count + n)))
                count += n
        order = torch.randperm(max(count, 1), generator=g).tolist()
        self.width = max(1, max(len(r) for r in rows))
        table = torch.zeros(len(rows), self.width, dtype=torch.int32)
        for i, r in enumerate(rows):
            table[i, :len(r)] = torch.tensor([order[p] for p in r], dtype=torch.int32)
        n_pages = max(count, 1)
        k = torch.randn(n_pages, KVH, 64, D, generator=g) * spread
        v = torch.randn(n_pages, KVH, D, 64, generator=g)
        used = torch.zeros(n_pages, dtype=torch.long)
        for r, row in enumerate(rows):
            for i, p in enumerate(row):
                used[order[p]] = max(int(used[order[p]]), min(64, kv_lens[r] - 64 * i))
        for p in range(n_pages):
            k[p, :, used[p]:] = math.nan
            v[p, :, :, used[p]:] = math.nan
        self.q = (torch.randn(len(rows), H * D + 8, generator=g) * spread).to(dtype).cuda()[:, :H * D]    # rows apart
        self.k, self.v = k.to(dtype).cuda(), v.to(dtype).cuda()
        self.table, self.lens = table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda()
        self.shared = torch.tensor(shared, dtype=torch.int32).cuda()

    def run(self, window=0, parts=None, shared=None, scratch=None):
        out = torch.full((self.G * self.B, self.H * self.D), 9.0, dtype=self.dtype, device="cuda")
        if parts is None:
            parts = ops.attention_beams_parts(self.G, self.B, self.H, self.KVH, self.D, self.width * 64, self.dtype, "cuda")
        ops.attention_decode_beams(self.q, self.q.stride(0), out, self.lens, self.table, self.shared if shared is None else shared, self.k, self.v,
                                   self.H, self.KVH, self.D, window, parts, scratch)
        return out

    def check(self, window=0, parts=None, shared=None):
        """Against 64 bits, each element within what roundings can make of it.  A score of D products is off by at most (D + 8) half steps of
        the sum of their sizes, a probability by as much of itself (e), twice over with its maximum's; sums over keys and pages by a half
        step an addition, with at most 64 of a page's in one chain.  bfloat16: probabilities and results are rounded to it, half a step
        2^-8 each; its power of two is off by 2^-22."""
        got = self.run(window, parts, shared).double().cpu()
        assert torch.isfinite(got).all()
        rep, low = self.H // self.KVH, self.dtype == torch.bfloat16
        for r, n in enumerate(self.kv_lens):
            lo = max(0, n - window) if window else 0
            if n == 0:
                assert bool((got[r] == 0).all())
                continue
            pages = self.table[r, :-(-n // 64)].long()
            for h in range(self.KVH):
                heads = slice(h * rep * self.D, (h + 1) * rep * self.D)
                q = self.q[r, heads].double().cpu().view(rep, self.D)
                k = self.k[pages, h].double().cpu().reshape(-1, self.D)[lo:n]
                v = self.v[pages, h].double().cpu().transpose(1, 2).reshape(-1, self.D)[lo:n]
                p = torch.softmax(q @ k.T / math.sqrt(self.D), dim=1)
                want, sizes = p @ v, p @ v.abs()
                e = (self.D + 8) * HALF_STEP * float((q.abs() @ k.abs().T).max()) / math.sqrt(self.D)
                rel = 2 * e + (80 + 2 * len(pages)) * HALF_STEP + (2.0 ** -8 + 2.0 ** -21 if low else 4 * HALF_STEP)
                bound = rel * (sizes + want.abs()) + (2.0 ** -8 if low else HALF_STEP) * want.abs() * (1 + rel) + 1e-30
                err = (got[r, heads].view(rep, self.D) - want).abs()
                assert bool((err <= bound).all()), (r, h, float((err / bound).max()))


SHAPES = [  # shared pages of each group, positions of each sequence, heads, kv heads, head size
    ([0], [1], 1, 1, 32),
    ([0], [1, 1], 4, 2, 64),
    ([1], [65, 64, 100], 8, 2, 64),                                       # one sequence with no key of its own
    ([3, 0], [200, 256, 193, 5, 64, 1], 8, 8, 128),
    ([2], [150] * 4, 16, 1, 64),                                          # 64 rows to a kv head
    ([2, 1], [150, 190, 129, 130, 180, 70, 91, 65, 127, 64], 16, 1, 96),   # 80 rows: two tiles of sequences
    ([5], [330] * 40, 6, 2, 32),                                          # 120 rows
    ([17, 4, 0, 9], [1100] * 3 + [300, 256, 257] + [3, 60, 64] + [580, 640, 600], 12, 4, 64),
    ([40], [2600, 2561], 8, 8, 64),
    ([4, 2], [257, 258, 140, 150], 15, 3, 128),                           # 5 heads to a kv head
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_of_groups_matches_64_bits(case, dtype):
    shared, lens, H, KVH, D = SHAPES[case]
    if len(lens) % len(shared):
        raise ValueError("groups of equal size")
    groups = Groups(shared, lens, H, KVH, D, dtype, seed=case)
    groups.check()
    for parts in (1, 3, 50):
        groups.check(parts=parts)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, 63, 64, 65, 130, 500, 5000])
def test_attention_of_groups_in_a_window(window, dtype):
    groups = Groups([6, 2], [400, 450, 385, 130, 129, 190], 8, 2, 64, dtype, seed=window)
    groups.check(window=window)
    groups.check(window=window, parts=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shared_pages_that_are_none_and_sequences_without_keys(dtype):
    groups = Groups([2], [200, 128, 0], 4, 2, 64, dtype)      # (nothing is shared with a sequence that has no key)
    groups.check()
    groups = Groups([3], [250, 230, 200], 4, 2, 64, dtype)
    for claimed in (-5, 0, 1, 2, 3, 1000):                     # fewer than there are; more than are full for all
        groups.check(shared=torch.tensor([claimed], dtype=torch.int32, device="cuda"))


def test_attention_of_groups_is_the_separate_sequences_attention():
    """Against the kernel that reads each sequence by itself, whose error has the same bound."""
    lens = [700, 690, 650, 645, 100, 101, 102, 103]
    groups = Groups([10, 1], lens, 32, 8, 64, torch.bfloat16, seed=5)
    one = torch.empty(8, 32 * 64, dtype=torch.bfloat16, device="cuda")
    q = groups.q.contiguous()
    ops.attention_decode(q, q.shape[1], one, groups.lens, groups.table, groups.k, groups.v, 32, 8, 64, 0, 4)
    both = (groups.run().float() - one.float()).abs()
    assert float(both.max()) <= 4 * 2.0 ** -8 * float(groups.v[~groups.v.isnan()].abs().max())


def test_large_scores_and_extreme_values():
    groups = Groups([2], [150, 140, 190], 4, 2, 64, torch.bfloat16, seed=2, spread=12.0)     # one key takes nearly all
    groups.check()
    groups.k.zero_()
    groups.v.nan_to_num_(0.0)
    groups.check()                                                                          # all keys alike


def test_offsets_past_32_bits():
    KVH, D, n_pages = 8, 128, 33000                   # 2.16e9 elements a pool
    k, v = (torch.empty(n_pages, KVH, *s, dtype=torch.bfloat16, device="cuda") for s in ((64, D), (D, 64)))
    small = Groups([2], [170, 180], 16, KVH, D, torch.bfloat16, seed=3)
    at = torch.arange(small.k.shape[0], device="cuda") + n_pages - small.k.shape[0]
    k[at], v[at] = small.k, small.v
    want = small.run()
    small.k, small.v, small.table = k, v, (small.table + int(at[0])).to(torch.int32)
    assert torch.equal(small.run(), want)
    ops.copy_pages(k, v, [(n_pages - 1, 0, 50), (n_pages - 2, n_pages - 5000, 64)])
    assert torch.equal(k[0, :, :50].nan_to_num(5.0), k[-1, :, :50].nan_to_num(5.0))
    assert torch.equal(v[n_pages - 5000].nan_to_num(5.0), v[n_pages - 2].nan_to_num(5.0))


def test_attention_of_groups_captured_and_on_two_streams():
    groups = [Groups([7, 3], [500, 460, 450, 200, 210, 230], 8, 2, 64, torch.bfloat16, seed=s) for s in (0, 1)]
    wants = [g.run() for g in groups]
    sides = [torch.cuda.Stream() for _ in groups]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(3):
        for s, g in zip(sides, groups):
            with torch.cuda.stream(s):
                outs.append(g.run())
    torch.cuda.synchronize()
    assert all(torch.equal(o, wants[i % 2]) for i, o in enumerate(outs))
    g = groups[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = g.run()
    # the recording serves other lengths, pages and shares
    g.kv_lens = [470, 449, 448, 199, 192, 201]     # (all within what is written)
    g.lens.copy_(torch.tensor(g.kv_lens, dtype=torch.int32))
    g.shared.copy_(torch.tensor([2, 1], dtype=torch.int32))
    graph.replay()
    assert torch.equal(out, g.run())
    g.check()


def test_attention_of_groups_refuses():
    groups = Groups([1, 1], [70, 71, 72, 73], 4, 2, 64, torch.bfloat16)
    with pytest.raises(ops.KernelError, match="equal groups"):
        groups.run(parts=1, shared=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ops.KernelError, match="equal groups"):
        groups.run(parts=1, shared=torch.zeros(0, dtype=torch.int32, device="cuda"))
    with pytest.raises(AssertionError):
        groups.run(shared=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ops.KernelError, match="bad argument"):
        groups.run(window=-1)
    with pytest.raises(ops.KernelError, match="bad argument"):
        groups.run(parts=0)
    groups.H = 34
    with pytest.raises(ops.KernelError, match="34 heads on 2"):
        groups.run(parts=1)


@pytest.mark.parametrize("pairing", [0, 1])
@pytest.mark.parametrize("write_cache", [True, False])
@pytest.mark.parametrize("shared, lens, H, KVH, D, window", [
    ([0], [1, 1], 4, 2, 64, 0), ([1], [65, 66, 128], 8, 2, 64, 0), ([3, 0], [200, 256, 193, 5, 64, 1], 8, 8, 128, 0), ([5], [330] * 40, 6, 2, 32, 0),
    ([2, 1], [150, 192, 129, 130, 180, 70, 91, 65, 128, 67], 16, 1, 96, 0), ([6, 2], [400, 450, 385, 130, 129, 192], 8, 2, 64, 100),
    ([17, 4], [1100] * 4 + [300, 257, 320, 260], 32, 8, 64, 0),
])
def test_fused_rotation_and_cache_write(shared, lens, H, KVH, D, window, write_cache, pairing):
    """The same bits as rotation and cache write in a kernel of their own and the attention behind it, in the cache too; and the same
    result from a plan made beforehand."""
    B = len(lens)
    parts = ops.attention_beams_parts(len(shared), B // len(shared), H, KVH, D, 64 * 20, torch.bfloat16, "cuda")
    one, two = (Groups(shared, lens, H, KVH, D, torch.bfloat16, seed=len(lens)) for _ in range(2))
    qkv = (torch.randn(B, (H + 2 * KVH) * D, generator=torch.Generator().manual_seed(3)) * 1.4).to(torch.bfloat16).cuda()
    inv_freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
    rotated = qkv.clone()
    ops.rope_cache_write(rotated, one.lens - 1, torch.arange(B, dtype=torch.int32, device="cuda"), one.table, inv_freq, one.k, one.v, H, KVH, D, D,
                         pairing, write_cache=write_cache)
    want, got, again = (torch.empty(B, H * D, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    # (shared pages that reach the new position are refused to be shared by the fused form alone: compared on what is left)
    fewer = torch.tensor([min(s, min(lens[i * (B // len(shared)):(i + 1) * (B // len(shared))]) - 1 >> 6) for i, s in enumerate(shared)],
                         dtype=torch.int32, device="cuda")
    ops.attention_decode_beams(rotated, rotated.shape[1], want, one.lens, one.table, fewer, one.k, one.v, H, KVH, D, window, parts)
    raw = qkv.clone()
    call = lambda out, plan: ops.attention_decode_beams_rope(raw, out, two.lens, two.table, two.shared if write_cache else fewer, two.k, two.v, inv_freq, H,
                                                             KVH, D, pairing, window, parts, write_cache, plan=plan)
    call(got, None)
    assert torch.equal(raw, qkv) and torch.isfinite(want).all()
    assert torch.equal(one.k.view(torch.int16), two.k.view(torch.int16)) and torch.equal(one.v.view(torch.int16), two.v.view(torch.int16))
    assert torch.equal(got, want)
    plan = ops.attention_beams_plan(two.lens, two.shared if write_cache else fewer, two.width, H, KVH, window, writes_cache=write_cache)
    call(again, plan)
    assert torch.equal(again, want)
    plain_plan = ops.attention_beams_plan(one.lens, fewer, one.width, H, KVH, window)
    again.zero_()
    ops.attention_decode_beams(rotated, rotated.shape[1], again, one.lens, one.table, fewer, one.k, one.v, H, KVH, D, window, parts, plan=plain_plan)
    assert torch.equal(again, want)


@pytest.mark.parametrize("case", [4, 5, 6, 7, 9])
@pytest.mark.parametrize("window", [0, 130])
def test_float32_attention_takes_any_plan_of_its_groups(case, window):
    """A plan shares the work out for one type; a call of the other takes it all the same: sums are cut elsewhere, nothing is left out."""
    shared, lens, H, KVH, D = SHAPES[case]
    groups = Groups(shared, lens, H, KVH, D, torch.float32, seed=case)
    out = torch.empty(len(lens), H * D, device="cuda")
    for parts in (2, 7, 30):
        direct = groups.run(window, parts)
        for dtype in (torch.float32, torch.bfloat16):
            plan = ops.attention_beams_plan(groups.lens, groups.shared, groups.width, H, KVH, window, dtype=dtype)
            ops.attention_decode_beams(groups.q, groups.q.stride(0), out, groups.lens, groups.table, groups.shared, groups.k, groups.v, H, KVH, D,
                                       window, parts, plan=plan)
            if dtype == torch.float32:
                assert torch.equal(out, direct)
            else:       # the same products in another order of sums: each within the bound of `check`, so within twice that of each other
                assert float((out - direct).norm() / direct.norm()) <= 2 * (80 + 2 * groups.width) * HALF_STEP
        groups.check(window, parts)


@pytest.mark.parametrize("power", [-60, -20, 40, 100])
def test_float32_attention_of_scaled_numbers_keeps_its_bits(power):
    """Powers of two go through every part and product unchanged: keys by 2^power and queries by 2^-power, and values by 2^power."""
    groups = Groups([3, 2], [250, 230, 200, 192, 140, 170], 8, 2, 64, torch.float32)
    want = groups.run()
    groups.k *= 2.0 ** power
    groups.q = groups.q * 2.0 ** -power
    assert torch.equal(groups.run(), want)
    groups.v *= 2.0 ** (power - 10)
    assert torch.equal(groups.run(), want * 2.0 ** (power - 10))
