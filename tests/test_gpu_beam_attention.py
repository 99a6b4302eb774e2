"""Attention of groups where numbers are not finite, hidden by a window or of the largest and smallest sizes, against 64 bits."""
import math

import pytest
import torch

from gpullama3.java_b200.kernels import ops
from test_gpu_beam_kernels import HALF_STEP, SHAPES, Groups

pytestmark = pytest.mark.gpu
INF = math.inf
DTYPES = [torch.bfloat16, torch.float32]


def _definition(g: Groups, window=0, absolute=0.0):
    """Results in 64 bits from what each sequence sees alone, and how far a kernel may be from them where they are finite.

    A score of D products is off by (D + 8) half steps of the sum of their sizes, a probability by as much of itself, twice over with its maximum's;
    sums over n keys by n half steps, those over blocks of 32 and pieces by 4 each.  bfloat16: a probability is two numbers of 8 bits, so half a step
    of 2^-9 of what is left after as much, twice with the sum's, its power of two 2^-21; a result half a step, 2^-8.  ``absolute``: of the
    numbers that went in."""
    rep, low = g.H // g.KVH, g.dtype == torch.bfloat16
    want, bound = torch.zeros(len(g.kv_lens), g.H * g.D, dtype=torch.float64), torch.zeros(len(g.kv_lens), g.H * g.D, dtype=torch.float64)
    for r, n in enumerate(g.kv_lens):
        lo = max(0, n - window) if window else 0
        pages = g.table[r, :-(-n // 64)].long()
        for h in range(g.KVH):
            heads = slice(h * rep * g.D, (h + 1) * rep * g.D)
            q = g.q[r, heads].double().cpu().view(rep, g.D)
            k = g.k[pages, h].double().cpu().reshape(-1, g.D)[lo:n]
            v = g.v[pages, h].double().cpu().transpose(1, 2).reshape(-1, g.D)[lo:n]
            s = q @ k.T / math.sqrt(g.D)
            p = torch.softmax(s, dim=1)
            w = (p.unsqueeze(2) * v).sum(1)          # (elementwise: what is not finite stays in its own column)
            sizes = (p.unsqueeze(2) * v.abs()).sum(1)
            seen = q.abs() @ k.abs().T
            seen = seen[torch.isfinite(seen)]
            e = (g.D + 8) * HALF_STEP * float(seen.max() if seen.numel() else 0.0) / math.sqrt(g.D)
            rel = 2 * e + (n - lo + n / 8 + 80) * HALF_STEP + (2.0 ** -17 + 2.0 ** -21 if low else 4 * HALF_STEP)
            want[r, heads] = w.reshape(-1)
            bound[r, heads] = (rel * (sizes + w.abs()) + (2.0 ** -8 if low else HALF_STEP) * w.abs() * (1 + rel) + absolute + 1e-30).reshape(-1)
    return want, bound


def _check(g: Groups, window=0, parts=None, absolute=0.0):
    got = g.run(window, parts).double().cpu()
    want, bound = _definition(g, window, absolute)
    finite = torch.isfinite(want)
    assert torch.equal(got[~finite].nan_to_num(7.0, 8.0, 9.0), want[~finite].nan_to_num(7.0, 8.0, 9.0))
    err = (got[finite] - want[finite]).abs()
    assert bool((err <= bound[finite]).all()), float((err / bound[finite]).nan_to_num(INF).max())
    return finite


@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_probabilities_of_bfloat16_attention_are_not_rounded_to_it(case):
    shared, lens, H, KVH, D = SHAPES[case]
    g = Groups(shared, lens, H, KVH, D, torch.bfloat16, seed=case + 50, spread=0.5)
    assert bool(_check(g).all()) and bool(_check(g, window=100).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", [math.nan, INF, -INF])
@pytest.mark.parametrize("window", [1, 40, 64, 100, 150])
def test_what_a_window_hides_counts_for_nothing(window, what, dtype):
    """Positions in front of every sequence's window, in the pages that it begins in, shared and own."""
    g = Groups([3, 3, 0], [330, 330, 330, 250, 250, 250, 90, 90, 90], 8, 2, 64, dtype, seed=window)
    for r, n in enumerate(g.kv_lens):
        for at in range(max(0, n - window)):
            page = int(g.table[r, at // 64])
            g.k[page, :, at % 64] = what
            g.v[page, :, :, at % 64] = what
    for parts in (None, 1, 5):
        assert bool(_check(g, window, parts).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_one_sequence_sees_and_another_does_not(dtype):
    """Sequences of unequal lengths in one group: a window hides a shared page's NaN from the longer ones only."""
    g = Groups([3], [200, 240, 300], 8, 2, 64, dtype, seed=1)
    page = int(g.table[0, 1])
    g.v[page, 1, 5, 30] = math.nan                   # position 94
    g.v[page, 0, 9, 60] = -INF                       # position 124
    finite = _check(g, 150)                          # from 50, 90 and 150 on
    assert not finite[0].all() and not finite[1].all() and finite[2].all()
    finite = _check(g, 110)                          # from 90, 130 and 190 on
    assert not finite[0].all() and finite[1:].all()


@pytest.mark.parametrize("D, H, KVH", [(64, 8, 2), (128, 4, 4), (32, 16, 1), (96, 6, 2)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_that_are_seen(dtype, D, H, KVH):
    g = Groups([2, 1], [190, 150, 170, 100, 64, 130], H, KVH, D, dtype, seed=D, spread=0.7)
    g.q.abs_()
    g.v[int(g.table[0, 1]), 0, 3, 17] = INF          # a value: this dimension of all heads that see it
    g.v[int(g.table[1, 2]), KVH - 1, 4, 5] = -INF    # of one sequence alone
    g.k[int(g.table[4, 0]), 0, 20] = -INF            # a key of score -inf: its weight is 0
    g.k[int(g.table[5, 2]), KVH - 1, 1, 7] = INF     # a key of score inf: no distribution
    g.k[int(g.table[3, 1]), KVH - 1, 2, 7] = math.nan
    finite = _check(g)
    assert not finite.all() and finite[4].all()
    g.k[int(g.table[4, 0])] = -INF                   # all keys of a sequence
    assert not _check(g)[4].any()


def test_hidden_numbers_of_the_fused_form():
    """Rotation and cache write in the same kernel: the same bits as by themselves, where rows are computed once more too."""
    dtype, H, KVH, D, lens, window = torch.bfloat16, 8, 2, 64, [330, 330, 250, 250], 70
    one, two = (Groups([4, 2], lens, H, KVH, D, dtype, seed=2) for _ in range(2))
    for g in (one, two):
        for r, n in enumerate(lens):
            for at in range(n - window - 12):
                g.v[int(g.table[r, at // 64]), :, :, at % 64] = math.nan
    for pairing in (0, 1):
        qkv = torch.randn(4, (H + 2 * KVH) * D, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
        inv_freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
        rotated = qkv.clone()
        ops.rope_cache_write(rotated, one.lens - 1, torch.arange(4, dtype=torch.int32, device="cuda"), one.table, inv_freq, one.k, one.v, H, KVH, D, D, pairing)
        want, got = (torch.empty(4, H * D, dtype=dtype, device="cuda") for _ in range(2))
        ops.attention_decode_beams(rotated, rotated.shape[1], want, one.lens, one.table, one.shared, one.k, one.v, H, KVH, D, window, 9)
        ops.attention_decode_beams_rope(qkv, got, two.lens, two.table, two.shared, two.k, two.v, inv_freq, H, KVH, D, pairing, window, 9)
        assert torch.isfinite(want).all() and torch.equal(got, want)


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_float32_attention_of_the_largest_numbers(sign):
    """Numbers that round to infinity in bfloat16, of which its parts are made: as queries, keys and values, where results are finite."""
    g = Groups([3, 2], [250, 230, 200, 192, 140, 170], 8, 2, 64, torch.float32, seed=4)
    big = sign * torch.finfo(torch.float32).max
    g.v[int(g.table[0, 1]), 0, 3, 17] = big
    g.v[int(g.table[4, 2]), 1, 60, 5] = big
    assert bool(_check(g).all())
    g.q[:, 7::64] = 2.0 ** -126                      # dimension 7 of every head
    g.k[int(g.table[1, 0]), :, 9, 7] = big
    g.k[int(g.table[5, 2]), 1, 30, 7] = big
    assert bool(_check(g).all())
    g.q[2, 11] = big                                 # a query of one head against keys of 2^-126
    g.k[:, 0, :, 11] = 2.0 ** -126
    assert bool(_check(g).all())


@pytest.mark.parametrize("power", [-110, -118, -125, -132])
def test_float32_attention_of_the_smallest_values(power):
    """Below 2^-109 the parts hold a number to half of bfloat16's last place there, 2^-134."""
    g = Groups([3, 2], [250, 230, 200, 192, 140, 170], 8, 2, 64, torch.float32, seed=5)
    g.v *= 2.0 ** power
    assert bool(_check(g, absolute=2.0 ** -133).all())
    assert float(g.run().abs().max()) > 0


@pytest.mark.parametrize("power", [-110, -114, -118])
def test_float32_attention_of_the_smallest_queries(power):
    """The same of queries, against keys as large: a score is off by D products of up to 2^-134 times a key."""
    g = Groups([3, 2], [250, 230, 200, 192, 140, 170], 8, 2, 64, torch.float32, seed=6)
    want = g.run()
    keys, values = (float(x[~x.isnan()].abs().max()) for x in (g.k, g.v))
    g.q, g.k = g.q * 2.0 ** power, g.k * 2.0 ** -power
    off = 64 * 2.0 ** (-134 - power) * keys / 8
    assert float((g.run() - want).abs().max()) <= (2 * math.expm1(2 * off) + 1e-5) * values


@pytest.mark.parametrize("G, B", [(1024, 1), (512, 3), (31, 64)])
def test_plans_of_the_most_groups_that_a_call_takes(G, B):
    """2,048 segments of pages or nearly: as many groups of one sequence, of three, of 64."""
    lens = [65 + (37 * i) % 90 for i in range(G * B)]
    g = Groups([1] * G, lens, 1, 1, 32, torch.bfloat16, seed=G)
    assert ops.attention_beams_takes(G, B, 1, 1) and not ops.attention_beams_takes(G + 1, B, 1, 1)
    direct, out = g.run(parts=300), torch.empty(G * B, 32, dtype=torch.bfloat16, device="cuda")
    plan = ops.attention_beams_plan(g.lens, g.shared, g.width, 1, 1, 0)
    ops.attention_decode_beams(g.q, g.q.stride(0), out, g.lens, g.table, g.shared, g.k, g.v, 1, 1, 32, 0, 300, plan=plan)
    assert torch.equal(out, direct)
    g.check(parts=300)
