"""A beam search's selection where its threads go on at different times: the same call gives the same bits however often it is made; and how
far a sum of log probabilities may be off."""
import math

import pytest
import torch

from gpullama3.java_b200.kernels import ops
from test_gpu_beam_kernels import HALF_STEP, _check_selection, _logits, _reference, _scores, _select

pytestmark = pytest.mark.gpu


def _repeated(logits, scores, n, times):
    """The selection, and how many of ``times`` more calls (recorded, one after the other) differ from it in any bit."""
    G = scores.shape[0]
    outs = lambda: (torch.empty(G, n, device="cuda"), *(torch.empty(G, n, dtype=torch.int32, device="cuda") for _ in range(2)))
    first, other = outs(), outs()
    ops.beam_select(logits, scores, *first)
    words = lambda o: torch.stack([o[0].view(torch.int32), o[1], o[2]])
    want, differing = words(first), torch.zeros((), dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.beam_select(logits, scores, *other)
        differing += (words(other) != want).any()
    for _ in range(times):
        graph.replay()
    return first, int(differing)


def _rising(rows, V, seed):
    """Rows that rise with some noise: the candidates of every tile pass those before it, so a list grows over its limit again and again."""
    return _logits(rows, V, seed=seed, spread=0.5) + torch.arange(V, device="cuda") * (40.0 / V)


@pytest.mark.parametrize("make", [_logits, _rising])
@pytest.mark.parametrize("G, B, V, n", [(8, 32, 128256, 64), (8, 8, 128256, 64), (4, 60, 50257, 200), (2, 150, 90001, 3)])
def test_rows_of_many_tiles_give_the_same_bits_each_time(G, B, V, n, make):
    """Each CTA goes through a row in several tiles and cuts its list of candidates down between them, or not."""
    logits, scores = make(G * B, V, seed=V), _scores(G, B, seed=V)
    first, differing = _repeated(logits, scores, n, 10000 if V * G * B > 8e6 else 2000)
    assert differing == 0
    _check_selection(logits, scores, n, first)


@pytest.mark.parametrize("G, B, V, n", [(8, 8, 4000, 16), (40, 4, 1000, 8), (3, 100, 2000, 30), (2, 500, 300, 50), (1, 4, 128256, 8), (8, 16, 128256, 33)])
@pytest.mark.parametrize("low", [0.5, 8.0, 120.0])
def test_merges_of_totals_of_all_sizes_give_the_same_bits_each_time(G, B, V, n, low):
    """Totals from -0.5 down to far below: the search over their bits skips what lies above the largest, so bits are counted in any order of
    odd and even; all candidates in registers, and in lists that are looked through."""
    logits = _logits(G * B, V, seed=n, spread=3.0)
    scores = -low * torch.rand(G, B, generator=torch.Generator().manual_seed(n)).cuda()
    for shift in (0.0, 0.3, 1.7):
        first, differing = _repeated(logits, scores - shift, n, 1000)
        assert differing == 0
        _check_selection(logits, scores - shift, n, first)


def test_beams_of_very_unequal_scores_give_the_same_bits_each_time():
    """The margin of the merge's rough totals follows the largest of the beams' scores, which all warps put together."""
    logits = _logits(6 * 16, 3000, seed=2)
    scores = _scores(6, 16, seed=2)
    scores[:, 11] = -3.0e4                     # one warp's alone
    scores[3:, 0] = -1.0e7
    first, differing = _repeated(logits, scores, 24, 5000)
    assert differing == 0
    _check_selection(logits, scores, 24, first)


@pytest.mark.parametrize("background", [0.0, 1.0, 4.0])
@pytest.mark.parametrize("above", [0.0, 15.9])
def test_log_probabilities_never_rise_and_are_off_by_a_bounded_amount(above, background):
    """Rows of one peak behind the first tile of a chunk, ``above`` and more above everything before it.

    A row's log sum is off by at most 2.3 (1 + log V) + 12 half steps, absolutely.  Relative to its reference, at most 1 below and never above the
    row's largest logit rounded up, a logit is -t with t at most 1 + the distance d to the largest, so its exponential is off by t half steps each
    from the difference, from the product with log2 e and 0.22 from that number's own rounding, by 4 from the power of two, by 8 from the additions in 32
    bits.  Weighed by the probabilities p, sum p d = entropy - log sum e^-d is at most log V.  The stored score is rounded once."""
    B, V = 64, 70001
    logits = _logits(B, V, seed=int(above), spread=background)
    at = 4096 + 131 * torch.arange(B, device="cuda")              # (second and third tiles)
    rows = torch.arange(B, device="cuda")
    logits[rows, at] = logits[:, :4096].amax(dim=1) + above + torch.linspace(0, 25 - above, B, device="cuda")
    bound = (2.3 * (1 + math.log(V)) + 12) * HALF_STEP
    for scores in (torch.zeros(1, B, device="cuda"), _scores(1, B, seed=1)):
        total, _ = _reference(logits, scores, 1)
        s, b, t = (o.cpu()[0] for o in _select(logits, scores, 2 * B))
        assert bool((s <= scores.cpu()[0][b.long()]).all())
        exact = total[0][b.long(), t.long()]
        assert bool(((s.double() - exact).abs() <= bound + HALF_STEP * exact.abs()).all())
        assert len(set(zip(b.tolist(), t.tolist()))) == 2 * B
        # with a beam to itself
        s, b, t = (o.cpu()[0] for o in _select(logits[7:8], scores[:, 7:8], 3))
        assert float(s[0]) <= float(scores[0, 7]) and (above == 0.0 or int(t[0]) == int(at[7]))


def test_tokens_whose_probability_is_one_are_ordered_by_beam_whatever_zeros_sign():
    logits = torch.full((4, 9000), -200.0, device="cuda")
    logits[:, 5000] = torch.tensor([0.0, -0.0, 30.0, -7.0], device="cuda")
    s, b, t = _select(logits, torch.tensor([[-0.0, 0.0, -0.0, 0.0]], device="cuda"), 4)
    assert s.tolist() == [[0.0] * 4] and b.tolist() == [[0, 1, 2, 3]] and t.tolist() == [[5000] * 4]
