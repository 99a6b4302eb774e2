"""Which attention a step of a beam search takes, at the sizes where both were measured (ms a step: of groups, of separate sequences)."""
import types

import pytest
import torch

from gpullama3.java_b200.kernels import fast

LLAMA_1B, LLAMA_3B, LLAMA_8B = (32, 8, 64), (24, 8, 128), (32, 8, 128)


def _shares(heads, groups, beams, positions, dtype=torch.bfloat16, window=None, recorded=True):
    n_heads, n_kv_heads, head_dim = heads
    capacity = 256 if recorded else positions + 1       # (a step launched by itself need be right for its own lengths alone)
    while capacity < positions + 1:
        capacity *= 2
    ctx = types.SimpleNamespace(beams=beams, all_decode=True, n_seqs=groups * beams)
    mixer = types.SimpleNamespace(n_heads=n_heads, n_kv_heads=n_kv_heads, head_dim=head_dim, window=window, keep_first=0, has_terms=False)
    return fast.beams_share_attention(ctx, mixer, dtype, capacity)


@pytest.mark.parametrize("heads, groups, beams, positions, shared, separate", [
    (LLAMA_1B, 1, 4, 1000, 0.995, 0.741), (LLAMA_1B, 5, 4, 600, 1.015, 0.970), (LLAMA_1B, 5, 4, 900, 1.025, 0.997), (LLAMA_1B, 5, 4, 1500, 1.058, 1.069),
    (LLAMA_1B, 5, 4, 1900, 1.076, 1.118), (LLAMA_1B, 8, 8, 450, 1.241, 1.156), (LLAMA_1B, 8, 8, 600, 1.264, 1.182), (LLAMA_1B, 8, 8, 1100, 1.298, 1.315),
    (LLAMA_1B, 8, 8, 1900, 1.347, 1.511), (LLAMA_1B, 8, 8, 4000, 1.466, 1.975), (LLAMA_1B, 32, 2, 900, 1.383, 1.304), (LLAMA_1B, 32, 2, 1100, 1.428, 1.353),
    (LLAMA_1B, 32, 2, 3500, 1.788, 1.968), (LLAMA_1B, 4, 8, 1100, 1.095, 1.156), (LLAMA_1B, 2, 16, 1100, 1.102, 1.156), (LLAMA_8B, 8, 8, 220, 4.601, 4.414),
    (LLAMA_8B, 8, 8, 600, 4.691, 4.735), (LLAMA_8B, 8, 8, 900, 4.759, 5.207), (LLAMA_8B, 8, 8, 3000, 5.160, 7.921), (LLAMA_8B, 5, 4, 900, 3.772, 4.073),
    (LLAMA_8B, 32, 2, 1500, 5.354, 6.336), (LLAMA_3B, 8, 8, 600, 2.814, 2.980), (LLAMA_3B, 5, 4, 900, 2.216, 2.434),
    (LLAMA_1B, 1, 4, 16000, 1.240, 0.965), (LLAMA_1B, 1, 4, 60000, 1.462, 1.624), (LLAMA_1B, 1, 8, 16000, 1.336, 1.217), (LLAMA_1B, 2, 8, 4000, 1.559, 1.369),
    (LLAMA_1B, 2, 8, 9000, 1.665, 1.669), (LLAMA_1B, 2, 8, 16000, 1.741, 2.033), (LLAMA_1B, 4, 4, 4000, 1.567, 1.386), (LLAMA_1B, 4, 4, 16000, 1.878, 2.074),
    (LLAMA_1B, 3, 4, 16000, 1.735, 1.970), (LLAMA_1B, 1, 12, 9000, 1.408, 1.582), (LLAMA_1B, 1, 16, 9000, 1.480, 1.652), (LLAMA_1B, 8, 2, 9000, 1.886, 1.735),
    (LLAMA_8B, 2, 8, 4000, 7.424, 6.023), (LLAMA_8B, 2, 8, 16000, 8.108, 9.618), (LLAMA_8B, 4, 4, 4000, 7.566, 6.057), (LLAMA_8B, 4, 4, 16000, 8.579, 9.770),
    (LLAMA_8B, 3, 4, 9000, 7.433, 7.604), (LLAMA_8B, 1, 16, 9000, 5.569, 7.542), (LLAMA_8B, 1, 8, 16000, 6.585, 5.878),
])
def test_the_faster_one_is_taken(heads, groups, beams, positions, shared, separate):
    assert _shares(heads, groups, beams, positions) == (shared < separate)


def test_a_window_counts_as_what_is_seen():
    assert _shares(LLAMA_1B, 8, 8, 4000, window=4096) and not _shares(LLAMA_1B, 8, 8, 4000, window=1000)
    assert _shares(LLAMA_8B, 8, 8, 4000, window=1024) and not _shares(LLAMA_8B, 8, 8, 4000, window=500)
    assert _shares(LLAMA_1B, 8, 8, 2000, torch.float32, window=256) and not _shares(LLAMA_1B, 8, 8, 2000, torch.float32, window=255)


@pytest.mark.parametrize("heads, groups, beams, last", [(LLAMA_1B, 8, 8, 1023), (LLAMA_1B, 5, 4, 1023), (LLAMA_1B, 32, 2, 2047), (LLAMA_8B, 8, 8, 511), (LLAMA_8B, 32, 2, 1023),
                                                        (LLAMA_1B, 4, 4, 8191), (LLAMA_8B, 1, 9, 8191), (LLAMA_1B, 1, 8, 32767)])
def test_recorded_and_launched_steps_change_over_at_the_same_length(heads, groups, beams, last):
    for recorded in (True, False):
        assert not _shares(heads, groups, beams, last, recorded=recorded) and _shares(heads, groups, beams, last + 1, recorded=recorded)
