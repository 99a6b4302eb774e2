"""Calls of the attention of groups whose queries are not what the call says: refused before anything is launched."""
import pytest
import torch

from gpullama3.java_b200.kernels import ops


def _operands(n=4, H=4, KVH=2, D=64):
    i32 = dict(dtype=torch.int32)
    return dict(out=torch.zeros(n, H * D), kv_lens=torch.full((n,), 70, **i32), page_table=torch.zeros(n, 2, **i32), shared_pages=torch.zeros(2, **i32),
                k_pool=torch.zeros(2, KVH, 64, D), v_pool=torch.zeros(2, KVH, D, 64), n_heads=H, n_kv_heads=KVH, head_dim=D, window=0, n_parts=1)


@pytest.mark.parametrize("q, stride", [
    (torch.zeros(4, 256), 320),                   # steps past the last row
    (torch.zeros(4, 320)[:, :256], 256),          # rows are further apart
    (torch.zeros(4, 192), 192),                   # too few columns
    (torch.zeros(3, 256), 256),                   # too few rows
    (torch.zeros(256, 4).t(), 4),                 # columns apart
    (torch.zeros(4, 1, 256), 256),
])
def test_rows_of_queries_that_are_not_where_the_call_says(monkeypatch, q, stride):
    def launched(name):
        raise RuntimeError(f"{name} was called")

    monkeypatch.setattr(ops, "_here", lambda *tensors: None)      # (the checks of CUDA tensors aside, on a machine without any)
    monkeypatch.setattr(ops, "_beams_numbers", lambda *numbers: (1 << 20, 64))
    monkeypatch.setattr(ops, "_fn", launched)
    with pytest.raises(AssertionError):
        ops.attention_decode_beams(q, stride, **_operands())
    with pytest.raises(RuntimeError, match="attention_beams was called"):
        ops.attention_decode_beams(torch.zeros(4, 320)[:, :256], 320, **_operands())
