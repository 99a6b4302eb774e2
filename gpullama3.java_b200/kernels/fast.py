"""Choice of the tensor-core kernels of the bfloat16 run.

``try_gemm`` and ``try_attention`` run the specialised sm_100a kernel that fits the operands and
return True, or return False when no specialised kernel takes these storage types or sizes (the
caller then runs the plain kernel, which takes every size).  The true 32-bit run never comes
here with anything but float32 operands and therefore always takes the kernels of ``ops`` that keep 32 bits."""
from __future__ import annotations

import torch

from . import ops


def try_gemm(a: torch.Tensor, w: torch.Tensor, c: torch.Tensor, epilogue: int, gate_args=(0.0, 0.0), bias=None,
             silu_columns: int = 0) -> bool:
    if a.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        return False
    M = a.shape[0]
    if M <= 16:
        return ops.gemm_decode(a, w, c, epilogue, gate_args, bias, silu_columns)
    if bias is not None or silu_columns:
        # (the few-token tensor-core kernel has neither: what it adds to the residual stream gets the bias behind it)
        if bias is not None and M <= 128 and epilogue == ops.EPILOGUE_RESIDUAL_ADD and c.is_contiguous() and ops.gemm_skinny(a, w, c, epilogue):
            ops.add_row(c, bias)
            return True
        if M <= 64 and ops.gemm_decode(a, w, c, epilogue, gate_args, bias, silu_columns):
            return True
        return ops.gemm_tcgen05(a, w, c, epilogue, gate_args=gate_args, bias=bias, silu_columns=silu_columns)
    # (the few-token tensor-core kernel has the gated epilogue with SiLU only; the other activations' sizes go to the other two)
    if M <= 128 and epilogue in (ops.EPILOGUE_STORE, ops.EPILOGUE_RESIDUAL_ADD, ops.EPILOGUE_GATED_SILU) and ops.gemm_skinny(a, w, c, epilogue):
        return True
    if M <= 64 and ops.gemm_decode(a, w, c, epilogue, gate_args):
        return True
    return ops.gemm_tcgen05(a, w, c, epilogue, gate_args=gate_args)


def try_projection_with_rope(x: torch.Tensor, w: torch.Tensor, qkv: torch.Tensor, ctx, page_table, cache, mixer,
                             writes_cache: bool) -> bool:
    """A prompt pass's query/key/value projection with rotation and cache write in the product's epilogue, where the
    sizes allow (whole heads of 64 or 128 in 256-column tiles, a position encoding that offers its angles per pass)."""
    pos = mixer.position
    if (ctx.all_decode or x.dtype != torch.bfloat16 or pos.rotary_dim != mixer.head_dim or mixer.head_dim not in (64, 128)
            or not hasattr(pos, "angles")):
        return False
    few = 16 < x.shape[0] <= 128 and ops.gemm_skinny_k_spans(x.shape[0], w.shape[0], x.shape[1], x.device) > 1
    whole_k = ops.gemm_tcgen05_k_spans(x.shape[0], w.shape[0], x.shape[1]) == 1
    if not few and not whole_k:
        return False
    operands = (x, w, qkv, ctx.positions, ctx.seq_ids, page_table, pos.angles(ctx), cache.k if writes_cache else None,
                cache.v if writes_cache else None, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim, pos.pairing, writes_cache)
    return (few and ops.gemm_skinny_qkv_rope(*operands)) or (whole_k and ops.gemm_tcgen05_qkv_rope(*operands))


def try_decode_attention_with_rope(qkv, out, ctx, page_table, cache, mixer, writes_cache: bool) -> bool:
    """A decode step's rotation, cache write and attention in one kernel, where the sizes allow."""
    pos = mixer.position
    if not (ctx.all_decode and ops.attention_decode_rope_supported(qkv.dtype, mixer.n_heads, mixer.n_kv_heads,
                                                                   mixer.head_dim, pos.rotary_dim, pos.pairing)):
        return False
    if beams_share_attention(ctx, mixer, qkv.dtype, _capacity(ctx, cache)):
        shared, parts, plan = _beam_launch(ctx, page_table, cache, mixer, qkv.dtype, bool(writes_cache))
        ops.attention_decode_beams_rope(qkv, out, ctx.kv_lens, page_table, shared, cache.k, cache.v, pos.inverse_frequencies(qkv.device),
                                        mixer.n_heads, mixer.n_kv_heads, mixer.head_dim, pos.pairing, mixer.window or 0, parts,
                                        write_cache=writes_cache, plan=plan)
        return True
    splits, early = mixer.plan_decode(ctx, cache)
    ops.attention_decode_rope(qkv, out, ctx.kv_lens, page_table, cache.k, cache.v, pos.inverse_frequencies(qkv.device),
                              mixer.n_heads, mixer.n_kv_heads, mixer.head_dim, pos.pairing, mixer.window or 0, splits,
                              write_cache=writes_cache, early_start=early)
    return True


def beams_share_attention(ctx, mixer, dtype, capacity: int) -> bool:
    """Whether a decode step's attention reads the pages that a group's sequences share once for all of them: a beam search's step of a
    mixer whose mask is causality and at most a window, where that is faster.  ``capacity``: the longest sequence the step must be right for.

    bfloat16: up to 16 sequences the products of a step stream through L1, and the attention of groups, which keeps its pages in shared memory,
    makes every SM change its split twice a layer, which pays where positions are many; beyond that the separate sequences' kernel is faster while they are short, for their pages
    are in L2 for all but the first of a group, and the shorter the wider the heads.  A step in ms, of groups / of separate sequences: 1B shape (heads
    of 64) 1 x 4 at 1,000 positions 1.00 / 0.74, at 16,000 1.24 / 0.97, at 60,000 1.46 / 1.62; 1 x 8 at 16,000 1.34 / 1.22, at 30,000 1.44 / 1.60; 4 x 4 at
    4,000 1.57 / 1.39, at 9,000 1.70 / 1.69, at 16,000 1.88 / 2.07; 2 x 8 at 4,000 1.56 / 1.37, at 9,000 1.67 / 1.67, at 16,000 1.74 / 2.03; 3 x 4 at 16,000
    1.74 / 1.97; 1 x 16 at 4,000 1.37 / 1.36, at 9,000 1.48 / 1.65; 8 x 2 at 9,000 1.89 / 1.74, at 16,000 2.16 / 2.17; 5 x 4 at 600 1.02 / 0.97, at 1,100 1.03 / 1.02, at 1,500 1.06 / 1.07, at 1,900 1.07 / 1.12; 4 x 8 at
    600 1.06 / 1.10; 8 x 8 at 600 1.26 / 1.18, at 900 1.27 / 1.27, at 1,100 1.30 / 1.32, at 1,900 1.35 / 1.51, at 4,000 1.47 / 1.98; 32 x 2 at 1,100 1.43 /
    1.35, at 1,900 1.55 / 1.57, at 3,500 1.79 / 1.97; 8B shape (of 128) 1 x 8 at 16,000 6.59 / 5.88; 4 x 4 at
    9,000 8.07 / 7.65, at 16,000 8.58 / 9.77; 2 x 8 at 16,000 8.11 / 9.62; 1 x 16 at 9,000 5.57 / 7.54; 8 x 8 at 220 4.60 / 4.41, at 600 4.69 / 4.74, at 900 4.76 / 5.21, at 3,000 5.16 /
    7.92; 5 x 4 at 600 3.81 / 3.82, at 900 3.77 / 4.07; 32 x 2 at 900 5.03 / 5.36, at 1,500 5.35 / 6.34.  So heads of 64
    change over at 1,025 positions (2 beams 2,049), heads of 128 at 513 (2 beams 1,025), 9 to 16 sequences at 8,193, fewer at 32,769: powers of two, as a
    recorded step's capacity is one.

    float32: faster as soon as there is enough to read, whatever the number of sequences.  1B shape: 1 x 4 at 900 1.51 / 1.45; 1 x 8 at 1,900 1.99 /
    2.06; 4 x 4 at 450 2.66 / 2.57, at 900 2.69 / 2.73, at 3,900 2.87 / 3.92; 8 x 4 at 200 2.72 / 2.71, at 450 2.78 / 2.84; 8 x 8 at 200
    2.98 / 2.99, at 1,900 3.38 / 5.08, at 3,900 3.73 / 7.44."""
    beams = getattr(ctx, "beams", 1)
    if beams == 1 or not ctx.all_decode or mixer.keep_first or getattr(mixer, "has_terms", False) or getattr(mixer, "chunk", None):
        return False
    seen = min(capacity, mixer.window or capacity)
    if dtype == torch.float32:
        enough = ctx.n_seqs * seen >= 16384
    else:
        if ctx.n_seqs > 16:
            enough = seen * mixer.head_dim > 1024 * 64 and beams * capacity * mixer.head_dim > 4096 * 64
        else:
            enough = beams > 2 and seen > (8192 if ctx.n_seqs > 8 else 32768)
    return (enough and ops.attention_beams_supported(dtype, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim)
            and ops.attention_beams_takes(ctx.n_seqs // beams, beams, mixer.n_heads, mixer.n_kv_heads))


def _capacity(ctx, cache) -> int:
    return ctx.capacity(cache.group) if getattr(ctx, "beams", 1) > 1 else 0


def _beam_launch(ctx, page_table, cache, mixer, dtype, writes_cache: bool):
    """What a call of the attention of groups needs beside its operands: the shared pages, how many CTAs, and the plan, which is made
    once for all layers of a kind."""
    shared = ctx.shared_pages[cache.group]
    parts = ops.attention_beams_parts(ctx.n_seqs // ctx.beams, ctx.beams, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim,
                                      ctx.capacity(cache.group), dtype, page_table.device)
    key = ("beam attention", cache.group, mixer.n_heads, mixer.n_kv_heads, mixer.window, writes_cache)
    plan = ctx.extras.get(key)
    if plan is None:
        plan = ctx.extras[key] = ops.attention_beams_plan(ctx.kv_lens, shared, page_table.shape[1], mixer.n_heads, mixer.n_kv_heads,
                                                          mixer.window or 0, writes_cache=writes_cache, dtype=dtype)
    return shared, parts, plan


def try_beam_attention(qkv, out, ctx, page_table, cache, mixer, gate=None) -> bool:
    if gate is not None or not beams_share_attention(ctx, mixer, qkv.dtype, _capacity(ctx, cache)) or qkv.shape[1] % 8 or qkv.data_ptr() & 15:
        return False
    shared, parts, plan = _beam_launch(ctx, page_table, cache, mixer, qkv.dtype, False)
    ops.attention_decode_beams(qkv, qkv.shape[1], out, ctx.kv_lens, page_table, shared, cache.k, cache.v, mixer.n_heads,
                               mixer.n_kv_heads, mixer.head_dim, mixer.window or 0, parts, plan=plan)
    return True


def try_attention(qkv, out, ctx, page_table, cache, mixer, gate=None) -> bool:
    if getattr(mixer, "has_terms", False):
        # kept first positions, runs of positions, distance penalty, sink, output gate, soft cap: the span kernel for decode steps,
        # for prompts the tcgen05 kernel without kept positions and penalty (heads of 64 and 128), else the flash kernel
        chunk = getattr(mixer, "chunk", None) or 0
        terms = dict(keep_first=mixer.keep_first, chunk=chunk, slopes=mixer.slopes, sinks=mixer.sinks, gate=gate,
                     softcap=getattr(mixer, "softcap", None) or 0.0)
        if qkv.dtype != torch.bfloat16 or mixer.head_dim not in (32, 64, 96, 128):
            return False
        if ctx.all_decode and ops.attention_decode_supported(qkv.dtype, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim):
            splits, early = mixer.plan_decode(ctx, cache)
            ops.attention_decode(qkv, qkv.shape[1], out, ctx.kv_lens, page_table, cache.k, cache.v, mixer.n_heads,
                                 mixer.n_kv_heads, mixer.head_dim, mixer.window or 0, splits, early_start=early, **terms)
            return True
        if qkv.shape[1] % 8 or (qkv.data_ptr() & 15):
            return False
        if not mixer.keep_first and mixer.slopes is None and ops.attention_prefill_tc(
                qkv, qkv.shape[1], out, ctx.cu_seqlens, ctx.kv_lens, page_table, cache.k, cache.v, ctx.n_seqs, ctx.max_q_len,
                mixer.n_heads, mixer.n_kv_heads, mixer.head_dim, mixer.window or 0, chunk=chunk, sinks=mixer.sinks, gate=gate,
                softcap=terms["softcap"], work_counters=getattr(cache, "work_counters", None)):
            return True
        ops.attention_prefill(qkv, qkv.shape[1], out, ctx.cu_seqlens, ctx.kv_lens, page_table, cache.k, cache.v,
                              ctx.n_seqs, ctx.max_q_len, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim,
                              mixer.window or 0, **terms)
        return True
    if ctx.all_decode and ops.attention_decode_supported(qkv.dtype, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim):
        splits, early = mixer.plan_decode(ctx, cache)
        ops.attention_decode(qkv, qkv.shape[1], out, ctx.kv_lens, page_table, cache.k, cache.v, mixer.n_heads,
                             mixer.n_kv_heads, mixer.head_dim, mixer.window or 0, splits, early_start=early)
        return True
    if qkv.dtype == torch.bfloat16 and ops.attention_prefill_tc(
            qkv, qkv.shape[1], out, ctx.cu_seqlens, ctx.kv_lens, page_table, cache.k, cache.v, ctx.n_seqs,
            ctx.max_q_len, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim, mixer.window or 0,
            work_counters=getattr(cache, "work_counters", None)):
        return True
    if qkv.dtype == torch.bfloat16 and mixer.head_dim in (32, 64, 96, 128):
        ops.attention_prefill(qkv, qkv.shape[1], out, ctx.cu_seqlens, ctx.kv_lens, page_table, cache.k, cache.v,
                              ctx.n_seqs, ctx.max_q_len, mixer.n_heads, mixer.n_kv_heads, mixer.head_dim,
                              mixer.window or 0)
        return True
    return False
