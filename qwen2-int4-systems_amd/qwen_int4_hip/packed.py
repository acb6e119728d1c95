"""Attention over whole prompts of different lengths on the HIP kernels.

The reference's ``QwenAttention.forward`` takes prompts padded to one length
(src/qwen_int4/model.py:61-122); here their rows are packed, as the paged operators'
are (``paged.py``), and a prompt's own attention reads the projections where they
stand, not the cache's pages:

    # qkv [rows, H + 2 G, head_dim]: the keys' heads go along with the queries', so that they come back rotated
    rotated = paged_append_hip(qkv[:, :H + G], qkv[:, H:H + G], qkv[:, H + G:], k_pages, v_pages, page_table, cu_rows,
                               lengths, inv_freq)
    attended = packed_attention_hip(rotated[:, :H], rotated[:, H:], qkv[:, H + G:], cu_rows)

A prompt that continues a cached one is ``paged_attention_hip``'s.
"""

from __future__ import annotations

import torch

from . import paged


def packed_attention_hip(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_rows: torch.Tensor, *,
                         scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompts: row r of a sequence attends its rows up to
    r, ``softmax_t(scale * q_r . k_t) v_t``, query head h reading key/value head
    ``h // (heads // kv_heads)``.

    ``q`` [rows, heads, head_dim], ``k``, ``v`` [rows, kv_heads, head_dim], bf16 or fp16,
    head_dim 64 or 128: views of a fused projection are read in place.  Sequence b is
    rows ``cu_rows[b]`` up to ``cu_rows[b + 1]`` (int32 [B + 1], not falling, from 0; on
    the GPU, bounded in the kernel, free to change between a graph's replays).
    ``scale`` is head_dim ** -0.5 unless given.

    Keys and values that a row does not see take no part, whatever they hold; an
    infinity or NaN that it sees reaches it, however small the key's weight (a call full
    of such rows takes three to seventeen times as long: 23 us instead of 6.5 for 37
    tokens, 400 instead of 42 for eight prompts of 1000).  Rows of no sequence (behind
    the last one, or before ``cu_rows[0]``) are left as they are in ``out``, and zeros in
    a new tensor.  Scores, softmax and sums are fp32, in a fixed order: the same inputs
    give the same bits.  A probability is rounded once to the tensors' type before it
    meets its value, and the sum that divides is the rounded ones'; values are summed
    before the division: the keys' number times the values' size has to stay in fp32.
    The result is rounded once.

    Launches on torch's current stream of the tensors' device; raises before anything is
    launched: TypeError for a dtype, ValueError for shapes, strides, devices and memory
    that overlaps, RuntimeError where a gradient would be due (it has none), under a
    dispatch mode, trace or function transform, and without the built library."""
    return paged._calls().packed_attention(q, k, v, cu_rows, scale, out)
