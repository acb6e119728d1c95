"""Paged serving on the HIP kernels: batches of sequences whose cached keys and
values lie in pages of one pool, several new positions per sequence and step.

The reference serves one growing cache per batch and one token per step
(src/qwen_int4/generation.py:10-115, src/qwen_int4/model.py:61-122).  A
speculative step over pages is three calls in its place:

    rotated = paged_append_hip(q, k, v, k_pages, v_pages, page_table, cu_rows, lengths, inv_freq)
    attended = paged_attention_hip(rotated, k_pages, v_pages, page_table, cu_rows, lengths, shared_pages=n)
    tokens, accepted = verify_drafts_hip(target_probs, draft_tokens, uniforms, draft_probs=draft_probs)

Common arguments.  Rows (tokens) are packed: sequence ``b``'s new positions are
rows ``cu_rows[b]`` up to ``cu_rows[b + 1]`` (int32 [B + 1], not falling, from 0),
and they are the last ones of its ``lengths[b]`` (int32 [B]) cached positions, so
that row i of n sits at position ``lengths[b] - n + i``.  ``k_pages`` and
``v_pages`` are [pages, kv_heads, page_size, head_dim], bf16 or fp16, with a page
size that is a power of two from 16; any strides (a [pages, page_size, kv_heads,
head_dim] pool is passed as its ``transpose(1, 2)``) whose last is 1 and whose
others are multiples of 8.  ``page_table`` (int32 [B, W]) names the pages of each
sequence in order.

``cu_rows``, ``lengths`` and ``page_table`` stay on the GPU: nothing is read back,
every call can be captured into a HIP graph, and what they hold can change
between replays.  The kernels bound every index they take from them; a row that
leads outside its table or the pool is not written (``paged_append_hip``) or
gives NaN (``paged_attention_hip``).

Every function launches on torch's current stream of its tensors' device and
raises before any of its kernels is launched (what is not laid out as they read it may
have been copied by then): TypeError for a dtype, ValueError for shapes,
strides, devices and memory that overlaps, RuntimeError where a gradient would be
due (they have none), under a dispatch mode, trace or function transform, and
without the built library.
"""

from __future__ import annotations

import torch

from . import _lib

_host = None


def _calls():
    global _host
    if _host is None:
        _host = _lib.host_module()
    return _host


def paged_append_hip(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     page_table: torch.Tensor, cu_rows: torch.Tensor, lengths: torch.Tensor,
                     inv_freq: torch.Tensor | None, *, interleaved: bool = False, rotary_scale: float = 1.0,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate the new rows' queries and keys by their positions and write keys
    and values into their pages; returns the rotated queries.

    ``q`` [rows, heads, head_dim], ``k``, ``v`` [rows, kv_heads, head_dim] (views
    of a fused projection are read in place).  ``inv_freq`` (fp32 [R / 2]) turns
    the first R dimensions (R a multiple of 16; None: none) in pairs (i, i + R / 2),
    or (2 i, 2 i + 1) with ``interleaved``, by ``position * inv_freq[i]``, formed in
    64 bits; ``rotary_scale`` multiplies what is turned.  Contexts stretched past
    the trained length are a matter of these two.  Results are rounded once.

    ``out`` may be ``q`` itself (whose rows then lie apart from k's and v's, as in a
    fused projection).  head_dim is a multiple of 16 up to 256.  Rows behind the last sequence are left as they
    are in ``out``, and zeros in a new tensor.  Two rows of one call must not
    share a place in the cache."""
    return _calls().paged_append(q, k, v, k_pages, v_pages, page_table, cu_rows, lengths, inv_freq, interleaved,
                                 rotary_scale, out)


def paged_attention_hip(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                        cu_rows: torch.Tensor, lengths: torch.Tensor, *, shared_pages: int = 0,
                        scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the new rows over their sequences' pages:
    ``softmax_t(scale * q . k_t) v_t`` over t up to the row's own position, query
    head h reading key/value head ``h // (heads // kv_heads)``; head_dim 64 or 128,
    ``scale`` head_dim ** -0.5 unless given.

    ``shared_pages``: the first so many entries of every row of ``page_table`` name
    the same pages (a prompt common to the batch).  They are taken from the first
    row and read once for all sequences; the result is the same.

    The call is cut into workgroups by the width of ``page_table``, for the lengths are
    on the GPU: columns behind the longest sequence change no result, but a table much
    wider than the sequences leaves too few workgroups to a shared prefix (32 rows over
    4096 common positions, 12 and 2 heads of 128: 18.7 us with a table of their
    length, 25.9 with one of 32768 positions, 68.1 with one of 131072).

    Keys and values that a row does not see take no part, whatever they hold; an
    infinity or NaN that it sees reaches it, however small the key's weight.  A row
    without a position gives zeros.  Rows behind the last sequence are left as they
    are in ``out``, and zeros in a new tensor.  Scores, softmax and sums are fp32, in a
    fixed order: the same inputs give the same bits.  Probabilities enter the value
    products as two terms of the tensors' type (16 bits or more of them), and values
    are summed before the sum is divided: the keys' number times the values'
    size has to stay in fp32.  The result is rounded once."""
    return _calls().paged_attention(q, k_pages, v_pages, page_table, cu_rows, lengths, shared_pages, scale, out)


def verify_drafts_hip(target_probs: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor, *,
                      draft_probs: torch.Tensor | None = None,
                      draft_lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens stand, from given random numbers, and the token after
    them; what is returned is distributed as the target's own tokens.

    ``target_probs`` [B, K + 1, V] (fp32, bf16 or fp16), ``draft_tokens`` int64
    [B, K], ``uniforms`` fp32 [B, K + 1] in [0, 1), ``draft_probs`` [B, K, V] of the
    target's dtype, or None for tokens that no model drew (probability 1 each),
    ``draft_lengths`` int32 [B] where a sequence has fewer than K drafts.

    Draft i stands if those before it do and ``uniforms[:, i] * q(x) < p(x)``.  The
    token after the n that stand is drawn with ``uniforms[:, K]`` from
    ``max(p - q, 0)`` at row n (from p, if all stand): the least entry at which the
    running sum passes the uniform's share of the total, all in 64 bits.  Returns
    (tokens int64 [B, K + 1]: the n, the new one, then -1; accepted int32 [B]: n).
    The new token is -1 where the weights' sum is zero, infinite or NaN or the uniform is
    NaN, and an entry of weight otherwise."""
    return _calls().verify_drafts(target_probs, draft_tokens, uniforms, draft_probs, draft_lengths)
