"""The pages of a paged cache on the HIP kernels: handing them out, forking
sequences, compacting the pool.

The reference keeps one growing cache per batch (src/qwen_int4/generation.py:10-115)
and has no pages.  Here a step's lengths are on the GPU (``verify_drafts_hip`` decides
there how many tokens stand), so the pages are dealt out there too:

    table, users, missing = paged_resize_hip(table, lengths + drafts, users, page_size=16, cached=lengths)
    table, lengths, users, missing = paged_fork_hip(k_pages, v_pages, table, lengths, users, parents)
    table, users, moved_to = paged_compact_hip(k_pages, v_pages, table, users)

``page_table`` (int32 [B, W]) names the pages of each sequence in order, -1 where
there is none (any number outside the pool counts as that).  ``page_users`` (int32
[pages]) counts what names a page: entries of tables, and whatever else keeps it (add
one for a prefix that stays cached without a sequence).  A page is free where it is 0:
a pool starts with zeros, a table with -1.  Several tables can share a pool through
one ``page_users``.

``k_pages`` and ``v_pages`` are the pools that the other paged operators take,
[pages, kv_heads, page_size, head_dim], or those of all layers whose pages one table
names, [layers, pages, kv_heads, page_size, head_dim], in any strides whose last is 1
and whose others are multiples of 8; bf16 or fp16, a page size that is a power of two
from 16.

Index tensors are returned new and the arguments stay as they are, so a step that has
to be given up leaves its state whole; keys and values are copied in place, to pages
that were free.  Pages given up in a call are free from the next one on.  Nothing is
read back: every call can be captured into a HIP graph (copy the answers to where the
graph reads them).  What the indices hold is bounded in the kernels.  Whole numbers
alone decide, in a fixed order: the same state gives the same answer.

Every function launches on torch's current stream of its tensors' device and raises
before anything is launched: TypeError for a dtype, ValueError for shapes, strides,
devices and pools that share memory, RuntimeError under a dispatch mode, trace or
function transform, where a gradient would be due, and without the built library.
Limits: 2^24 pages, 2^20 rows, 2^31 - 1 table entries.
"""

from __future__ import annotations

import torch

from . import paged


def paged_resize_hip(page_table: torch.Tensor, lengths: torch.Tensor, page_users: torch.Tensor, *,
                     page_size: int, cached: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Give every sequence the pages that its length needs, and take the others.

    Row b's first ``ceil(lengths[b] / page_size)`` entries keep the pages that they
    name, or get the lowest free ones, row after row; the rest become -1 and their
    pages are given up.  A length of 0 (or below) frees a sequence; a length ahead of
    the cached positions reserves pages.

    Returns (table, page_users, missing): ``missing`` (int32 [B]) counts the pages that
    a row still lacks because the pool (then the last columns of the last rows go
    without) or its table's width was too small; ``paged_append_hip`` does not write
    there, ``paged_attention_hip`` gives NaN.

    ``cached`` (int32 [B]): how many positions of each row hold keys and values already.
    A page that such a position should lie in and that the table does not name is lost (a
    resize or a fork found none free): a page given there now would hold what another
    sequence left in it.  With ``cached`` it is not given; the row goes on missing it, and
    giving NaN, at every call until its length is set below it (0 frees the row) or it is
    filled anew and ``cached`` says so.  Without ``cached`` every missing page is given,
    which is right only where none of a row's positions at such pages counts as cached: a
    row that an earlier ``missing`` names is then to be freed, or that step redone from the state
    before it.

    A sequence that is cut back into a page which something else names must be passed
    through ``paged_fork_hip`` (with itself as its parent) before it is written again."""
    return paged._calls().paged_resize(page_table, lengths, page_users, page_size, cached)


def paged_fork_hip(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                   page_users: torch.Tensor, parents: torch.Tensor,
                   ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The next batch, made of copies of this one's sequences: samples of one prompt,
    beams, another order.  Row i is sequence ``parents[i]`` (int32 [C]), or empty where
    that is outside [0, B).

    Rows share full pages.  Of a last page that is not full, the sequence's first row
    keeps the page itself if nothing else names it; every other row gets the lowest free
    page, row after row, and a copy of the filled positions (all layers).  So every row
    can be written at its next position.  Sequences without a row give up their pages,
    and all give up the pages behind their length.

    Returns (table [C, W], lengths [C], page_users, missing [C]): ``missing`` is 1 where
    a copy found no free page (its entry is -1).  Such a row keeps its length without the
    positions of its last page: free it, redo the fork from the state before it, or give the
    next ``paged_resize_hip`` these lengths as ``cached``, which then goes on calling it missing."""
    return paged._calls().paged_fork(k_pages, v_pages, page_table, lengths, page_users, parents)


def paged_compact_hip(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                      page_users: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the n pages in use to the pool's first n places (all layers), so that the
    rest can be given back: those that lie behind, the lowest first, go to the free
    ones before, the lowest first.

    Returns (table, page_users, moved_to): ``moved_to`` (int32 [pages]) says where each
    page lies now, -1 for a free one, for whatever names pages besides this table.  Pages
    behind the first n keep what they held."""
    return paged._calls().paged_compact(k_pages, v_pages, page_table, page_users)
