"""What a server does with the paged caches of ``ops.reshape_and_cache`` and ``ops.paged_attention`` besides decoding:
attention of many new tokens per sequence, and the pages themselves, shared, given out, taken back, copied and packed
on the device.

The pool's state is ``ref_counts``, int32 ``[num_blocks]``: how many sequences hold each page; a page is free where that is
not positive.  ``block_tables`` int32 ``[sequences, max_pages]`` and ``context_lens`` int32 ``[sequences]`` are those of
``ops.paged_attention``; a sequence holds the first ``ceil(context_len / block_size)`` entries of its row.  Every operator
returns new tables and counts and leaves its arguments alone; only the caches are written in place.  Pages are given out
lowest first in the order of the requests, so a host that keeps a copy of the state can follow without asking.
``key_caches``/``value_caches`` are lists with the caches of all layers (256 at most together), each
``[num_blocks, kv_heads*D/16, block_size, 16]``."""
from __future__ import annotations

from typing import Optional, Sequence

import torch

import ascend910a_extras.ascend910a_extras_C as _C

Tensor = torch.Tensor


def paged_attention_chunk(
    q: Tensor,
    key_cache: Tensor,
    value_cache: Tensor,
    block_tables: Tensor,
    context_lens: Tensor,
    query_starts: Tensor,
    scale: Optional[float] = None,
    window: int = 0,
    return_lse: bool = False,
    out: Optional[Tensor] = None,
):
    """Attention of any number of new tokens per sequence over the paged caches, which hold their K and V already
    (``ops.reshape_and_cache``): prompts, chunks of prompts, drafted tokens and single tokens in one batch.

    ``q [tokens, heads, D]`` holds the new tokens of all sequences one after the other; sequence ``b`` has the rows
    ``query_starts[b]:query_starts[b+1]`` (int32 ``[sequences + 1]``), which are the last tokens of its ``context_lens[b]``.  A
    row sees the keys up to its own position, only the last ``window`` of them where ``window > 0``; kv head and page of a key
    as in ``ops.paged_attention``, ``scale`` (positive, at most 2^56) 1/sqrt(D) if not given.  A row that sees nothing (a
    context shorter than the new tokens) is 0.  Lengths and tables are read on the device only.

    Returns ``o`` like ``q``, with ``return_lse`` also the natural log-sum-exp of the scaled scores, fp32 ``[tokens, heads]``
    (-inf where nothing is seen), by which results over parts of a context can be joined.  Rows of no sequence (a batch padded
    behind ``query_starts[-1]``) are not written: they keep what ``out`` held, if that is given, and are undefined if not."""
    return _C.paged_attention_chunk(q, key_cache, value_cache, block_tables, context_lens, query_starts, scale, window,
                                    return_lse, out)


def copy_pages(key_caches: Sequence[Tensor], value_caches: Sequence[Tensor], src_pages: Tensor, dst_pages: Tensor) -> None:
    """Copies page ``src_pages[i]`` to page ``dst_pages[i]`` (int32 ``[pairs]``) in every cache, in place.  Pairs that name
    a page outside the caches are skipped; a page that two pairs write, or that one pair reads and another writes, ends up
    with unspecified contents."""
    _C.copy_pages(list(key_caches), list(value_caches), src_pages, dst_pages)


def fork_sequences(block_tables: Tensor, context_lens: Tensor, parents: Tensor, ref_counts: Tensor,
                   key_caches: Sequence[Tensor], value_caches: Sequence[Tensor]) -> tuple[Tensor, Tensor, Tensor]:
    """Sequences that begin as copies of ``parents`` (int32 ``[children]``, rows of ``block_tables``): the parent's full pages
    are shared, the tokens behind them are copied, in every cache, into a page of the child's own (the rest of which is
    left as it was).  Returns ``(child_tables [children, max_pages], child_lens [children], new_ref_counts)``; entries behind a
    child's pages are -1.  A child for which there is no free page, or whose parent is no row of the table, gets length 0 and
    no pages."""
    return _C.fork_sequences(block_tables, context_lens, parents, ref_counts, list(key_caches), list(value_caches))


def extend_sequences(block_tables: Tensor, context_lens: Tensor, wanted_lens: Tensor, ref_counts: Tensor,
                     block_size: int) -> tuple[Tensor, Tensor, Tensor]:
    """Pages for ``wanted_lens`` (int32 ``[sequences]``) tokens.  Returns ``(new_tables, granted_lens, new_ref_counts)``: where a
    row of the table is too short, or the free pages do not suffice for a sequence and all those in front of it, its
    row and length stay as they are, and likewise where the length wanted is not greater than the present one.  A present length
    that its row cannot hold counts, and comes back, as what the row holds, a negative one as 0."""
    return _C.extend_sequences(block_tables, context_lens, wanted_lens, ref_counts, block_size)


def free_sequences(block_tables: Tensor, context_lens: Tensor, rows: Tensor, ref_counts: Tensor, block_size: int) -> Tensor:
    """Takes back the pages of the sequences ``rows`` (int32, rows of ``block_tables``; others are skipped): returns new counts,
    lower by one for every time a page is named, and never below 0."""
    return _C.free_sequences(block_tables, context_lens, rows, ref_counts, block_size)


def compact_pages(block_tables: Tensor, context_lens: Tensor, ref_counts: Tensor, key_caches: Sequence[Tensor],
                  value_caches: Sequence[Tensor]) -> tuple[Tensor, Tensor, Tensor]:
    """Packs the used pages into the lowest page numbers, moving as few as possible: the used pages from number ``used`` on go, in
    ascending order, to the free pages below.  ``block_tables`` has to hold every sequence of the pool.  Returns
    ``(new_tables, new_ref_counts, used)``, ``used`` int32 ``[1]``."""
    return _C.compact_pages(block_tables, context_lens, ref_counts, list(key_caches), list(value_caches))
