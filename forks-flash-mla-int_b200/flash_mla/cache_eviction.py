"""Eviction of rows from the paged bf16 cache of dense MLA decode, by the attention they got.

A cached latent row that hardly any query looks at can go when the pool is full.  Three calls, each one kernel (the
weights of a window two), none of which synchronises:

``mla_cache_row_weights``   adds up, for every cached row, the attention weight that the queries of a
                            ``flash_mla_with_kvcache`` call gave it, from the log-sum-exp that call returned;
``mla_select_cache_rows``   names the rows of each sequence that stay: its last ones and the heaviest of the others;
``mla_compact_cache``       moves those rows to the front of the sequence's pages (or to other pages).

The heads share one latent row, so a row's weight is the sum over all of them.  Rows keep the rotary position they
were written with.  After the move the sequence has ``kept`` rows; its remaining pages are free.  A program that evicts
again and again keeps two tensors of sums, each as wide as the table's rows, and lets the selection write one from the
other, so that the rows appended later have their place in it:

    mla_cache_row_weights(q, k_cache, block_table, cache_seqlens, lse, causal=True, weights=sums)      # every step
    rows, kept, other = mla_select_cache_rows(sums, cache_seqlens, budget, recent, kept_weights=other)
    mla_compact_cache(k_cache, block_table, rows, kept)
    cache_seqlens, sums, other = kept, other, sums

No counterpart in the reference.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._loader import load_torch_extension

load_torch_extension()

# The ops check their arguments themselves, in C++; the checks here are made when an op has refused, to say what is wrong
# with a ValueError.  A small call is bound by the host, and checking twice would cost it several microseconds.
_new_weights = torch.ops.flash_mla.mla_cache_row_weights.default
_add_weights = torch.ops.flash_mla.add_mla_cache_row_weights.default
_select = torch.ops.flash_mla.mla_select_cache_rows.default
_select_into = torch.ops.flash_mla.mla_select_cache_rows_into.default
_compact = torch.ops.flash_mla.mla_compact_cache.default


def _check_table(name: str, table: torch.Tensor, batch: int) -> None:
    if table.dim() != 2 or table.shape[0] != batch or table.dtype != torch.int32:
        raise ValueError(f"expected {name} int32 [{batch}, pages], got {table.dtype} {tuple(table.shape)}")


def _check_lens(name: str, lens: torch.Tensor, batch: int) -> None:
    if lens.dim() != 1 or lens.shape[0] != batch or lens.dtype != torch.int32:
        raise ValueError(f"expected {name} int32 [{batch}], got {lens.dtype} {tuple(lens.shape)}")


def _check_cache(k_cache: torch.Tensor) -> None:
    if k_cache.dim() != 4 or k_cache.shape[2] != 1 or k_cache.dtype != torch.bfloat16:
        raise ValueError("expected k_cache bfloat16 [num_blocks, page_block_size, 1, head_dim], got "
                         f"{k_cache.dtype} {tuple(k_cache.shape)}")


def mla_cache_row_weights(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor, cache_seqlens: torch.Tensor,
                          softmax_lse: torch.Tensor, softmax_scale: Optional[float] = None, causal: bool = False,
                          weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention weight of each cached row, summed over heads and query positions: fp32 (batch_size, rows) with

        w[b, r] = sum over positions i and heads h that see row r of exp(scale * q[b, i, h] . K[b, r] - lse[b, h, i]).

    Arguments:
        q, k_cache, block_table, cache_seqlens, softmax_scale, causal: those of the ``flash_mla_with_kvcache`` call;
            q (batch_size, seq_len_q, num_heads_q, 576 or 512) bfloat16, the last ``seq_len_q`` positions of
            each sequence (a window of a prompt counts as such a call); page sizes that are multiples of 8.
        softmax_lse: (batch_size, num_heads_q, seq_len_q) float32 as that call returned it.  A query whose entry is
            -inf saw no row and adds nothing.
        weights: float32 (batch_size, rows) with contiguous rows to add to, in place; the entries behind a
            sequence's length stay as they are, and rows past the tensor's width are left out (a selection from it
            would not see them either).  None: a new tensor with one column per row that ``block_table`` can name, 0
            behind each length.

    Returns ``weights``.  The sums are formed in a fixed order: the same call gives the same bits.  They are fp32; the tensor
    cores cut the sums of a score off toward zero, which with more than 32 (position, head) pairs leaves a row that all queries
    look at lighter by up to 4e-6 of its weight, in proportion more for scores beyond 7."""
    try:
        scale = q.shape[-1] ** (-0.5) if softmax_scale is None else float(softmax_scale)
        if weights is None:
            return _new_weights(q, k_cache, block_table, cache_seqlens, softmax_lse, scale, causal)
        _add_weights(q, k_cache, block_table, cache_seqlens, softmax_lse, scale, causal, weights)
        return weights
    except (RuntimeError, NotImplementedError, IndexError, ZeroDivisionError):
        _check_weights_call(q, k_cache, block_table, cache_seqlens, softmax_lse, weights)
        raise


def _check_weights_call(q, k_cache, block_table, cache_seqlens, softmax_lse, weights) -> None:
    if q.dim() != 4 or q.shape[-1] not in (576, 512) or q.dtype != torch.bfloat16:
        raise ValueError(f"expected q bfloat16 [batch, seq_len_q, heads, 576 or 512], got {q.dtype} {tuple(q.shape)}")
    batch = q.shape[0]
    _check_cache(k_cache)
    if k_cache.shape[3] != q.shape[3]:
        raise ValueError(f"q has head_dim {q.shape[3]}, k_cache {k_cache.shape[3]}")
    if k_cache.shape[1] % 8 != 0:
        raise ValueError(f"expected a page_block_size that is a multiple of 8, got {k_cache.shape[1]}")
    _check_table("block_table", block_table, batch)
    _check_lens("cache_seqlens", cache_seqlens, batch)
    if tuple(softmax_lse.shape) != (batch, q.shape[2], q.shape[1]) or softmax_lse.dtype != torch.float32:
        raise ValueError(f"expected softmax_lse float32 {(batch, q.shape[2], q.shape[1])}, got {softmax_lse.dtype} "
                         f"{tuple(softmax_lse.shape)}")
    if weights is not None and (weights.dim() != 2 or weights.shape[0] != batch or weights.dtype != torch.float32):
        raise ValueError(f"expected weights float32 [{batch}, rows], got {weights.dtype} {tuple(weights.shape)}")


def mla_select_cache_rows(weights: torch.Tensor, cache_seqlens: torch.Tensor, budget: int, recent: int = 0,
                          kept_weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The rows of each sequence that stay when at most ``budget`` of them may.

    A sequence of at most ``budget`` rows (its length counts up to the width of ``weights``) keeps them all.  A
    longer one keeps its last ``recent`` rows and, of those in front of them, the ``budget - recent`` with the
    largest weights; the lower row goes first where weights are equal, and a NaN counts as less than every number.

    Rows past the width of ``weights`` are not seen, and they would be the newest: it has to be as wide as the longest
    sequence, in a second eviction too.

    Arguments: weights float32 (batch_size, rows); cache_seqlens int32 (batch_size,); 0 <= recent <= budget;
        kept_weights: float32 (batch_size, columns) with contiguous rows to write the weights of the rows that stay to, 0
            behind them: sums to go on adding to, as wide as the table's rows so that rows appended later have their
            place.  At least min(budget, rows) columns; it must not overlap ``weights``.  None: a new tensor with budget columns.

    Returns rows int32 (batch_size, budget), ascending, -1 behind the last; kept int32 (batch_size,), how many;
    kept_weights, their weights, 0 behind."""
    try:
        if kept_weights is None:
            return _select(weights, cache_seqlens, budget, recent)
        rows, kept = _select_into(weights, cache_seqlens, budget, recent, kept_weights)
        return rows, kept, kept_weights
    except (RuntimeError, NotImplementedError):
        if weights.dim() != 2 or weights.dtype != torch.float32:
            raise ValueError(f"expected weights float32 [batch, rows], got {weights.dtype} {tuple(weights.shape)}")
        _check_lens("cache_seqlens", cache_seqlens, weights.shape[0])
        if budget < 1 or not 0 <= recent <= budget:
            raise ValueError(f"expected 0 <= recent <= budget and budget >= 1, got budget {budget}, recent {recent}")
        if kept_weights is not None:
            batch, columns = weights.shape[0], min(budget, weights.shape[1])
            if kept_weights.dim() != 2 or kept_weights.shape[0] != batch or kept_weights.dtype != torch.float32 or kept_weights.shape[1] < columns:
                raise ValueError(f"expected kept_weights float32 [{batch}, at least {columns}], got {kept_weights.dtype} {tuple(kept_weights.shape)}")
            if kept_weights.untyped_storage().data_ptr() == weights.untyped_storage().data_ptr():
                raise ValueError("kept_weights must not overlap weights")
        raise


def mla_compact_cache(k_cache: torch.Tensor, block_table: torch.Tensor, rows: torch.Tensor, kept: torch.Tensor,
                      out_block_table: Optional[torch.Tensor] = None) -> None:
    """Move row ``rows[b, j]`` of sequence b to its row j, for j < kept[b], inside ``k_cache``.

    ``block_table`` names the pages that the rows are in, ``out_block_table`` the pages that they go to.  None moves
    them to the front of their own pages, and so does a table that names a sequence's pages in the columns in which
    ``block_table`` has them (``block_table`` itself, its first columns, a copy); this needs ascending ``rows`` (as
    ``mla_select_cache_rows`` returns them).  All other target pages must not be among those read.  No page may be
    written for two sequences: a page that sequences share (a common prefix) has to be left to the others by moving to new pages.
    Rows of the cache that are not written keep their contents.

    Arguments: k_cache bfloat16 (num_blocks, page_block_size, 1, head_dim), head_dim a multiple of 8; tables int32
    (batch_size, pages); rows int32 (batch_size, budget); kept int32 (batch_size,)."""
    try:
        _compact(k_cache, block_table, rows, kept, out_block_table)
    except (RuntimeError, NotImplementedError):
        _check_cache(k_cache)
        if rows.dim() != 2 or rows.dtype != torch.int32:
            raise ValueError(f"expected rows int32 [batch, budget], got {rows.dtype} {tuple(rows.shape)}")
        if k_cache.shape[3] % 8 != 0:
            raise ValueError(f"expected a head_dim that is a multiple of 8, got {k_cache.shape[3]}")
        batch = rows.shape[0]
        _check_table("block_table", block_table, batch)
        _check_lens("kept", kept, batch)
        if out_block_table is not None:
            _check_table("out_block_table", out_block_table, batch)
        raise
