"""float64 / integer CPU oracles of cache-row eviction (test infrastructure, not product).  Written from the
definitions; the reference has no such operators."""
from __future__ import annotations

import math

import torch


def sequence_slots(block_table_row, page, n):
    """Slot of each of the first n rows of a sequence."""
    r = torch.arange(n)
    return block_table_row.cpu().long()[r // page] * page + r % page


def cache_row_weights(q, k_cache, block_table, cache_seqlens, lse, scale=None, causal=False, weights=None, width=None):
    """-> (w [b, width] float64, bound): ``bound`` is sum_terms term * (scale sum |q k| + |lse| + |s|), what the
    rounding of scores and exponents is relative to.  Pages outside the cache are rows of zeros."""
    q = q.detach().cpu().double()
    nb, page, _, d = k_cache.shape
    rows = torch.cat([k_cache.detach().cpu().reshape(nb * page, d).double(), torch.zeros(1, d).double()])
    b, sq, h, _ = q.shape
    scale = d ** -0.5 if scale is None else scale
    cap = block_table.shape[1] * page
    width = cap if width is None else width
    w = torch.zeros(b, width, dtype=torch.float64) if weights is None else weights.detach().cpu().double().clone()
    bound = torch.zeros_like(w)
    lse = lse.detach().cpu().double()
    for i in range(b):
        n = min(max(int(cache_seqlens[i]), 0), cap, width)
        length = min(max(int(cache_seqlens[i]), 0), cap)
        if n == 0:
            continue
        pages = block_table[i].cpu().long()[torch.arange(n) // page]
        slots = pages * page + torch.arange(n) % page
        slots = torch.where((pages < 0) | (pages >= nb), torch.full_like(slots, nb * page), slots)
        keys = rows[slots]
        for t in range(sq):
            see = min(n, length - (sq - 1 - t)) if causal else n
            if see <= 0:
                continue
            s = keys[:see] @ q[i, t].T * scale                       # [see, h]
            a = keys[:see].abs() @ q[i, t].abs().T * abs(scale)
            z = lse[i, :, t]
            live = z != float("-inf")
            e = torch.exp(s[:, live] - z[live])
            w[i, :see] += e.sum(1)
            bound[i, :see] += (e * (a[:, live] + z[live].abs() + s[:, live].abs())).sum(1)
    return w, bound


def select_cache_rows(weights, cache_seqlens, budget, recent=0, columns=None):
    """-> rows, kept, kept weights in ``columns`` (default: budget) columns."""
    b, width = weights.shape
    rows = torch.full((b, budget), -1, dtype=torch.int32)
    kept = torch.zeros(b, dtype=torch.int32)
    vals = torch.zeros(b, budget if columns is None else columns, dtype=torch.float32)
    for i in range(b):
        n = min(max(int(cache_seqlens[i]), 0), width)
        w = weights[i].cpu().tolist()
        if n <= budget:
            ids = list(range(n))
        else:
            old = n - recent
            key = [float("-inf") if math.isnan(x) else x for x in w[:old]]
            # a NaN below -inf, equal weights by row
            order = sorted(range(old), key=lambda r: (math.isnan(w[r]), -key[r], r))
            ids = sorted(order[: budget - recent]) + list(range(old, n))
        rows[i, : len(ids)] = torch.tensor(ids, dtype=torch.int32)
        kept[i] = len(ids)
        vals[i, : len(ids)] = weights[i].cpu()[ids] if ids else vals[i, :0]
    return rows, kept, vals


def compact_cache(k_cache, block_table, rows, kept, out_block_table=None):
    """The cache after the move (a copy)."""
    cache = k_cache.detach().cpu().clone()
    src = k_cache.detach().cpu()
    nb, page = cache.shape[:2]
    table = block_table.cpu()
    out_table = table if out_block_table is None else out_block_table.cpu()

    def place(t, b, r):
        if r < 0 or r // page >= t.shape[1]:
            return None
        p = int(t[b, r // page])
        return (p, r % page) if 0 <= p < nb else None
    for b in range(rows.shape[0]):
        for j in range(min(max(int(kept[b]), 0), rows.shape[1])):
            dst = place(out_table, b, j)
            if dst is None:
                continue
            at = place(table, b, int(rows[b, j]))
            cache[dst] = src[at] if at is not None else 0
    return cache
