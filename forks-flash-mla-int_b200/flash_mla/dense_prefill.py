"""Prefill of dense MLA layers: attention of whole prompts over keys and values expanded to heads.

``flash_mla_with_kvcache`` attends to the latent rows themselves (the absorbed form, one kv head of 576 dims), which
is right for a few query positions.  For a whole prompt the expanded form needs 3.4 times less arithmetic:
192 dims for the scores and 128 for the values of each head instead of 576 and 512.  No counterpart in the
reference.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._loader import load_torch_extension

load_torch_extension()

# The op checks its arguments itself, in C++; the checks below are made when it has refused, to say what is wrong with a
# ValueError (a small call is bound by the host).
_prefill = torch.ops.flash_mla.dense_mla_prefill.default


def dense_mla_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                      cu_seqlens_k: torch.Tensor, softmax_scale: Optional[float] = None,
                      causal: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of packed prompts.

    Arguments:
        q: (total_q, num_heads, 192 or 128) bfloat16 or float16.
        k: (total_k, num_kv_heads, 192 or 128), v: (total_k, num_kv_heads, 128), of q's type; num_heads is a
            multiple of num_kv_heads, and query head h reads kv head h // (num_heads // num_kv_heads).
        cu_seqlens_q, cu_seqlens_k: (batch_size + 1,) int32 offsets; sequence b owns the rows
            [cu_seqlens_q[b], cu_seqlens_q[b + 1]) of q and [cu_seqlens_k[b], cu_seqlens_k[b + 1]) of k and v.
        softmax_scale: defaults to head_dim ** -0.5.
        causal: query i of a sequence with nq queries and nk keys sees its first nk - (nq - 1 - i) keys, so the
            queries are the last nq positions and an earlier part of the prompt may stand in front of the keys.

    Rows of any stride are read in place as long as they start on 16 bytes and their dims are contiguous; others
    are copied first.

    Returns out (total_q, num_heads, 128) of q's type and softmax_lse (num_heads, total_q) float32, the natural
    logarithm of the sum of exponentials.  Scores, sums and the output before its last rounding are fp32; the weights
    are rounded to q's type for the second product, so out is up to 1.5 times as far from the exact value as one
    rounding at the end would leave it.  A query that sees no key gets zeros and -inf; rows of q behind the
    last sequence are not written."""
    try:
        scale = q.shape[-1] ** (-0.5) if softmax_scale is None else float(softmax_scale)
        return _prefill(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal)
    except (RuntimeError, NotImplementedError, IndexError, ZeroDivisionError):
        _check_call(q, k, v, cu_seqlens_q, cu_seqlens_k)
        raise


def _check_call(q, k, v, cu_seqlens_q, cu_seqlens_k) -> None:
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("expected q, k and v of shape [tokens, heads, head_dim]")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"expected q, k and v all bfloat16 or all float16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.shape[2] not in (192, 128) or k.shape[2] != q.shape[2] or v.shape[2] != 128:
        raise ValueError(f"expected head dims 192 or 128 (q, k) and 128 (v), got {q.shape[2]}, {k.shape[2]}, {v.shape[2]}")
    if k.shape[:2] != v.shape[:2]:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ in tokens or heads")
    if q.shape[1] < 1 or k.shape[1] < 1 or q.shape[1] % k.shape[1] != 0:
        raise ValueError(f"{q.shape[1]} query heads are not a multiple of {k.shape[1]} kv heads")
    for name, cu in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        if cu.dim() != 1 or cu.dtype != torch.int32 or cu.shape[0] < 1:
            raise ValueError(f"expected {name} int32 [batch + 1], got {cu.dtype} {tuple(cu.shape)}")
    if cu_seqlens_q.shape != cu_seqlens_k.shape:
        raise ValueError(f"cu_seqlens_q has {cu_seqlens_q.shape[0]} entries, cu_seqlens_k {cu_seqlens_k.shape[0]}")
