"""float64 CPU oracle of dense MLA prefill (test infrastructure, not product).  Written from the definition; the
reference has no such operator.

Sequence b owns query rows [cu_q[b], cu_q[b + 1]) and key rows [cu_k[b], cu_k[b + 1]); with nq and nk of them, query i
sees the first nk - (nq - 1 - i) keys under the causal mask, else all; s = scale q . k, lse = log sum exp s,
out = sum exp(s - lse) v; a query that sees no key has zeros and -inf.
"""
from __future__ import annotations

import torch


def dense_mla_prefill(q, k, v, cu_q, cu_k, scale=None, causal=True):
    """-> out [tq, h, dv], lse [h, tq], and two quantities that rounding bounds need: sum_j p_j |v_j| in out's
    layout, and the largest |scale| sum_d |q_d k_d| over a query's keys in lse's."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    cu_q, cu_k = cu_q.tolist(), cu_k.tolist()
    h, hk = q.shape[1], k.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape[0], h, v.shape[2], dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((h, q.shape[0]), float("-inf"), dtype=torch.float64)
    size = torch.zeros(h, q.shape[0], dtype=torch.float64)
    for b in range(len(cu_q) - 1):
        qs, ks = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        nq, nk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if nq == 0 or nk == 0:
            continue
        keep = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            keep = torch.arange(nk)[None, :] < (nk - (nq - 1 - torch.arange(nq)))[:, None]
        for head in range(h):
            kk, vv = k[ks, head // (h // hk)], v[ks, head // (h // hk)]
            s = (q[qs, head] @ kk.T * scale).masked_fill(~keep, float("-inf"))
            z = torch.logsumexp(s, dim=1)
            p = torch.where(keep & torch.isfinite(z)[:, None], torch.exp(s - z[:, None]), torch.zeros(()).double())
            lse[head, qs] = z
            out[qs, head] = p @ vv
            mag[qs, head] = p @ vv.abs()
            size[head, qs] = torch.where(keep, q[qs, head].abs() @ kk.abs().T * abs(scale), torch.zeros(()).double()).amax(1)
    return out, lse, mag, size
