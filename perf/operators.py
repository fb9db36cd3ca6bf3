"""Dense MLA prefill and the eviction of cache rows by attention weight: what is timed, and on which inputs.

Four operators, in the order in which a serving loop calls them:

* ``prefill``  attention over whole prompts, packed one behind the other, causal, with grouped heads; the keys may
               reach further back than the queries (a prefix); output and log-sum-exp;
* ``weights``  how much attention each row of a paged latent cache got from a step's (or a window's) queries:
               sums over heads and query positions of exp(score - lse);
* ``select``   which rows of each sequence stay when only ``budget`` of them may: the last ``recent`` ones and the
               heaviest of the others, ties to the lowest row;
* ``compact``  the rows that stay, moved to the front of each sequence's (new) pages.

``own`` chooses between the plain forms below and the library's calls.  Lengths are given as text ("17,300")
because a case holds plain values only.
"""
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _lib():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forks-flash-mla-int_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flash_mla
    return flash_mla


def _ints(text):
    return [int(x) for x in text.split(",")]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


# ----------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One short question, alone on the GPU: the latency of a call.
        dict(name="prompt_short", op="prefill", dtype="bf16", heads=16, kv_heads=16, d_qk=192, d_v=128, causal=True,
             q_lens="23", k_lens="23"),
        # The prompts of a batch that arrived together, from one token to a few thousand, 16 heads a GPU.
        dict(name="prompts_ragged", op="prefill", dtype="bf16", heads=16, kv_heads=16, d_qk=192, d_v=128, causal=True,
             q_lens="1,7,64,129,255,300,511,640,777,1000,1023,1500,2047,2111,3300,4095",
             k_lens="1,7,64,129,255,300,511,640,777,1000,1023,1500,2047,2111,3300,4095"),
        # One long document.
        dict(name="prompt_long", op="prefill", dtype="bf16", heads=32, kv_heads=32, d_qk=192, d_v=128, causal=True,
             q_lens="16384", k_lens="16384"),
        # Grouped heads without a rotary part of their own, in fp16.
        dict(name="prompts_grouped", op="prefill", dtype="fp16", heads=32, kv_heads=8, d_qk=128, d_v=128, causal=True,
             q_lens="4096,2500,1333,3001", k_lens="4096,2500,1333,3001"),
        # The last piece of prompts that are taken in pieces: few queries, many keys before them.
        dict(name="prompt_pieces", op="prefill", dtype="bf16", heads=64, kv_heads=64, d_qk=192, d_v=128, causal=True,
             q_lens="512,301", k_lens="8192,4999"),
        # Weights of one decode step of a full batch, added to what earlier steps left.
        dict(name="weights_decode", op="weights", batch=128, s_q=1, heads=16, dim=576, page=64, lens=",".join(["4096"] * 128),
             causal=True, accumulate=True),
        # Weights that the last 64 tokens of long prompts give to all rows, before the first eviction.
        dict(name="weights_window", op="weights", batch=4, s_q=64, heads=128, dim=576, page=64,
             lens="8192,7001,5555,8191", causal=True, accumulate=False),
        # One sequence in its first steps.
        dict(name="weights_one", op="weights", batch=1, s_q=1, heads=16, dim=576, page=64, lens="700", causal=False,
             accumulate=False),
        # A few sequences just over their budget.
        dict(name="select_few", op="select", batch=4, lens="2048,1999,513,300", width=2048, budget=512, recent=64),
        # A full batch of long sequences cut down to an eighth.
        dict(name="select_batch", op="select", batch=64, lens=",".join(str(32768 - 37 * i) for i in range(64)),
             width=32768, budget=4096, recent=256),
        # The same two steps for the rows themselves.
        dict(name="compact_few", op="compact", batch=2, lens="1024,777", dim=576, page=64, budget=256),
        dict(name="compact_batch", op="compact", batch=16, lens=",".join(str(16384 - 101 * i) for i in range(16)),
             dim=576, page=64, budget=4096),
    ]


def _log_int(rng, lo, hi):
    import math
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(xs):
    return ",".join(str(x) for x in xs)


def draw(rng):
    cap = {"prefill": 2.6e12, "weights": 2.5e11, "bytes": 5.0e8}
    op = rng.choice(["prefill", "prefill", "weights", "weights", "select", "compact"])
    if op == "prefill":
        kv = rng.choice([1, 2, 4, 8, 16, 32])
        group = rng.choice([1, 1, 1, 2, 4, 5, 8])
        while kv * group > 64:
            group = max(1, group // 2)
        q = [_log_int(rng, 1, 16384) for _ in range(_log_int(rng, 1, 24))]
        before = rng.random() < 0.3
        k = [x + (_log_int(rng, 1, 8192) if before else 0) for x in q]
        d_qk = rng.choice([192, 192, 128])
        case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), heads=kv * group, kv_heads=kv, d_qk=d_qk, d_v=128,
                    causal=rng.random() < 0.8, q_lens=_text(q), k_lens=_text(k))
        while work(case)["flops"] > cap["prefill"] or work(case)["bytes"] > 2 * cap["bytes"] or max(k) > 16384:
            i = max(range(len(q)), key=lambda j: k[j])
            cut = max(1, q[i] * 3 // 4)
            k[i], q[i] = max(cut, k[i] * 3 // 4), cut
            case.update(q_lens=_text(q), k_lens=_text(k))
        return case
    if op == "weights":
        batch = _log_int(rng, 1, 128)
        lens = [_log_int(rng, 1, 16384) for _ in range(batch)]
        s_q = rng.choice([1, 1, 2, 3, 16, 33, 64])
        case = dict(op=op, batch=batch, s_q=s_q, heads=rng.choice([4, 16, 20, 32, 64, 128]), dim=rng.choice([576, 576, 512]),
                    page=rng.choice([16, 32, 64, 128, 256]), lens=_text(lens), causal=rng.random() < 0.7,
                    accumulate=rng.random() < 0.5)
        while work(case)["flops"] > cap["weights"] or work(case)["bytes"] > cap["bytes"]:
            lens = [max(1, x * 3 // 4) for x in lens]
            case["lens"] = _text(lens)
        return case
    if op == "select":
        batch = _log_int(rng, 1, 128)
        width = _log_int(rng, 64, 65536)
        while batch * width > 64 * 32768:
            batch = max(1, batch // 2)
        lens = [rng.randint(1, width) for _ in range(batch)]
        budget = _log_int(rng, 8, max(8, width // 2))
        return dict(op=op, batch=batch, lens=_text(lens), width=width, budget=budget, recent=rng.randint(0, budget))
    batch = _log_int(rng, 1, 32)
    lens = [_log_int(rng, 16, 16384) for _ in range(batch)]
    while sum(lens) > 16 * 15000:
        lens = [max(16, x // 2) for x in lens]
    return dict(op=op, batch=batch, lens=_text(lens), dim=rng.choice([576, 576, 512]), page=rng.choice([16, 32, 64, 128]),
                budget=_log_int(rng, 16, 4096))


def _visible(nq, nk, causal):
    """(query, key) pairs that the mask leaves: query i of nq sees the first nk - (nq - 1 - i) keys."""
    if not causal:
        return nq * nk
    first = nk - nq + 1                      # keys of query 0 (may be <= 0)
    if first >= 0:
        return nq * first + nq * (nq - 1) // 2
    return nk * (nk + 1) // 2                # the queries before the first key see none


def work(case):
    if case["op"] == "prefill":
        q, k = _ints(case["q_lens"]), _ints(case["k_lens"])
        h, hk, dq, dv = case["heads"], case["kv_heads"], case["d_qk"], case["d_v"]
        pairs = sum(_visible(a, b, case["causal"]) for a, b in zip(q, k))
        return {"bytes": 2 * (sum(q) * h * (dq + dv) + sum(k) * hk * (dq + dv)) + 4 * sum(q) * h,
                "flops": 2 * (dq + dv) * h * pairs}
    lens = _ints(case["lens"])
    if case["op"] == "weights":
        h, d, n = case["heads"], case["dim"], case["s_q"]
        pairs = sum(_visible(n, x, case["causal"]) for x in lens)
        return {"bytes": 2 * d * sum(lens) + case["batch"] * n * h * (2 * d + 4) + (8 if case["accumulate"] else 4) * sum(lens),
                "flops": 2 * d * h * pairs}
    if case["op"] == "select":
        return {"bytes": 4 * sum(lens) + 8 * case["batch"] * case["budget"] + 8 * case["batch"], "flops": sum(lens)}
    kept = sum(min(x, case["budget"]) for x in lens)
    return {"bytes": kept * (4 * case["dim"] + 4), "flops": 0}


# ----------------------------------------------------------------------------------------------- inputs
def _cu(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


def _paged(g, case, extra_pages=0):
    """A paged bf16 cache whose pages lie in scrambled order, the rows past each length NaN.  A few rows of each
    sequence (its first ones and a random 2 %) lie along a direction that the queries share: they get most of the
    attention, as in a trained model."""
    lens, page, dim, batch = _ints(case["lens"]), case["page"], case["dim"], case["batch"]
    pages = [(n + page - 1) // page for n in lens]
    most = max(pages) + (1 if extra_pages == 0 else 0)
    total = sum(pages) + extra_pages
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(batch, most, dtype=torch.int32, device=DEV)
    cache = torch.empty(total, page, 1, dim, dtype=torch.bfloat16, device=DEV)
    dirs = _randn(g, batch, dim)
    at = 0
    for b, n in enumerate(lens):
        mine = perm[at:at + pages[b]]
        at += pages[b]
        table[b, :pages[b]] = mine
        rows = _randn(g, pages[b] * page, dim)
        heavy = torch.rand(pages[b] * page, generator=g, device=DEV) < 0.02
        heavy[:4] = True
        rows += 0.4 * heavy[:, None] * dirs[b]
        rows[n:] = float("nan")
        cache[mine.long()] = rows.to(torch.bfloat16).view(pages[b], page, 1, dim)
    return cache, table, perm[at:], dirs


def _sequence_rows(cache, table_row, n):
    page = cache.shape[1]
    ids = table_row[: (n + page - 1) // page].long()
    return cache[ids].reshape(-1, cache.shape[-1])[:n]


def _keep_mask(nq, nk):
    """True where query i of nq may see key j of nk: the queries are the sequence's last nq positions."""
    i = torch.arange(nq, device=DEV)[:, None]
    j = torch.arange(nk, device=DEV)[None, :]
    return j <= i + (nk - nq)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "prefill":
        ql, kl = _ints(case["q_lens"]), _ints(case["k_lens"])
        dt = DTYPES[case["dtype"]]
        u = _randn(g, case["kv_heads"], case["d_qk"])
        group = case["heads"] // case["kv_heads"]
        q = _randn(g, sum(ql), case["heads"], case["d_qk"]) + 0.5 * u.repeat_interleave(group, 0)
        k = _randn(g, sum(kl), case["kv_heads"], case["d_qk"])
        heavy = torch.rand(sum(kl), generator=g, device=DEV) < 0.02
        at = 0
        for n in kl:
            heavy[at] = True                 # the first token of a prompt draws attention from all others
            at += n
        k += 0.8 * heavy[:, None, None] * u
        v = _randn(g, sum(kl), case["kv_heads"], case["d_v"])
        return dict(case=case, q=q.to(dt), k=k.to(dt), v=v.to(dt), cu_q=_cu(ql), cu_k=_cu(kl))
    lens = _ints(case["lens"])
    seqlens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if op == "weights":
        cache, table, _, dirs = _paged(g, case)
        b, n, h, d = case["batch"], case["s_q"], case["heads"], case["dim"]
        q = (_randn(g, b, n, h, d) + 0.5 * dirs[:, None, None, :]).to(torch.bfloat16)
        lse = torch.empty(b, h, n, dtype=torch.float32, device=DEV)      # what the attention call returned
        for i, m in enumerate(lens):
            s = torch.einsum("nhd,md->hnm", q[i].float(), _sequence_rows(cache, table[i], m).float()) * d ** -0.5
            if case["causal"]:
                s = s.masked_fill(~_keep_mask(n, m), float("-inf"))
            lse[i] = torch.logsumexp(s, dim=-1)
        state = dict(case=case, q=q, cache=cache, table=table, seqlens=seqlens, lse=lse)
        if case["accumulate"]:
            state["weights"] = torch.rand(b, table.shape[1] * case["page"], generator=g, device=DEV)
        return state
    if op == "select":
        # Sums over many queries: heavy-tailed, with rows that nobody looked at (exact zeros, so ties).
        w = torch.exp(2.0 * _randn(g, case["batch"], case["width"]))
        w = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.3, torch.zeros_like(w), w)
        return dict(case=case, weights=w, seqlens=seqlens)
    # compact: a random ascending choice of rows, and fresh pages of the same cache to move them to
    page, budget = case["page"], case["budget"]
    per = (budget + page - 1) // page
    cache, table, spare, _ = _paged(g, case, extra_pages=per * case["batch"])
    rows = torch.full((case["batch"], budget), -1, dtype=torch.int32, device=DEV)
    for i, n in enumerate(lens):
        m = min(n, budget)
        rows[i, :m] = torch.randperm(n, generator=g, device=DEV)[:m].sort().values.to(torch.int32)
    kept = seqlens.clamp(max=budget)
    cache[spare.long()] = 0
    return dict(case=case, cache=cache, table=table, rows=rows, kept=kept, new_table=spare.view(case["batch"], per).contiguous())


# ----------------------------------------------------------------------------------------------- plain forms
def _plain_prefill(st):
    case = st["case"]
    h, hk = case["heads"], case["kv_heads"]
    scale = case["d_qk"] ** -0.5
    out = torch.zeros(st["q"].shape[0], h, case["d_v"], dtype=torch.float32, device=DEV)
    lse = torch.full((h, st["q"].shape[0]), float("-inf"), dtype=torch.float32, device=DEV)
    qa = ka = 0
    for nq, nk in zip(_ints(case["q_lens"]), _ints(case["k_lens"])):
        step = max(1, min(hk, (1 << 28) // max(1, nq * nk * (h // hk))))        # kv heads at a time: about 1 GB of scores
        mask = _keep_mask(nq, nk) if case["causal"] else None
        for a in range(0, hk, step):
            c = min(hk, a + step)
            heads = slice(a * (h // hk), c * (h // hk))
            q = st["q"][qa:qa + nq, heads].float().reshape(nq, c - a, h // hk, -1)
            k = st["k"][ka:ka + nk, a:c].float()
            v = st["v"][ka:ka + nk, a:c].float()
            s = torch.einsum("qcgd,kcd->cgqk", q, k) * scale
            if mask is not None:
                s = s.masked_fill(~mask, float("-inf"))
            m = s.amax(-1, keepdim=True)
            m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
            p = torch.exp(s - m)
            del s
            l = p.sum(-1, keepdim=True)
            o = torch.einsum("cgqk,kcd->qcgd", p, v) / l.squeeze(-1).permute(2, 0, 1).unsqueeze(-1).clamp(min=1e-30)
            del p
            out[qa:qa + nq, heads] = o.reshape(nq, -1, case["d_v"])
            lse[heads, qa:qa + nq] = (m + torch.log(l)).squeeze(-1).reshape(-1, nq)
        qa += nq
        ka += nk
    return out.to(st["q"].dtype), lse


def _plain_weights(st):
    case = st["case"]
    width = st["table"].shape[1] * case["page"]
    w = st["weights"].clone() if case["accumulate"] else torch.zeros(case["batch"], width, dtype=torch.float32, device=DEV)
    n, h = case["s_q"], case["heads"]
    for i, m in enumerate(_ints(case["lens"])):
        k = _sequence_rows(st["cache"], st["table"][i], m).float()
        s = (st["q"][i].float().reshape(n * h, -1) @ k.t()).view(n, h, m) * case["dim"] ** -0.5
        p = torch.exp(s - st["lse"][i].t().unsqueeze(-1))
        if case["causal"]:
            p = torch.where(_keep_mask(n, m)[:, None, :], p, torch.zeros_like(p))
        w[i, :m] += p.sum((0, 1))
    return w


def _plain_select(st):
    case = st["case"]
    b, budget, recent = case["batch"], case["budget"], case["recent"]
    rows = torch.full((b, budget), -1, dtype=torch.int32, device=DEV)
    kept = torch.zeros(b, dtype=torch.int32, device=DEV)
    vals = torch.zeros(b, budget, dtype=torch.float32, device=DEV)
    for i, n in enumerate(_ints(case["lens"])):
        w = st["weights"][i, :n]
        if n <= budget:
            ids = torch.arange(n, device=DEV)
        else:
            old = n - recent
            top = torch.sort(w[:old], descending=True, stable=True).indices[: budget - recent].sort().values
            ids = torch.cat([top, torch.arange(old, n, device=DEV)])
        rows[i, : ids.numel()] = ids.to(torch.int32)
        vals[i, : ids.numel()] = w[ids]
        kept[i] = ids.numel()
    return rows, kept, vals


def _plain_compact(st):
    page = st["case"]["page"]
    flat = st["cache"].view(-1, st["cache"].shape[-1])
    j = torch.arange(st["rows"].shape[1], device=DEV)[None, :]
    live = j < st["kept"][:, None]
    src = st["rows"].clamp(min=0).long()
    src = torch.gather(st["table"].long(), 1, src // page) * page + src % page
    dst = torch.gather(st["new_table"].long(), 1, (j // page).expand_as(src)) * page + j % page
    flat[dst[live]] = flat[src[live]]
    return st["cache"]


# ----------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"prefill": _plain_prefill, "weights": _plain_weights, "select": _plain_select,
                "compact": _plain_compact}[op](state)
    lib = _lib()
    if op == "prefill":
        return lib.dense_mla_prefill(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], causal=case["causal"])
    if op == "weights":
        # A program keeps one accumulator and adds to it in place; the copy lets the pass be repeated.
        acc = state["weights"].clone() if case["accumulate"] else None
        return lib.mla_cache_row_weights(state["q"], state["cache"], state["table"], state["seqlens"], state["lse"],
                                         causal=case["causal"], weights=acc)
    if op == "select":
        return lib.mla_select_cache_rows(state["weights"], state["seqlens"], case["budget"], case["recent"])
    lib.mla_compact_cache(state["cache"], state["table"], state["rows"], state["kept"], out_block_table=state["new_table"])
    return state["cache"]


# ----------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """``prefill`` and ``weights`` from their definitions, one query head at a time in float64.  ``select`` and
    ``compact`` choose and move values and compute none."""
    if case["op"] not in ("prefill", "weights"):
        return None
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "prefill":
        if work(case)["flops"] > 4e12:
            return None
        q, k, v = st["q"], st["k"], st["v"]
        out = torch.zeros(q.shape[0], case["heads"], case["d_v"], dtype=f64, device=DEV)
        lse = torch.full((case["heads"], q.shape[0]), float("-inf"), dtype=f64, device=DEV)
        group = case["heads"] // case["kv_heads"]
        qb, kb = st["cu_q"].tolist(), st["cu_k"].tolist()
        for s in range(len(qb) - 1):
            nq, nk = qb[s + 1] - qb[s], kb[s + 1] - kb[s]
            for h in range(case["heads"]):
                kk = k[kb[s]:kb[s + 1], h // group].to(f64)
                vv = v[kb[s]:kb[s + 1], h // group].to(f64)
                for a in range(0, nq, 4096):
                    c = min(nq, a + 4096)
                    x = torch.matmul(q[qb[s] + a:qb[s] + c, h].to(f64), kk.t()) / case["d_qk"] ** 0.5
                    if case["causal"]:
                        last = torch.arange(a, c, device=DEV) + (nk - nq)
                        x[torch.arange(nk, device=DEV)[None, :] > last[:, None]] = float("-inf")
                    z = torch.logsumexp(x, dim=1)
                    seen = torch.isfinite(z)
                    p = torch.exp(x - torch.where(seen, z, torch.zeros_like(z))[:, None])
                    out[qb[s] + a:qb[s] + c, h] = torch.matmul(p, vv)
                    lse[h, qb[s] + a:qb[s] + c] = z
        return out, lse
    lens, page = _ints(case["lens"]), case["page"]
    res = torch.zeros(case["batch"], st["table"].shape[1] * page, dtype=f64, device=DEV)
    if case["accumulate"]:
        res += st["weights"].to(f64)
    for b, m in enumerate(lens):
        slots = torch.arange(m, device=DEV)
        slots = st["table"][b].long()[slots // page] * page + slots % page
        keys = st["cache"].view(-1, case["dim"])[slots].to(f64)
        for i in range(case["s_q"]):
            sees = m if not case["causal"] else m - (case["s_q"] - 1 - i)
            if sees <= 0:
                continue
            x = torch.matmul(keys[:sees], st["q"][b, i].to(f64).t()) / case["dim"] ** 0.5
            res[b, :sees] += torch.exp(x - st["lse"][b, :, i].to(f64)[None, :]).sum(1)
    return res
