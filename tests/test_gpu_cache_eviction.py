"""GPU tests of cache-row eviction: weights against the float64 oracle, selection and compaction exactly.

Tolerance of the weights: each term exp(s - lse) is off by what its exponent is off, d 2^-23 scale sum |q k| for the
dot product in fp32 plus 2^-22 of |s| and |lse| for scaling and subtraction, and by 2^-21 for the exponential; the sum of
c terms adds c 2^-23 of itself.  The oracle returns sum term * (scale sum |q k| + |s| + |lse|), so the bound is
(d + 4) 2^-23 times that plus (c 2^-23 + 2^-21) w.
"""
import ctypes
import random

import pytest
import torch

from helpers import device_status
import oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fm():
    import flash_mla
    return flash_mla


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert device_status() == 0, "a kernel wait ran out (device status word set)"


def paged(lens, s_q=1, h=16, d=576, page=64, seed=0, extra=0, spare_columns=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [(n + page - 1) // page for n in lens]
    perm = torch.randperm(sum(pages) + extra, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(pages + [1]) + spare_columns), -1, dtype=torch.int32)
    cache = torch.full((sum(pages) + extra + 1, page, 1, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        table[b, :pages[b]] = perm[at:at + pages[b]]
        at += pages[b]
        rows = torch.full((pages[b] * page, d), float("nan"), device="cuda")
        rows[:n] = torch.randn(n, d, generator=g, device="cuda")
        cache[table[b, :pages[b]].long().cuda()] = rows.to(torch.bfloat16).view(pages[b], page, 1, d)
    q = torch.randn(len(lens), s_q, h, d, generator=g, device="cuda").to(torch.bfloat16)
    return dict(q=q, k_cache=cache, block_table=table.cuda(), cache_seqlens=torch.tensor(lens, dtype=torch.int32, device="cuda")), perm[at:]


def lse_of(kw, causal, scale=None):
    """log-sum-exp of the queries, in float64 on the host, as fp32."""
    q, cache = kw["q"].cpu().double(), kw["k_cache"].cpu()
    nb, page, _, d = cache.shape
    b, sq, h, _ = q.shape
    lse = torch.full((b, h, sq), float("-inf"), dtype=torch.float64)
    table = kw["block_table"].cpu()
    for i in range(b):
        n = min(max(int(kw["cache_seqlens"][i]), 0), table.shape[1] * page)
        if n == 0:
            continue
        pages = table[i].long()[torch.arange(n) // page]
        rows = torch.zeros(n, d, dtype=torch.float64)
        ok = (pages >= 0) & (pages < nb)
        rows[ok] = cache[pages[ok], (torch.arange(n) % page)[ok], 0].double()
        for t in range(sq):
            see = n - (sq - 1 - t) if causal else n
            if see > 0:
                lse[i, :, t] = torch.logsumexp(rows[:see] @ q[i, t].T * (d ** -0.5 if scale is None else scale), dim=0)
    return lse.float().cuda()


def check_weights(got, kw, lse, causal, weights=None, scale=None, what=""):
    ref, bound = oracle.cache_row_weights(kw["q"], kw["k_cache"], kw["block_table"], kw["cache_seqlens"], lse, scale=scale, causal=causal,
                                          weights=weights, width=got.shape[1])
    d, c = kw["q"].shape[3], kw["q"].shape[1] * kw["q"].shape[2]
    tol = (d + 4) * 2.0 ** -23 * bound + (c * 2.0 ** -23 + 2.0 ** -21) * ref.abs() + 1e-30
    w = got.cpu().double()
    assert torch.isfinite(w).all(), f"{what}: non-finite weight"
    bad = (w - ref).abs() - tol
    assert bad.max() <= 0, f"{what}: off by {float((w - ref).abs().max()):.3e}, over the bound at {torch.nonzero(bad > 0)[:4].tolist()}"


@pytest.mark.parametrize("d", [576, 512])
@pytest.mark.parametrize("h", [1, 4, 16, 20, 32, 64, 128])
@pytest.mark.parametrize("s_q", [1, 2, 5])
def test_weights_heads_and_positions(fm, d, h, s_q):
    kw, _ = paged([300, 1, 129, 64], s_q=s_q, h=h, d=d, seed=h + s_q)
    lse = lse_of(kw, True)
    got = fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=True)
    assert got.shape == (4, kw["block_table"].shape[1] * 64)
    check_weights(got, kw, lse, True, what=f"d={d} h={h} s_q={s_q}")


@pytest.mark.parametrize("lens", [[1], [127], [128], [129], [255], [256], [257], [0, 3], [700, 0, 5], [1500]])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_lengths(fm, lens, causal):
    kw, _ = paged(lens, s_q=3, h=16, seed=len(lens))
    lse = lse_of(kw, causal)
    check_weights(fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=causal), kw, lse, causal, what=f"{lens}")


@pytest.mark.parametrize("page", [8, 16, 24, 32, 48, 64, 96, 128, 256, 384])
def test_weights_page_sizes(fm, page):
    kw, _ = paged([500, 77], h=16, page=page, seed=page)
    lse = lse_of(kw, False)
    check_weights(fm.mla_cache_row_weights(**kw, softmax_lse=lse), kw, lse, False, what=f"page={page}")


@pytest.mark.parametrize("s_q,h", [(40, 16), (16, 128), (33, 20), (64, 64)])
def test_weights_of_a_window(fm, s_q, h):
    """Hundreds to thousands of query columns; some sequences shorter than the window."""
    kw, _ = paged([400, 20, 129], s_q=s_q, h=h, seed=s_q)
    lse = lse_of(kw, True)
    check_weights(fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=True), kw, lse, True, what=f"{s_q} x {h}")
    lse = lse_of(kw, False)
    check_weights(fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=False), kw, lse, False, what=f"{s_q} x {h} full")


def test_weights_accumulate_into_views(fm):
    kw, _ = paged([200, 130], s_q=2, h=16, seed=3)
    lse = lse_of(kw, True)
    g = torch.Generator(device="cuda").manual_seed(4)
    for width in (150, 256, 300, 131):                       # narrower and wider than the sequences
        buf = torch.rand(2, width + 5, generator=g, device="cuda")
        w = buf[:, 3:3 + width]
        before = w.clone()
        got = fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=True, weights=w)
        assert got.data_ptr() == w.data_ptr()
        check_weights(got, kw, lse, True, weights=before, what=f"width {width}")
        for b, n in enumerate((200, 130)):
            assert torch.equal(w[b, min(n, width):], before[b, min(n, width):])
        assert (buf[:, :3] != 0).all() and (buf[:, 3 + width:] != 0).all()


def test_weights_from_the_lse_of_the_decode(fm):
    """The decode's own lse: a query's weights sum to one (its scores round differently: 1e-3)."""
    kw, _ = paged([900, 64, 333], s_q=2, h=16, seed=5)
    meta, splits = fm.get_mla_metadata(kw["cache_seqlens"], 32, 1)
    _, lse = fm.flash_mla_with_kvcache(kw["q"], kw["k_cache"], kw["block_table"], kw["cache_seqlens"], 512, meta, splits, causal=True)
    w = fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=True)
    check_weights(w, kw, lse, True)
    assert (w.sum(1) - 32).abs().max() < 32e-3


def test_weights_skip_queries_without_rows_and_bad_pages(fm):
    kw, _ = paged([100, 200], s_q=2, h=4, seed=6)
    lse = lse_of(kw, False)
    lse[0, 1, 0] = float("-inf")
    kw["block_table"][1, 1] = -5
    kw["block_table"][1, 2] = 1 << 20
    got = fm.mla_cache_row_weights(**kw, softmax_lse=lse)
    check_weights(got, kw, lse, False)


def test_weights_lengths_out_of_range(fm):
    kw, _ = paged([100, 64], h=4, seed=7, spare_columns=0)
    kw["cache_seqlens"] = torch.tensor([-3, 100000], dtype=torch.int32, device="cuda")
    kw["k_cache"].nan_to_num_()
    lse = lse_of(kw, False)
    check_weights(fm.mla_cache_row_weights(**kw, softmax_lse=lse), kw, lse, False)


def test_weights_strided_cache_table_and_q(fm):
    kw, _ = paged([300, 40], s_q=2, h=8, d=512, seed=8)
    wide = torch.full((kw["k_cache"].shape[0], 64, 1, 576 + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[..., :512] = kw["k_cache"]
    kw["k_cache"] = wide[..., :512]
    kw["block_table"] = torch.cat([kw["block_table"], torch.full_like(kw["block_table"], 3)], 1)[:, : kw["block_table"].shape[1]]
    kw["q"] = kw["q"].transpose(1, 2).contiguous().transpose(1, 2)
    lse = lse_of(kw, True)
    check_weights(fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=True, softmax_scale=0.03), kw, lse, True, scale=0.03)


def test_weights_many_sequences_same_bits_streams_and_graph(fm):
    kw, _ = paged([(37 * i) % 300 for i in range(150)], h=16, seed=9)
    lse = lse_of(kw, False)
    one = fm.mla_cache_row_weights(**kw, softmax_lse=lse)
    check_weights(one, kw, lse, False)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        two = fm.mla_cache_row_weights(**kw, softmax_lse=lse)
    torch.cuda.synchronize()
    assert torch.equal(one, two)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        three = fm.mla_cache_row_weights(**kw, softmax_lse=lse)
    kw["cache_seqlens"].copy_(kw["cache_seqlens"].flip(0).minimum(kw["cache_seqlens"]))
    lse.copy_(lse_of(kw, False))
    graph.replay()
    torch.cuda.synchronize()
    check_weights(three, kw, lse, False, what="replay")


# ----------------------------------------------------------------------------- selection
def same_selection(fm, w, lens, budget, recent):
    got = fm.mla_select_cache_rows(w, lens, budget, recent)
    ref = oracle.select_cache_rows(w, lens, budget, recent)
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.int32
    assert torch.equal(got[1].cpu(), ref[1])
    assert torch.equal(got[0].cpu(), ref[0]), f"budget {budget} recent {recent}"
    assert torch.equal(got[2].cpu().view(torch.int32), ref[2].view(torch.int32))


@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (7, 3), (64, 0), (64, 64), (500, 17), (2000, 100)])
@pytest.mark.parametrize("width", [1, 33, 700, 1999])
def test_select_sizes(fm, budget, recent, width):
    g = torch.Generator(device="cuda").manual_seed(budget + width)
    lens = torch.tensor([width, 0, max(1, width // 2), min(width, budget), min(width, budget + 1)], dtype=torch.int32, device="cuda")
    w = torch.randn(5, width, generator=g, device="cuda").exp()
    same_selection(fm, w, lens, budget, recent)


def test_select_ties_signs_and_specials(fm):
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.tensor([0.0, -0.0, 1.0, -1.0, float("inf"), float("-inf"), float("nan"), 1e-40, -1e-40, 3e38], device="cuda")
    w = base[torch.randint(0, 10, (6, 1500), generator=g, device="cuda")]
    w[4] = 0.0                                                # nothing but ties
    w[5] = float("nan")
    lens = torch.tensor([1500, 1499, 1000, 700, 1500, 1400], dtype=torch.int32, device="cuda")
    for budget, recent in ((10, 0), (100, 33), (333, 1), (999, 0), (1499, 0)):
        same_selection(fm, w, lens, budget, recent)


def test_select_long_rows_and_views(fm):
    g = torch.Generator(device="cuda").manual_seed(2)
    buf = torch.rand(3, 140000, generator=g, device="cuda")
    buf = torch.where(buf < 0.4, torch.zeros_like(buf), buf)
    lens = torch.tensor([139990, 70001, 5000], dtype=torch.int32, device="cuda")
    same_selection(fm, buf[:, 7:139997], lens, 9000, 128)
    same_selection(fm, buf.t().contiguous().t(), lens, 333, 0)


def test_select_very_long_row(fm):
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.rand(1, 1_000_003, generator=g, device="cuda").mul(1 << 18).floor()
    lens = torch.tensor([1_000_003], dtype=torch.int32, device="cuda")
    rows, kept, vals = fm.mla_select_cache_rows(w, lens, 65536, 1000)
    old = 1_000_003 - 1000
    top = torch.sort(w[0, :old], descending=True, stable=True).indices[: 65536 - 1000].sort().values
    ids = torch.cat([top, torch.arange(old, 1_000_003, device="cuda")])
    assert torch.equal(rows[0].long(), ids) and int(kept) == 65536 and torch.equal(vals[0], w[0, ids])


def test_select_lengths_out_of_range(fm):
    w = torch.rand(3, 50, device="cuda")
    same_selection(fm, w, torch.tensor([-7, 1000, 50], dtype=torch.int32, device="cuda"), 20, 5)
    rows, kept, _ = fm.mla_select_cache_rows(w[:, :0], torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), 4)
    assert (rows == -1).all() and (kept == 0).all()


def test_select_many_sequences_and_graph(fm):
    g = torch.Generator(device="cuda").manual_seed(5)
    w = torch.rand(400, 600, generator=g, device="cuda")
    lens = torch.randint(0, 601, (400,), generator=g, device="cuda").to(torch.int32)
    same_selection(fm, w, lens, 100, 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fm.mla_select_cache_rows(w, lens, 100, 20)
    w.copy_(torch.rand(400, 600, generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, oracle.select_cache_rows(w, lens, 100, 20)):
        assert torch.equal(a.cpu(), b)


# ----------------------------------------------------------------------------- compaction
def same_bytes(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


def ascending(lens, budget, seed):
    g = torch.Generator().manual_seed(seed)
    rows = torch.full((len(lens), budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        m = min(n, budget)
        rows[b, :m] = torch.randperm(n, generator=g)[:m].sort().values.to(torch.int32)
    return rows.cuda(), torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page", [1, 5, 16, 64, 100, 128])
@pytest.mark.parametrize("d", [576, 512, 8, 40])
@pytest.mark.parametrize("in_place", [True, False])
def test_compact(fm, page, d, in_place):
    lens, budget = [500, 3, 0, 129, 260], 120
    per = (budget + page - 1) // page
    kw, spare = paged(lens, h=1, d=d, page=page, seed=page + d, extra=0 if in_place else per * len(lens))
    rows, kept = ascending(lens, budget, page)
    out = None if in_place else spare.view(len(lens), per).cuda()
    want = oracle.compact_cache(kw["k_cache"], kw["block_table"], rows, kept, out)
    assert fm.mla_compact_cache(kw["k_cache"], kw["block_table"], rows, kept, out_block_table=out) is None
    assert same_bytes(kw["k_cache"], want)


def test_compact_long_in_place_and_own_table_as_target(fm):
    lens = [20000, 9000]
    for budget, given in ((12000, False), (19999, True), (300, False)):
        kw, _ = paged(lens, h=1, d=64, page=16, seed=budget)
        rows, kept = ascending(lens, budget, budget)
        want = oracle.compact_cache(kw["k_cache"], kw["block_table"], rows, kept)
        table = kw["block_table"]
        if given:                                             # a strided table that the binding has to copy
            table = torch.stack([table, table], 2)[:, :, 0]
        fm.mla_compact_cache(kw["k_cache"], table, rows, kept, out_block_table=table if given else None)
        assert same_bytes(kw["k_cache"], want)


def test_compact_rows_and_pages_out_of_range(fm):
    kw, spare = paged([100, 50], h=1, d=64, page=16, seed=1, extra=8)
    rows = torch.tensor([[3, -4, 100000, 17], [49, 48, 47, 5]], dtype=torch.int32, device="cuda")     # any order into other pages
    for kept in ([4, 4], [-2, 9], [2, 0]):
        kept = torch.tensor(kept, dtype=torch.int32, device="cuda")
        for out in (spare.view(2, 4)[:, :1], torch.tensor([[-1], [1 << 20]], dtype=torch.int32)):
            cache = kw["k_cache"].clone()
            want = oracle.compact_cache(cache, kw["block_table"], rows, kept, out)
            fm.mla_compact_cache(cache, kw["block_table"], rows, kept, out_block_table=out.cuda().contiguous())
            assert same_bytes(cache, want)
    kw["block_table"][0, 0] = -1
    cache = kw["k_cache"].clone()
    kept = torch.tensor([4, 4], dtype=torch.int32, device="cuda")
    want = oracle.compact_cache(cache, kw["block_table"], rows, kept, spare.view(2, 4)[:, :1])
    fm.mla_compact_cache(cache, kw["block_table"], rows, kept, out_block_table=spare.view(2, 4)[:, :1].cuda())
    assert same_bytes(cache, want)


def test_compact_strided_cache_and_empty_calls(fm):
    kw, _ = paged([70, 33], h=1, d=64, page=16, seed=2)
    wide = torch.randn(kw["k_cache"].shape[0], 2, 16, 1, 96, device="cuda").to(torch.bfloat16)
    wide[:, 1, :, :, :64] = kw["k_cache"]
    view = wide[:, 1, :, :, :64]
    rest = wide[:, 1, :, :, 64:].clone(), wide[:, 0].clone()
    rows, kept = ascending([70, 33], 20, 3)
    want = oracle.compact_cache(view, kw["block_table"], rows, kept)
    fm.mla_compact_cache(view, kw["block_table"], rows, kept)
    assert same_bytes(view.contiguous(), want)
    assert torch.equal(wide[:, 1, :, :, 64:], rest[0]) and torch.equal(wide[:, 0], rest[1])
    fm.mla_compact_cache(view, kw["block_table"], rows[:, :0], kept)
    fm.mla_compact_cache(view, kw["block_table"][:0], rows[:0], kept[:0])
    assert same_bytes(view.contiguous(), want)


# ----------------------------------------------------------------------------- as they are used together
def test_prompt_decode_evict_decode(fm):
    """A small dense MLA layer: the prompt by prefill in the expanded form, its latent rows in the paged cache, a
    decode step and the weights of its queries, eviction in place, and a decode over what stayed.  The prefill's
    last position equals a decode of the same query in the absorbed form; the decode after the eviction equals
    attention over the rows that were kept."""
    torch.manual_seed(0)
    dev, h, page, lens, budget, recent = "cuda", 16, 16, [130, 300, 40], 64, 16
    total = sum(lens)
    latent = torch.randn(total, 576, device=dev).to(torch.bfloat16)             # 512 latent + 64 rotary dims
    w_k = (torch.randn(h, 128, 512, device=dev) / 512 ** 0.5).to(torch.bfloat16)
    w_v = (torch.randn(h, 128, 512, device=dev) / 512 ** 0.5).to(torch.bfloat16)
    q = torch.randn(total, h, 192, device=dev).to(torch.bfloat16)
    scale = 192 ** -0.5
    k = torch.cat([torch.einsum("tl,hnl->thn", latent[:, :512].float(), w_k.float()), latent[:, None, 512:].float().expand(-1, h, -1)], -1).to(torch.bfloat16)
    v = torch.einsum("tl,hnl->thn", latent[:, :512].float(), w_v.float()).to(torch.bfloat16)
    cu = torch.tensor([0, 130, 430, 470], dtype=torch.int32, device=dev)
    out, lse = fm.dense_mla_prefill(q, k, v, cu, cu, softmax_scale=scale)

    # the latent rows go to the pages; a decode of the last position must give the same as the prefill
    per = 20
    table = torch.randperm(3 * per).to(torch.int32).view(3, per).to(dev)
    cache = torch.zeros(3 * per, page, 1, 576, dtype=torch.bfloat16, device=dev)
    for b, n in enumerate(lens):
        r = torch.arange(n, device=dev)
        cache[table[b].long()[r // page], r % page, 0] = latent[cu[b]:cu[b + 1]]
    seqlens = torch.tensor(lens, dtype=torch.int32, device=dev)
    last = (cu[1:] - 1).long()

    def absorbed(x):
        return torch.cat([torch.einsum("bhn,hnl->bhl", x[..., :128].float(), w_k.float()), x[..., 128:].float()], -1).to(torch.bfloat16)[:, None]
    meta, splits = fm.get_mla_metadata(seqlens, h, 1)
    q_abs = absorbed(q[last])
    o_abs, lse_dec = fm.flash_mla_with_kvcache(q_abs, cache, table, seqlens, 512, meta, splits, softmax_scale=scale, causal=True)
    o_dec = torch.einsum("bhl,hnl->bhn", o_abs[:, 0].float(), w_v.float())
    # k, v, absorbed q and the outputs are each rounded to bf16 on one of the two ways: a few 2^-8 of O(1) values
    assert (o_dec - out[last].float()).abs().max() < 4 * 2.0 ** -8 * float(v.abs().max())
    assert (lse_dec[:, :, 0] - lse[:, last].t()).abs().max() < 4 * 2.0 ** -8 * 10

    weights = fm.mla_cache_row_weights(q_abs, cache, table, seqlens, lse_dec, softmax_scale=scale, causal=True)
    assert (weights.sum(1) - h).abs().max() < 1e-2 * h
    rows, kept, sums = fm.mla_select_cache_rows(weights, seqlens, budget, recent)
    ref_rows, ref_kept, ref_sums = oracle.select_cache_rows(weights, seqlens, budget, recent)
    assert torch.equal(rows.cpu(), ref_rows) and torch.equal(kept.cpu(), ref_kept) and torch.equal(sums.cpu(), ref_sums)
    stay = [latent[cu[b]:cu[b + 1]][ref_rows[b, : int(ref_kept[b])].long().to(dev)] for b in range(3)]
    fm.mla_compact_cache(cache, table, rows, kept)

    meta, splits = fm.get_mla_metadata(kept, h, 1)
    o2, lse2 = fm.flash_mla_with_kvcache(q_abs, cache, table, kept, 512, meta, splits, softmax_scale=scale, causal=True)
    for b in range(3):
        s = q_abs[b, 0].double() @ stay[b].double().t() * scale
        ref = s.softmax(-1) @ stay[b][:, :512].double()
        assert oracle.cos_diff(o2[b, 0].float().cpu().numpy(), ref.float().cpu().numpy()) < 8e-5
        assert (lse2[b, :, 0].double() - s.logsumexp(-1)).abs().max() < 2e-3
    # the sums go on: the rows that stayed keep what they had
    acc = torch.zeros(3, per * page, device=dev)
    acc[:, :budget] = sums
    before = acc.clone()
    fm.mla_cache_row_weights(q_abs, cache, table, kept, lse2, softmax_scale=scale, causal=True, weights=acc)
    assert ((acc - before).sum(1) - h).abs().max() < 1e-2 * h


# ----------------------------------------------------------------------------- scales, plain C calls, several calls at once
@pytest.mark.parametrize("scale", [-0.05, 0.0, 1e-30, 1e-3, 0.5])
@pytest.mark.parametrize("s_q,h", [(1, 16), (1, 40), (1, 100), (3, 128)])
def test_weights_scales(fm, s_q, h, scale):
    kw, _ = paged([270, 65], s_q=s_q, h=h, seed=h)
    lse = lse_of(kw, True, scale)
    check_weights(fm.mla_cache_row_weights(**kw, softmax_lse=lse, softmax_scale=scale, causal=True), kw, lse, True, scale=scale)


@pytest.mark.parametrize("s_q,h", [(1, 64), (1, 128), (2, 128), (9, 60)])
def test_weights_of_rows_that_all_queries_look_at(fm, s_q, h):
    # Scores up to about 10.  The rounding of the products' sums must not leave a bias: 38 steps that cut off up to one unit
    # of 2^j 2^-23 (2^j times the scale <= 16) are 38^0.5 0.29 16 2^-23 = 3.4e-6 of one term where the steps' means cancel, but
    # 38 / 2 x 16 x 2^-23 = 3.6e-5 where they do not; over the columns the former averages out, the latter does not.  Held to
    # 2^-20 (3.4e-6 over 13 columns of equal weight; there are 64 and more) and 20 x 2^-22 for the exponents' rounding.
    kw, _ = paged([500, 130], s_q=s_q, h=h, seed=3)
    d = 576
    u = torch.randn(d, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    kw["q"] = (kw["q"].float() * 0.6 + 0.6 * u).to(torch.bfloat16)
    cache = kw["k_cache"].float()
    cache[:, ::7] = cache[:, ::7] * 0.6 + 0.5 * u
    kw["k_cache"] = cache.to(torch.bfloat16)
    lse = lse_of(kw, False)
    got = fm.mla_cache_row_weights(**kw, softmax_lse=lse).cpu().double()
    ref, _ = oracle.cache_row_weights(kw["q"], kw["k_cache"], kw["block_table"], kw["cache_seqlens"], lse, width=got.shape[1])
    for b, n in enumerate([500, 130]):
        heavy = torch.zeros(got.shape[1], dtype=torch.bool)
        heavy[:n] = ref[b, :n] > 0.2 * ref[b].max()
        off = ((got - ref)[b, heavy] / ref[b, heavy])
        assert heavy.sum() >= 10 and off.square().mean().sqrt() <= 2.0 ** -20 + 2.0 ** -22 * 20


def _weights_params(abi, kw, lse, w, workspace=None, workspace_bytes=0, causal=1):
    b, s_q, h, d = kw["q"].shape
    k, t = kw["k_cache"], kw["block_table"]
    return abi.SmlaRowWeightsParams(
        batch=b, seqlen_q=s_q, num_heads=h, causal=causal, head_dim=d, softmax_scale=d ** -0.5, q=kw["q"].data_ptr(), softmax_lse=lse.data_ptr(),
        k_cache=k.data_ptr(), k_block_stride=2 * k.stride(0), k_row_stride=2 * k.stride(1), num_blocks=k.shape[0], page_block_size=k.shape[1],
        max_blocks_per_seq=t.shape[1], block_table=t.data_ptr(), block_table_stride=t.stride(0), cache_seqlens=kw["cache_seqlens"].data_ptr(),
        weights=w.data_ptr(), weights_stride=w.stride(0), weights_width=w.shape[1], accumulate=0, workspace=workspace, workspace_bytes=workspace_bytes)


@pytest.mark.parametrize("s_q,h", [(2, 128), (33, 20)])
def test_weights_c_call_with_and_without_scratch(fm, s_q, h):
    from flash_mla import c_abi
    lib = c_abi.load()
    kw, _ = paged([700, 1, 0, 513], s_q=s_q, h=h, seed=11)
    lse = lse_of(kw, True)
    need, none = ctypes.c_size_t(0), ctypes.c_size_t(1)
    assert lib.smla_cache_row_weights_workspace(s_q, h, ctypes.byref(need)) == 0 and need.value > 0
    assert lib.smla_cache_row_weights_workspace(1, 128, ctypes.byref(none)) == 0 and none.value == 0
    scratch = torch.full((need.value + 16,), 255, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for given in ((None, 0), (scratch.data_ptr(), need.value - 1), (scratch.data_ptr(), need.value)):
        w = torch.full((4, kw["block_table"].shape[1] * 64), float("nan"), device="cuda")
        assert lib.smla_cache_row_weights(ctypes.byref(_weights_params(c_abi, kw, lse, w, *given)), stream) == 0
        check_weights(w, kw, lse, True, what=str(given))
    assert (scratch[need.value:] == 255).all()
    assert lib.smla_cache_row_weights(ctypes.byref(_weights_params(c_abi, kw, lse, w, scratch.data_ptr() + 4, need.value)), stream) == -2


def test_calls_on_several_streams_at_once(fm):
    calls = []
    for i, (s_q, h) in enumerate([(1, 16), (4, 128), (1, 64), (16, 32)]):
        kw, _ = paged([3000, 77, 1500], s_q=s_q, h=h, seed=20 + i)
        lse = torch.full((3, h, s_q), 7.5, device="cuda")

        def run(kw=kw, lse=lse):
            w = fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=True)
            rows, kept, sums = fm.mla_select_cache_rows(w, kw["cache_seqlens"], 600, 50)
            cache = kw["k_cache"].clone()
            fm.mla_compact_cache(cache, kw["block_table"], rows, kept)
            return w, rows, kept, sums, cache.view(torch.int16)
        calls.append(run)
    want = [run() for run in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for _ in range(3):
        for run, s in zip(calls, streams):
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for a, b in zip(out, want[i % len(calls)]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("in_place", [True, False])
def test_eviction_in_a_graph(fm, in_place):
    lens, budget = [400, 90, 260], 100
    kw, spare = paged(lens, s_q=2, h=128, seed=31, extra=0 if in_place else 6)
    out = None if in_place else spare.view(3, 2).cuda()
    start = kw["k_cache"].clone()
    lse = lse_of(kw, True)

    def step():
        w = fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=True)
        rows, kept, sums = fm.mla_select_cache_rows(w, kw["cache_seqlens"], budget, 30)
        fm.mla_compact_cache(kw["k_cache"], kw["block_table"], rows, kept, out_block_table=out)
        return rows, kept, sums
    want = [x.clone() for x in step()]
    moved = kw["k_cache"].clone()
    assert same_bytes(moved, oracle.compact_cache(start, kw["block_table"], want[0], want[1], out))
    torch.cuda.synchronize()
    kw["k_cache"].copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        kw["k_cache"].copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert same_bytes(kw["k_cache"], moved)


def test_pages_far_into_a_large_cache(fm):
    # element offsets past 2^31: 65600 pages of 64 rows (4.8 GB), of which the last hold the sequences
    nb, lens = 65600, [200, 70]
    kw, _ = paged(lens, h=16, seed=41)
    small, table = kw["k_cache"], kw["block_table"]
    big = torch.empty(nb, 64, 1, 576, dtype=torch.bfloat16, device="cuda")
    big[nb - small.shape[0]:] = small
    far = torch.where(table >= 0, table + (nb - small.shape[0]), table)
    lse = lse_of(kw, True)
    w = fm.mla_cache_row_weights(kw["q"], big, far, kw["cache_seqlens"], lse, causal=True)
    check_weights(w, kw, lse, True)
    rows, kept, _ = fm.mla_select_cache_rows(w, kw["cache_seqlens"], 64, 10)
    want = oracle.compact_cache(small, table, rows, kept)
    fm.mla_compact_cache(big, far, rows, kept)
    assert same_bytes(big[nb - small.shape[0]:], want)


@pytest.mark.parametrize("copied", [False, True])
def test_compact_into_the_first_pages_of_the_table(fm, copied):
    lens, budget = [700, 300, 90], 200
    kw, _ = paged(lens, h=1, d=64, page=16, seed=51)
    rows, kept = ascending(lens, budget, 7)
    table = kw["block_table"]
    if copied:                                                # a strided table that the binding has to copy
        table = torch.stack([table, table], 2)[:, :, 0]
    want = oracle.compact_cache(kw["k_cache"], table, rows, kept, table[:, :5])
    fm.mla_compact_cache(kw["k_cache"], table, rows, kept, out_block_table=table[:, :5])
    assert same_bytes(kw["k_cache"], want)


_FIRST_CALL = """
import torch, flash_mla as fm
dev = "cuda"
g = torch.Generator(device=dev).manual_seed(0)
q = torch.randn(1, 2, 128, 576, generator=g, device=dev).to(torch.bfloat16)
cache = torch.randn(8, 64, 1, 576, generator=g, device=dev).to(torch.bfloat16)
table = torch.arange(8, dtype=torch.int32, device=dev)[None]
lens = torch.full((1,), 500, dtype=torch.int32, device=dev)
lse = torch.full((1, 128, 2), 7.0, device=dev)
p = torch.randn(300, 4, 192, generator=g, device=dev).to(torch.bfloat16)
v = torch.randn(300, 4, 128, generator=g, device=dev).to(torch.bfloat16)
cu = torch.tensor([0, 300], dtype=torch.int32, device=dev)

def step():
    w = fm.mla_cache_row_weights(q, cache, table, lens, lse)
    w1 = fm.mla_cache_row_weights(q[:, :1, :16].contiguous(), cache, table, lens, lse[:, :16, :1].contiguous())
    rows, kept, sums = fm.mla_select_cache_rows(w, lens, 100, 10)
    moved = cache.clone()
    fm.mla_compact_cache(moved, table, rows, kept)
    out, z = fm.dense_mla_prefill(p, p, v, cu, cu)
    return w, w1, rows, kept, sums, moved.view(torch.int16), out, z

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(got, step()):
    assert torch.equal(a, b)
print("captured", fm.__name__)
"""


def test_the_first_call_of_a_process_may_be_a_captured_one(fm):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(fm.__file__)))
    run = subprocess.run([sys.executable, "-c", _FIRST_CALL], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


# ----------------------------------------------------------------------------- sums that go on through several evictions
@pytest.mark.parametrize("lens,width,budget,recent,columns", [([90, 300, 0, 5, 64], 300, 64, 16, 300), ([700, 699, 1], 700, 333, 333, 1000),
                                                              ([50, 9], 60, 500, 4, 60), ([9000, 8192], 9000, 700, 1, 20001), ([40], 40, 40, 0, 41)])
def test_select_into_sums_with_room_to_grow(fm, lens, width, budget, recent, columns):
    g = torch.Generator(device="cuda").manual_seed(width)
    w = torch.rand(len(lens), width, generator=g, device="cuda")
    w[w < 0.3] = 0
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    buf = torch.full((len(lens), columns + 7), float("nan"), device="cuda")
    place = buf[:, 3:3 + columns]
    rows, kept, sums = fm.mla_select_cache_rows(w, lens, budget, recent, kept_weights=place)
    want = oracle.select_cache_rows(w, lens, budget, recent, columns=columns)
    assert sums.data_ptr() == place.data_ptr()
    assert torch.equal(rows.cpu(), want[0]) and torch.equal(kept.cpu(), want[1]) and torch.equal(place.cpu(), want[2])
    assert torch.isnan(buf[:, :3]).all() and torch.isnan(buf[:, 3 + columns:]).all()


def test_select_into_the_other_half_of_a_buffer(fm):
    """Rows of the two that lie between one another do not overlap; the sums themselves, or a part of them, are refused."""
    buf = torch.rand(5, 2, 100, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    w = buf[:, 0].clone()
    lens = torch.tensor([100, 70, 30, 0, 99], dtype=torch.int32, device="cuda")
    want = oracle.select_cache_rows(w, lens, 40, 5, columns=100)
    fm.mla_select_cache_rows(buf[:, 0], lens, 40, 5, kept_weights=buf[:, 1])
    assert torch.equal(buf[:, 1].cpu(), want[2]) and torch.equal(buf[:, 0], w)
    for bad in (buf[:, 0], buf[:, 0, 50:], buf.view(5, 200)[:, 40:150]):
        with pytest.raises(ValueError):
            fm.mla_select_cache_rows(buf[:, 0], lens, 40, 5, kept_weights=bad)
    assert torch.equal(buf[:, 0], w)


@pytest.mark.parametrize("captured", [False, True])
def test_several_evictions_with_rows_appended_between(fm, captured):
    """What the guide's loop does: rows are appended, a decode step, its weights added to the sums, and an eviction, four times.
    Each row has a number; the host follows which numbers a sequence has and what weights each has had."""
    h, page, per, budget, recent, fresh, rounds = 4, 16, 20, 64, 16, 40, 4
    g = torch.Generator(device="cuda").manual_seed(7)
    lens = [200, 30, 130]
    b = len(lens)
    table = torch.randperm(b * per, generator=torch.Generator().manual_seed(8)).to(torch.int32).view(b, per).cuda()
    cache = torch.zeros(b * per, page, 1, 576, dtype=torch.bfloat16, device="cuda")
    rows_of = torch.randn(b, 200 + fresh * rounds, 576, generator=g, device="cuda").to(torch.bfloat16)     # by number
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def put(i, first, numbers):
        r = torch.arange(first, first + len(numbers), device="cuda")
        cache[table[i].long()[r // page], r % page, 0] = rows_of[i, numbers]
    numbers = [list(range(n)) for n in lens]
    for i in range(b):
        put(i, 0, numbers[i])
    sums = [torch.zeros(b, per * page, device="cuda"), torch.full((b, per * page), float("nan"), device="cuda")]
    had = [dict.fromkeys(x, 0.0) for x in numbers]
    q = torch.randn(b, 1, h, 576, generator=g, device="cuda").to(torch.bfloat16)
    meta, splits = fm.get_mla_metadata(seqlens, h, 1)

    def step(now, other):
        _, lse = fm.flash_mla_with_kvcache(q, cache, table, seqlens, 512, meta, splits, causal=True)
        fm.mla_cache_row_weights(q, cache, table, seqlens, lse, causal=True, weights=now)
        rows, kept, _ = fm.mla_select_cache_rows(now, seqlens, budget, recent, kept_weights=other)
        fm.mla_compact_cache(cache, table, rows, kept)
        return lse, rows, kept
    graphs = []
    if captured:
        keep = cache.clone()
        step(sums[0], sums[1])
        sums[0].zero_()
        cache.copy_(keep)
        torch.cuda.synchronize()
        for k in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                graphs.append((graph, step(sums[k], sums[1 - k])))
    for turn in range(rounds):
        now, other = sums[turn & 1], sums[1 - (turn & 1)]
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        if turn:
            for i in range(b):
                new = list(range(200 + fresh * turn, 200 + fresh * (turn + 1)))
                put(i, len(numbers[i]), new)
                numbers[i] += new
                had[i].update(dict.fromkeys(new, 0.0))
            seqlens.copy_(torch.tensor([len(x) for x in numbers], dtype=torch.int32))
        if captured:
            graphs[turn & 1][0].replay()
            lse, rows, kept = graphs[turn & 1][1]
        else:
            lse, rows, kept = step(now, other)
        torch.cuda.synchronize()
        assert kept.tolist() == [min(len(x), budget) for x in numbers]
        for i in range(b):
            s = rows_of[i, numbers[i]].double() @ q[i, 0].double().t() * 576 ** -0.5
            for number, x in zip(numbers[i], torch.exp(s - lse[i, :, 0].double()).sum(1).tolist()):
                had[i][number] += x
            total = torch.tensor([had[i][x] for x in numbers[i]], dtype=torch.float64)
            # d 2^-23 scale sum |q k| and the like, as in check_weights: far below 1e-3 of a weight, four times
            assert ((now[i, : total.numel()].cpu().double() - total).abs() <= 1e-3 * total + 1e-9).all()
            ids, _, vals = oracle.select_cache_rows(now[i:i + 1], seqlens[i:i + 1], budget, recent, columns=per * page)
            m = int(kept[i])
            assert rows[i, :m].tolist() == ids[0, :m].tolist() and torch.equal(other[i].cpu(), vals[0])
            before = len(numbers[i])
            assert rows[i, :m].tolist()[-min(recent, m):] == list(range(before - min(recent, m), before))      # the newest are there
            numbers[i] = [numbers[i][r] for r in rows[i, :m].tolist()]
            r = torch.arange(m, device="cuda")
            assert torch.equal(cache[table[i].long()[r // page], r % page, 0], rows_of[i, numbers[i]])
        seqlens.copy_(kept)


_MOST = 2 ** 31 - 1


@pytest.mark.parametrize("width,budget,recent", [(100, _MOST, 0), (_MOST, _MOST, 3), (_MOST, 5000, 77), (_MOST, _MOST - 1, _MOST - 2)])
def test_select_sizes_up_to_the_largest_integer(fm, width, budget, recent):
    """"Keep all" said as the largest budget; the longest row of weights; the most recent rows.  Up to 27 GB."""
    w = torch.zeros(1, width, device="cuda")
    heavy = torch.arange(3, width - 1, max(1, width // 40), device="cuda")[:37]
    w[0, heavy] = torch.rand(heavy.numel(), device="cuda") + 1.0
    lens = torch.tensor([width], dtype=torch.int32, device="cuda")
    rows, kept, sums = fm.mla_select_cache_rows(w, lens, budget, recent)
    stay, old = min(width, budget), width - recent
    assert int(kept) == stay and rows.shape == sums.shape == (1, budget)
    if width <= budget:
        front = torch.arange(min(stay, 10 ** 6), device="cuda")
    else:                                                     # heavy ones first, then the lowest of the zeros
        top = heavy[heavy < old]
        lowest = torch.arange(min(old, budget), device="cuda")
        lowest = lowest[~torch.isin(lowest, top)]
        pick = torch.cat([top[torch.sort(w[0, top], descending=True, stable=True).indices], lowest])[: budget - recent]
        front = pick.sort().values
        assert rows[0, budget - recent] == old and rows[0, -1] == width - 1
        step = rows[0, budget - recent:]
        for at in range(0, recent, 1 << 28):
            piece = step[at:at + (1 << 28)]
            assert torch.equal(piece, torch.arange(old + at, old + at + piece.numel(), dtype=torch.int32, device="cuda"))
    assert torch.equal(rows[0, : front.numel()].long(), front) and torch.equal(sums[0, : front.numel()], w[0, front])
    if width == budget:
        assert torch.equal(sums, w) and int(rows[0, -1]) == width - 1
    for at in range(stay, budget, 1 << 28):
        assert (rows[0, at:at + (1 << 28)] == -1).all() and (sums[0, at:at + (1 << 28)] == 0).all()


@pytest.mark.parametrize("in_place", [True, False])
def test_compact_with_the_largest_budget(fm, in_place):
    """The rows of a selection that was told to keep all, and a count that says so too: what the table has places for is moved."""
    kw, spare = paged([75], h=1, d=64, page=16, seed=61, extra=5)
    out = None if in_place else spare.view(1, 5).cuda()
    rows = torch.full((1, _MOST), -1, dtype=torch.int32, device="cuda")
    rows[0, :60] = torch.arange(15, 75, device="cuda")
    kept = torch.tensor([_MOST], dtype=torch.int32, device="cuda")
    want = oracle.compact_cache(kw["k_cache"], kw["block_table"], rows[:, :96].cpu(), torch.tensor([96]), out)
    fm.mla_compact_cache(kw["k_cache"], kw["block_table"], rows, kept, out_block_table=out)
    assert same_bytes(kw["k_cache"], want)


def _same_pages(table, spare, per, kind):
    """Targets that name the source's pages in their own columns: all of them, the first or the last half, those of some sequences."""
    out = spare.view(table.shape[0], per).clone() if kind != "all" else table[:, :per].cpu().clone()
    own = table[:, :per].cpu()
    if kind == "first":
        out[:, : per // 2] = own[:, : per // 2]
    elif kind == "last":
        out[:, per // 2:] = own[:, per // 2:]
    elif kind == "some":
        out[::2] = own[::2]
    return out.cuda()


@pytest.mark.parametrize("kind", ["all", "first", "last", "some"])
@pytest.mark.parametrize("page,d,lens,budget", [(16, 64, [20000, 9000, 11000], 8000), (1, 40, [3000, 2000, 2500], 1111), (100, 8, [700, 2000, 1000], 600),
                                                (64, 576, [9000, 5000, 7001], 4096)])
def test_compact_to_a_copy_of_the_own_pages(fm, kind, page, d, lens, budget):
    per = (budget + page - 1) // page
    kw, spare = paged(lens, h=1, d=d, page=page, seed=page, extra=per * len(lens))
    rows, kept = ascending(lens, budget, page)
    out = _same_pages(kw["block_table"], spare, per, kind)
    want = oracle.compact_cache(kw["k_cache"], kw["block_table"], rows, kept, out)
    start = kw["k_cache"].clone()
    for _ in range(5):
        kw["k_cache"].copy_(start)
        fm.mla_compact_cache(kw["k_cache"], kw["block_table"], rows, kept, out_block_table=out)
        assert same_bytes(kw["k_cache"], want)


def test_compact_to_a_copy_of_a_table_with_other_strides(fm):
    lens, budget = [5000, 3000], 2000
    kw, _ = paged(lens, h=1, d=64, page=16, seed=71)
    rows, kept = ascending(lens, budget, 72)
    want = oracle.compact_cache(kw["k_cache"], kw["block_table"], rows, kept)
    fm.mla_compact_cache(kw["k_cache"], kw["block_table"], rows, kept, out_block_table=kw["block_table"].t().contiguous().t())
    assert same_bytes(kw["k_cache"], want)


@pytest.mark.parametrize("in_place", [True, False])
def test_compact_more_sequences_than_a_grid_counts_in_one_dimension(fm, in_place):
    n, page = 140001, 8
    g = torch.Generator(device="cuda").manual_seed(81)
    cache = torch.randn(2 * n, page, 1, 8, generator=g, device="cuda").to(torch.bfloat16)
    table = torch.randperm(2 * n, generator=g, device="cuda").to(torch.int32)
    table, out = table[:n, None], None if in_place else table[n:, None]
    rows = torch.tensor([1, 4, 5], dtype=torch.int32, device="cuda").repeat(n, 1)
    kept = torch.randint(0, 4, (n,), generator=g, device="cuda").to(torch.int32)
    want = cache.clone()
    for j in range(3):
        live = kept > j
        want[(table if in_place else out)[live, 0].long(), j] = cache[table[live, 0].long(), (1, 4, 5)[j]]
    fm.mla_compact_cache(cache, table, rows, kept, out_block_table=out)
    assert same_bytes(cache, want)


# ----------------------------------------------------------------------------- the columns beside the sums
@pytest.mark.parametrize("s_q,h", [(1, 16), (2, 40), (5, 60), (33, 20)])
@pytest.mark.parametrize("width", [1, 150, 256, 513, 1100, 5000])
def test_weights_touch_nothing_beside_them(fm, s_q, h, width):
    """Added to, and written with zeros behind the rows, inside a wider buffer: its other columns keep their bits."""
    from flash_mla import c_abi
    lib = c_abi.load()
    kw, _ = paged([700, 0, 130, 1], s_q=s_q, h=h, seed=width)
    lse = lse_of(kw, True)
    buf = torch.rand(4, width + 13, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    before, w = buf.clone(), buf[:, 5:5 + width]
    got = fm.mla_cache_row_weights(**kw, softmax_lse=lse, causal=True, weights=w)
    assert torch.equal(buf[:, :5], before[:, :5]) and torch.equal(buf[:, 5 + width:], before[:, 5 + width:])
    check_weights(got, kw, lse, True, weights=before[:, 5:5 + width])
    need = ctypes.c_size_t(0)
    assert lib.smla_cache_row_weights_workspace(s_q, h, ctypes.byref(need)) == 0
    scratch = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    for given in ((None, 0), (scratch.data_ptr(), need.value)):
        buf.copy_(before)
        assert lib.smla_cache_row_weights(ctypes.byref(_weights_params(c_abi, kw, lse, w, *given)), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(buf[:, :5], before[:, :5]) and torch.equal(buf[:, 5 + width:], before[:, 5 + width:])
        check_weights(w, kw, lse, True)
        for b, n in enumerate((700, 0, 130, 1)):
            assert (w[b, n:] == 0).all()
