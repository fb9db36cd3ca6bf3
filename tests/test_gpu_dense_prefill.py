"""GPU tests of dense MLA prefill against the float64 oracle.

Tolerances, from the arithmetic (u = eps / 2 of the type: 2^-8 bf16, 2^-11 fp16):
* the weights are rounded to the type before the second product and the output once at the end:
  u * sum p |v| + u * |out|;
* a score is a sum of d exact products in fp32, off by at most d 2^-23 scale sum |q k| (=: ds) however the sum is
  ordered, and its scaling, the difference to the running maximum and the exponential add a few 2^-22 of the
  exponent's size, at most 2 scale sum |q k|: a weight is off by the factor 1 + ds + 2^-20 scale sum |q k| + 2^-21, a
  quotient of such sums by twice that, relative to sum p |v|;
* sums of n terms in fp32: n 2^-23 sum p |v|;
* fp16 weights below 2^-14 of the row's largest are subnormal, off by 2^-25 each (the largest is at least 1):
  n 2^-25 max |v|.
The lse is off by the weights' factor, n 2^-23 and the rounding of its own size, 2^-22 |lse|.
"""
import ctypes
import math

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


def cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def inputs(q_lens, k_lens=None, h=2, hk=None, d=192, dt=torch.bfloat16, seed=0, gain=1.0):
    k_lens = q_lens if k_lens is None else k_lens
    hk = h if hk is None else hk
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")
    return ((gain * r(sum(q_lens), h, d)).to(dt), r(sum(k_lens), hk, d).to(dt), r(sum(k_lens), hk, 128).to(dt), cu(q_lens), cu(k_lens))


def check(got, args, causal=True, scale=None, what=""):
    q, k, v, cu_q, cu_k = args
    out, lse = got
    ro, rl, mag, size = oracle.dense_mla_prefill(q, k, v, cu_q, cu_k, scale=scale, causal=causal)
    assert out.dtype == q.dtype and out.shape == ro.shape and lse.dtype == torch.float32 and lse.shape == rl.shape
    u = torch.finfo(q.dtype).eps / 2
    n, d = (int((cu_k[1:] - cu_k[:-1]).max()) if cu_k.numel() > 1 else 0), q.shape[2]
    factor = d * 2.0 ** -23 * size + 2.0 ** -20 * size + 2.0 ** -21
    tol = (u + 2 * factor.T[:, :, None] + n * 2.0 ** -23) * mag + u * ro.abs()
    if q.dtype == torch.float16 and v.numel():
        tol = tol + n * 2.0 ** -25 * float(v.abs().max())
    o = out.detach().cpu().double()
    assert torch.isfinite(o).all(), f"{what}: non-finite output"
    bad = (o - ro).abs() - tol * 1.0001 - 1e-30
    assert bad.max() <= 0, f"{what}: out off by {float((o - ro).abs().max()):.3e}, {float(bad.max()):.3e} over the bound at {torch.nonzero(bad > 0)[:3].tolist()}"
    z = lse.detach().cpu().double()
    seen = torch.isfinite(rl)
    assert ((z == float("-inf")) == ~seen).all(), f"{what}: lse finiteness"
    tl = factor + n * 2.0 ** -23 + 2.0 ** -22 * rl.abs() + 1e-7
    assert ((z - rl).abs()[seen] <= tl[seen]).all(), f"{what}: lse off by {float((z - rl).abs()[seen].max()):.3e}"


@pytest.mark.parametrize("d", [192, 128])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[1], [2], [16], [17], [127], [128], [129], [255], [256], [257], [300], [513], [1, 1, 3], [130, 5, 64, 200]])
def test_lengths(fm, d, dt, lens):
    a = inputs(lens, d=d, dt=dt, seed=sum(lens))
    check(fm.dense_mla_prefill(*a), a, what=f"{lens}")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,k_lens", [([1], [1000]), ([5, 128], [300, 129]), ([130, 1], [128, 640]), ([40], [7]), ([300, 3], [64, 1]),
                                           ([0, 7, 0, 33], [5, 7, 0, 0]), ([513], [1025]), ([200], [456])])
def test_keys_before_and_fewer_keys_than_queries(fm, causal, q_lens, k_lens):
    """A prefix in front of the queries, rows that the mask leaves empty, sequences without queries or without keys."""
    a = inputs(q_lens, k_lens, h=3, seed=1)
    check(fm.dense_mla_prefill(*a, causal=causal), a, causal=causal, what=f"{q_lens} {k_lens}")


@pytest.mark.parametrize("h,hk", [(1, 1), (8, 1), (8, 2), (6, 2), (5, 5), (40, 8)])
def test_grouped_heads(fm, h, hk):
    a = inputs([150, 33], h=h, hk=hk, d=128, seed=h)
    check(fm.dense_mla_prefill(*a), a, what=f"{h}/{hk}")


def test_long_prompt(fm):
    a = inputs([2500, 1100], h=2, seed=3)
    check(fm.dense_mla_prefill(*a), a)


def test_many_short_prompts(fm):
    lens = [(7 * i) % 40 for i in range(300)]
    a = inputs(lens, h=4, hk=2, seed=4)
    check(fm.dense_mla_prefill(*a), a)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_scores_that_climb(fm, dt):
    """Each key scores higher than the one before: the running maximum moves all the time, and the last keys weigh all."""
    q, k, v, cq, ck = inputs([700], h=2, dt=dt, seed=5)
    q[:] = 1.0
    k[:] = (torch.arange(700, device="cuda") / 700.0 * 4)[:, None, None].to(dt) - 2
    check(fm.dense_mla_prefill(q, k, v, cq, ck), (q, k, v, cq, ck))
    k = k.flip(0).contiguous()
    check(fm.dense_mla_prefill(q, k, v, cq, ck), (q, k, v, cq, ck))


def test_large_scores_and_scales(fm):
    a = inputs([400], h=2, seed=6, gain=12.0)
    check(fm.dense_mla_prefill(*a), a)
    check(fm.dense_mla_prefill(*a, softmax_scale=0.001), a, scale=0.001)
    check(fm.dense_mla_prefill(*a, softmax_scale=-0.05), a, scale=-0.05)
    check(fm.dense_mla_prefill(*a, softmax_scale=0.0), a, scale=0.0)


def test_strides(fm):
    """Views of wider buffers, transposed heads, kv heads broadcast from one, rows that start off 16 bytes."""
    g = torch.Generator(device="cuda").manual_seed(7)
    lens = [130, 70]
    big = torch.randn(200, 3, 4 * 192 + 64, generator=g, device="cuda").to(torch.bfloat16)
    q = big[:, 1, :768].view(200, 4, 192)
    kv = torch.randn(4, 200, 320, generator=g, device="cuda").to(torch.bfloat16).transpose(0, 1)
    k, v = kv[..., :192], kv[..., 192:]
    a = (q, k, v, cu(lens), cu(lens))
    check(fm.dense_mla_prefill(*a), a, what="views")
    one = k[:, :1].expand(200, 4, 192)
    a = (q, one, v, cu(lens), cu(lens))
    check(fm.dense_mla_prefill(*a), a, what="broadcast")
    odd = torch.randn(200, 4, 193, generator=g, device="cuda").to(torch.bfloat16)[..., 1:]
    a = (odd, k, v, cu(lens), cu(lens))
    check(fm.dense_mla_prefill(*a), a, what="odd start")


def test_rows_of_other_sequences_do_not_leak(fm):
    """NaN and infinity in a neighbour's rows, and in rows behind the last sequence, stay there; the queries behind the
    last sequence are left alone by the C entry."""
    lens = [100, 60, 140]
    q, k, v, cq, _ = inputs(lens + [50], h=2, seed=8)
    cq = cq[:4].contiguous()
    clean = fm.dense_mla_prefill(q, k, v, cq, cq)
    bad = [x.clone() for x in (q, k, v)]
    for x in bad:
        x[100:160] = float("nan")
        x[300:] = float("inf")
    out, lse = fm.dense_mla_prefill(*bad, cq, cq)
    keep = torch.cat([torch.arange(0, 100), torch.arange(160, 300)]).cuda()
    assert torch.equal(out[keep], clean[0][keep]) and torch.equal(lse[:, keep], clean[1][:, keep])
    assert torch.isnan(out[100:160]).all()


def test_rows_behind_the_last_sequence_are_not_written(fm):
    from flash_mla import c_abi
    lib = c_abi.load()
    q, k, v, cq, _ = inputs([90, 40, 70], h=2, seed=9)
    cq = cq[:3].contiguous()
    out = torch.full((200, 2, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((2, 200), 7.0, device="cuda")
    p = c_abi.prefill_params(q, k, v, cq, cq, out, lse)
    c_abi.check(lib.smla_dense_mla_prefill(ctypes.byref(p), torch.cuda.current_stream().cuda_stream))
    ref, rl = fm.dense_mla_prefill(q, k, v, cq, cq)
    assert torch.equal(out[:130], ref[:130]) and torch.equal(lse[:, :130], rl[:, :130])
    assert (out[130:] == 7).all() and (lse[:, 130:] == 7).all()
    p.softmax_lse = None                                     # the lse may be left out
    out.zero_()
    c_abi.check(lib.smla_dense_mla_prefill(ctypes.byref(p), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[:130], ref[:130])


def test_offsets_out_of_range_are_clamped(fm):
    """Offsets past the totals or running backwards touch nothing outside; the sequences before them are right."""
    q, k, v, _, _ = inputs([120], h=2, seed=10)
    good = cu([50])
    ref = fm.dense_mla_prefill(q, k, v, good, good)
    bad = torch.tensor([0, 50, 4000], dtype=torch.int32, device="cuda")
    out, _ = fm.dense_mla_prefill(q, k, v, bad, bad)
    assert torch.equal(out[:50], ref[0][:50])
    back = torch.tensor([0, 50, 20], dtype=torch.int32, device="cuda")
    out, _ = fm.dense_mla_prefill(q, k, v, back, back)
    assert torch.equal(out[:50], ref[0][:50])


def test_empty_calls(fm):
    q, k, v, _, _ = inputs([4], h=2, seed=11)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = fm.dense_mla_prefill(q[:0], k, v, zero, zero)
    assert out.shape == (0, 2, 128) and lse.shape == (2, 0)
    a = (q, k[:0], v[:0], cu([4]), cu([0]))
    check(fm.dense_mla_prefill(*a), a)
    check(fm.dense_mla_prefill(*a, causal=False), a, causal=False)


def test_same_bits_twice_and_on_another_stream(fm):
    a = inputs([600, 333, 20], h=4, seed=12)
    one = fm.dense_mla_prefill(*a)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        two = fm.dense_mla_prefill(*a)
    with torch.cuda.stream(t):
        three = fm.dense_mla_prefill(*a)
    torch.cuda.synchronize()
    for x in (two, three):
        assert torch.equal(one[0], x[0]) and torch.equal(one[1], x[1])


def test_graph_replays_follow_the_buffers(fm):
    a = inputs([200, 100], h=2, seed=13)
    fm.dense_mla_prefill(*a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fm.dense_mla_prefill(*a)
    b = inputs([37, 263], h=2, seed=14)
    for dst, src in zip(a, b):
        dst.copy_(src)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    check(got, a)


def test_random_shapes(fm):
    import random
    rng = random.Random(15)
    for i in range(25):
        ql = [rng.choice([0, 1, 5, 64, 100, 128, 200, 256, 300, 390]) for _ in range(rng.randint(1, 5))]
        kl = [x if rng.random() < 0.6 else rng.choice([0, 1, 90, 128, 250, 513]) for x in ql]
        if sum(ql) == 0:
            continue
        hk = rng.choice([1, 2, 3])
        a = inputs(ql, kl, h=hk * rng.choice([1, 2, 3]), hk=hk, d=rng.choice([128, 192]), dt=rng.choice([torch.bfloat16, torch.float16]), seed=i)
        causal = rng.random() < 0.7
        check(fm.dense_mla_prefill(*a, causal=causal), a, causal=causal, what=f"{i}: {ql} {kl} causal={causal}")


def test_offsets_past_2_31_elements(fm):
    # 66000 tokens of 256 x 192 (6.5 GB) and 256 x 128 elements; the only sequence lies at the end
    n, h, m = 66000, 256, 150
    a = inputs([m], h=h, hk=2, seed=16)
    q = torch.empty(n, h, 192, dtype=torch.bfloat16, device="cuda")
    q[n - m:] = a[0]
    k, v = (torch.cat([torch.full((n - m,) + x.shape[1:], float("nan"), dtype=x.dtype, device="cuda"), x]) for x in a[1:3])
    at = torch.tensor([n - m, n], dtype=torch.int32, device="cuda")
    out, lse = fm.dense_mla_prefill(q, k, v, at, at)
    check((out[n - m:], lse[:, n - m:]), a)


def test_many_prompts_of_mixed_lengths(fm):
    import random
    rng = random.Random(17)
    ql = [rng.choice([0, 1, 2, 30, 130, 257, 600]) for _ in range(75)]
    kl = [x + rng.choice([0, 0, 1, 200, 700]) for x in ql]
    a = inputs(ql, kl, h=3, seed=18)
    check(fm.dense_mla_prefill(*a), a)


@pytest.mark.parametrize("d", [192, 128])
@pytest.mark.parametrize("q_lens,k_lens", [([700, 1, 390, 1100, 129], None), ([40, 300, 2], [2000, 1500, 1411]), ([30] * 60, [385] * 60)])
def test_references_that_move_at_every_tile(fm, d, q_lens, k_lens):
    """Each block of 128 keys scores about 2^9 and more above the one before, in items of one to sixteen blocks, so that the output is
    moved to a new reference at every tile of every item, and items follow one another on the same pair of CTAs.  The same bits twice."""
    a = inputs(q_lens, k_lens, h=24, hk=12, d=d, seed=d + len(q_lens), gain=0.25)
    q, k, _, _, cu_k = a
    at = torch.arange(k.shape[0], device="cuda") - cu_k[:-1].long().repeat_interleave((cu_k[1:] - cu_k[:-1]).long())
    # scores climb by 0.05 a key, 6.4 = 9.2 ln 2 a block, in one product (bf16 rounds the largest, 100, by a quarter)
    q[:, :, 0] = d ** 0.5
    k[:, :, 0] = (0.05 * at).to(k.dtype)[:, None]
    one = fm.dense_mla_prefill(*a)
    check(one, a)
    for _ in range(20):
        two = fm.dense_mla_prefill(*a)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("below", [17.0, 18.5, 20.0])
def test_many_keys_far_below_the_largest(fm, dt, below):
    """One key outweighs the 300000 others, which together are up to 1 % of the row, each of them near or below the smallest fp16 number.  With
    v = 0 for the one and 1 for the others the output is their share.  Off it, relative: the roundings of a weight and of the output, u
    each (all weights are alike, so nothing averages out); an fp16 weight of 2^7 e^-below is subnormal, 2^-25 at most, so 2^-32
    e^below; the sum of the weights has eight partial sums of n / 8 terms, each rounded to 2^-24 of the sum, the product
    n / 16 steps cut off at 2^-23: n 2^-26 together; the exponent, 32 x 2^-23, and the exponential less than 2^-17."""
    n, d = 300000, 128
    q = torch.zeros(1, 1, d, dtype=dt, device="cuda")
    k = torch.zeros(n, 1, d, dtype=dt, device="cuda")
    v = torch.ones(n, 1, 128, dtype=dt, device="cuda")
    q[..., 0], k[12345, 0, 0], v[12345] = 1.0, below, 0.0
    out, lse = fm.dense_mla_prefill(q, k, v, cu([1]), cu([n]), softmax_scale=1.0, causal=False)
    rest = (n - 1) * math.exp(-below)
    share = rest / (1 + rest)
    tol = 2 * torch.finfo(dt).eps / 2 + n * 2.0 ** -26 + 2.0 ** -17 + (2.0 ** -32 * math.exp(below) if dt == torch.float16 else 0.0)
    assert (out.double() - share).abs().max() <= tol * share, f"{float(out.double().mean()):.4e} for {share:.4e}"
    assert (lse.double() - (below + math.log1p(rest))).abs().max() <= n * 2.0 ** -27 + 2.0 ** -17
