"""CPU tests of dense MLA prefill and cache eviction: what the Python wrappers and the C entry points refuse (before
any CUDA call), the C structs against the compiler, and the oracles against independent formulations."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMLA_OK, SMLA_EINVAL, SMLA_EALIGN, SMLA_ETOOBIG = 0, -1, -2, -5


@pytest.fixture(scope="module")
def fm():
    import flash_mla
    return flash_mla


@pytest.fixture(scope="module")
def abi():
    from flash_mla import c_abi
    c_abi.load()
    return c_abi


def test_struct_layout_matches_c_compiler(abi, tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    checks = [("smla_prefill_params_t", abi.SmlaPrefillParams), ("smla_row_weights_params_t", abi.SmlaRowWeightsParams),
              ("smla_compact_params_t", abi.SmlaCompactParams)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "sparse_mla_b200.h"', 'int main(void){']
    want = []
    for cname, cls in checks:
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(cls))
        for fname, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cname}, {fname}));')
            want.append(getattr(cls, fname).offset)
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


# ----------------------------------------------------------------------------- Python refusals
def _qkv(tq=4, tk=4, h=4, hk=2, d=192, dv=128, dt=torch.bfloat16):
    return torch.zeros(tq, h, d, dtype=dt), torch.zeros(tk, hk, d, dtype=dt), torch.zeros(tk, hk, dv, dtype=dt)


CU = torch.tensor([0, 4], dtype=torch.int32)


@pytest.mark.parametrize("change", [
    dict(d=96), dict(dv=64), dict(h=3), dict(dt=torch.float32), dict(dt=torch.float64), dict(d=576),
])
def test_prefill_refuses_shapes_and_types(fm, change):
    q, k, v = _qkv(**change)
    with pytest.raises(ValueError):
        fm.dense_mla_prefill(q, k, v, CU, CU)


def test_prefill_refuses_mixed_types_tokens_and_offsets(fm):
    q, k, v = _qkv()
    with pytest.raises(ValueError):
        fm.dense_mla_prefill(q, k.half(), v, CU, CU)
    with pytest.raises(ValueError):
        fm.dense_mla_prefill(q, k[:3], v, CU, CU)
    with pytest.raises(ValueError):
        fm.dense_mla_prefill(q[None], k, v, CU, CU)
    with pytest.raises(ValueError):
        fm.dense_mla_prefill(q, k, v, CU.long(), CU)
    with pytest.raises(ValueError):
        fm.dense_mla_prefill(q, k, v, CU, torch.tensor([0, 2, 4], dtype=torch.int32))
    with pytest.raises(ValueError):
        fm.dense_mla_prefill(q, k, v, CU[:0], CU[:0])


def test_cpu_tensors_are_refused(fm):
    """The ops are registered for CUDA only."""
    q, k, v = _qkv()
    with pytest.raises((RuntimeError, NotImplementedError)):
        fm.dense_mla_prefill(q, k, v, CU, CU)
    a = _weights_args()
    with pytest.raises((RuntimeError, NotImplementedError)):
        fm.mla_cache_row_weights(**a)
    with pytest.raises((RuntimeError, NotImplementedError)):
        fm.mla_select_cache_rows(torch.zeros(1, 4), torch.zeros(1, dtype=torch.int32), 2)
    with pytest.raises((RuntimeError, NotImplementedError)):
        fm.mla_compact_cache(a["k_cache"], a["block_table"], torch.zeros(2, 3, dtype=torch.int32), a["cache_seqlens"])


def _weights_args(b=2, sq=1, h=4, d=576, page=16):
    return dict(q=torch.zeros(b, sq, h, d, dtype=torch.bfloat16), k_cache=torch.zeros(5, page, 1, d, dtype=torch.bfloat16),
                block_table=torch.zeros(b, 2, dtype=torch.int32), cache_seqlens=torch.zeros(b, dtype=torch.int32),
                softmax_lse=torch.zeros(b, h, sq))


@pytest.mark.parametrize("key,value", [
    ("q", torch.zeros(2, 1, 4, 576)), ("q", torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16)),
    ("k_cache", torch.zeros(5, 16, 1, 512, dtype=torch.bfloat16)), ("k_cache", torch.zeros(5, 16, 2, 576, dtype=torch.bfloat16)),
    ("k_cache", torch.zeros(5, 12, 1, 576, dtype=torch.bfloat16)), ("k_cache", torch.zeros(5, 16, 1, 576)),
    ("block_table", torch.zeros(3, 2, dtype=torch.int32)), ("block_table", torch.zeros(2, 2)),
    ("cache_seqlens", torch.zeros(2)), ("cache_seqlens", torch.zeros(3, dtype=torch.int32)),
    ("softmax_lse", torch.zeros(2, 1, 4)), ("softmax_lse", torch.zeros(2, 4, 1, dtype=torch.float64)),
    ("weights", torch.zeros(3, 32)), ("weights", torch.zeros(2, 32, dtype=torch.float16)),
])
def test_row_weights_refuse(fm, key, value):
    a = _weights_args()
    a[key] = value
    with pytest.raises(ValueError):
        fm.mla_cache_row_weights(**a)


@pytest.mark.parametrize("budget,recent", [(0, 0), (-1, 0), (4, 5), (4, -1)])
def test_select_refuses_budgets(fm, budget, recent):
    with pytest.raises(ValueError):
        fm.mla_select_cache_rows(torch.zeros(1, 9), torch.zeros(1, dtype=torch.int32), budget, recent)


def test_select_and_compact_refuse_types(fm):
    with pytest.raises(ValueError):
        fm.mla_select_cache_rows(torch.zeros(1, 9).half(), torch.zeros(1, dtype=torch.int32), 2)
    with pytest.raises(ValueError):
        fm.mla_select_cache_rows(torch.zeros(1, 9), torch.zeros(2, dtype=torch.int32), 2)
    a = _weights_args()
    rows, kept = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(rows=rows.long()), dict(kept=kept.long()), dict(k_cache=a["k_cache"].float()),
                dict(block_table=a["block_table"][:1]), dict(out_block_table=torch.zeros(1, 2, dtype=torch.int32)),
                dict(k_cache=torch.zeros(5, 16, 1, 12, dtype=torch.bfloat16))):
        args = dict(k_cache=a["k_cache"], block_table=a["block_table"], rows=rows, kept=kept)
        args.update(bad)
        with pytest.raises(ValueError):
            fm.mla_compact_cache(**args)


# ----------------------------------------------------------------------------- C refusals
FAKE = 0x100000


def _prefill_params(abi, **kw):
    p = abi.SmlaPrefillParams()
    vals = dict(batch=1, num_heads=4, num_kv_heads=2, head_dim=192, head_dim_v=128, dtype=0, causal=1, softmax_scale=0.1, total_q=8,
                total_k=8, q=FAKE, k=FAKE, v=FAKE, q_token_stride=768, q_head_stride=192, k_token_stride=384, k_head_stride=192,
                v_token_stride=256, v_head_stride=128, out=FAKE, out_token_stride=512, out_head_stride=128, softmax_lse=FAKE,
                lse_head_stride=8, cu_seqlens_q=FAKE, cu_seqlens_k=FAKE)
    vals.update(kw)
    for k, v in vals.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), SMLA_EINVAL), (dict(num_heads=3), SMLA_EINVAL), (dict(num_kv_heads=0), SMLA_EINVAL), (dict(head_dim=64), SMLA_EINVAL),
    (dict(head_dim_v=192), SMLA_EINVAL), (dict(dtype=2), SMLA_EINVAL), (dict(softmax_scale=float("nan")), SMLA_EINVAL),
    (dict(q=0), SMLA_EINVAL), (dict(k=0), SMLA_EINVAL), (dict(v=0), SMLA_EINVAL), (dict(out=0), SMLA_EINVAL), (dict(cu_seqlens_q=0), SMLA_EINVAL),
    (dict(cu_seqlens_k=0), SMLA_EINVAL), (dict(q=FAKE + 2), SMLA_EALIGN), (dict(k_head_stride=100), SMLA_EALIGN),
    (dict(v=FAKE + 8), SMLA_EALIGN), (dict(out_token_stride=513), SMLA_EALIGN), (dict(total_q=2 ** 31), SMLA_ETOOBIG),
    (dict(total_k=2 ** 31), SMLA_ETOOBIG), (dict(total_q=2 ** 30, num_heads=2048), SMLA_ETOOBIG),
    (dict(batch=0), SMLA_OK), (dict(total_q=0), SMLA_OK),
])
def test_prefill_c_refusals(abi, change, code):
    assert abi.load().smla_dense_mla_prefill(ctypes.byref(_prefill_params(abi, **change)), None) == code


def test_null_structs_are_refused(abi):
    lib = abi.load()
    assert lib.smla_dense_mla_prefill(None, None) == SMLA_EINVAL
    assert lib.smla_cache_row_weights(None, None) == SMLA_EINVAL
    assert lib.smla_compact_cache(None, None) == SMLA_EINVAL


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), SMLA_EINVAL), (dict(seqlen_q=0), SMLA_EINVAL), (dict(head_dim=192), SMLA_EINVAL), (dict(page_block_size=0), SMLA_EINVAL),
    (dict(block_table_stride=1), SMLA_EINVAL), (dict(weights_stride=8), SMLA_EINVAL), (dict(q=0), SMLA_EINVAL), (dict(softmax_lse=0), SMLA_EINVAL),
    (dict(weights=0), SMLA_EINVAL), (dict(block_table=0), SMLA_EINVAL), (dict(k_cache=0), SMLA_EINVAL), (dict(page_block_size=12), SMLA_EALIGN),
    (dict(q=FAKE + 8), SMLA_EALIGN), (dict(k_row_stride=1024), SMLA_EALIGN), (dict(k_row_stride=1160), SMLA_EALIGN),
    (dict(num_blocks=2 ** 30), SMLA_ETOOBIG), (dict(seqlen_q=2 ** 20, num_heads=128), SMLA_ETOOBIG), (dict(batch=0), SMLA_OK),
    (dict(weights_width=0), SMLA_OK),
])
def test_row_weights_c_refusals(abi, change, code):
    p = abi.SmlaRowWeightsParams()
    vals = dict(batch=2, seqlen_q=1, num_heads=4, causal=0, head_dim=576, softmax_scale=0.1, q=FAKE, softmax_lse=FAKE, k_cache=FAKE,
                k_block_stride=16 * 1152, k_row_stride=1152, num_blocks=5, page_block_size=16, max_blocks_per_seq=2, block_table=FAKE,
                block_table_stride=2, cache_seqlens=FAKE, weights=FAKE, weights_stride=32, weights_width=32, accumulate=0)
    vals.update(change)
    for k, v in vals.items():
        setattr(p, k, v)
    assert abi.load().smla_cache_row_weights(ctypes.byref(p), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), SMLA_EINVAL), (dict(budget=0), SMLA_EINVAL), (dict(recent=5), SMLA_EINVAL), (dict(recent=-1), SMLA_EINVAL),
    (dict(stride=3), SMLA_EINVAL), (dict(weights=0), SMLA_EINVAL), (dict(lens=0), SMLA_EINVAL), (dict(rows=0), SMLA_EINVAL),
    (dict(kept=0), SMLA_EINVAL), (dict(batch=0), SMLA_OK),
])
def test_select_c_refusals(abi, change, code):
    a = dict(weights=FAKE, stride=8, width=8, lens=FAKE, batch=1, budget=4, recent=0, rows=FAKE, kept=FAKE, vals=FAKE)
    a.update(change)
    assert abi.load().smla_select_cache_rows(a["weights"], a["stride"], a["width"], a["lens"], a["batch"], a["budget"], a["recent"],
                                             a["rows"], a["kept"], a["vals"], None) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), SMLA_EINVAL), (dict(row_bytes=0), SMLA_EINVAL), (dict(row_stride=512), SMLA_EINVAL), (dict(cache=0), SMLA_EINVAL),
    (dict(rows=0), SMLA_EINVAL), (dict(kept=0), SMLA_EINVAL), (dict(block_table=0), SMLA_EINVAL), (dict(out_block_table=0), SMLA_EINVAL),
    (dict(row_bytes=1148), SMLA_EALIGN), (dict(cache=FAKE + 8), SMLA_EALIGN), (dict(num_blocks=2 ** 30), SMLA_ETOOBIG),
    (dict(budget=0), SMLA_OK), (dict(batch=0), SMLA_OK), (dict(num_blocks=0), SMLA_OK),
])
def test_compact_c_refusals(abi, change, code):
    p = abi.SmlaCompactParams()
    vals = dict(batch=1, budget=4, cache=FAKE, block_stride=16 * 1152, row_stride=1152, row_bytes=1152, num_blocks=4, page_block_size=16,
                block_table=FAKE, block_table_stride=2, max_blocks_per_seq=2, out_block_table=FAKE, out_block_table_stride=2,
                out_max_blocks_per_seq=2, rows=FAKE, kept=FAKE)
    vals.update(change)
    for k, v in vals.items():
        setattr(p, k, v)
    assert abi.load().smla_compact_cache(ctypes.byref(p), None) == code


# ----------------------------------------------------------------------------- oracles
def test_prefill_oracle_against_softmax():
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(5, 2, 192, generator=g), torch.randn(9, 1, 192, generator=g), torch.randn(9, 1, 128, generator=g)
    cu_q, cu_k = torch.tensor([0, 5]), torch.tensor([0, 9])
    out, lse, _, _ = oracle.dense_mla_prefill(q, k, v, cu_q, cu_k, causal=True)
    s = torch.einsum("qhd,kd->hqk", q.double(), k[:, 0].double()) * 192 ** -0.5
    s = s.masked_fill(~torch.ones(5, 9, dtype=torch.bool).tril(4), float("-inf"))
    torch.testing.assert_close(out, torch.einsum("hqk,kd->qhd", s.softmax(-1), v[:, 0].double()))
    torch.testing.assert_close(lse, s.logsumexp(-1))


def test_weight_oracle_sums_to_the_number_of_queries():
    """Each query's weights sum to one, so the weights of all rows sum to heads x positions."""
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 3, 4, 512, generator=g)
    cache = torch.randn(6, 8, 1, 512, generator=g)
    table = torch.tensor([[3, 1, 5], [0, 2, 4]], dtype=torch.int32)
    lens = torch.tensor([20, 9], dtype=torch.int32)
    _, lse = oracle.dense_mla_decode(q, cache, table, lens, causal=True)
    w, _ = oracle.cache_row_weights(q, cache, table, lens, torch.from_numpy(lse), causal=True)
    torch.testing.assert_close(w.sum(1), torch.full((2,), 12.0).double(), rtol=1e-5, atol=1e-5)
    assert (w[0, 20:] == 0).all() and (w[1, 9:] == 0).all()


def test_select_oracle():
    nan, inf = float("nan"), float("inf")
    w = torch.tensor([[1.0, 5.0, 5.0, nan, -inf, 2.0, 0.0, -0.0, 9.0, 9.0]])
    rows, kept, vals = oracle.select_cache_rows(w, torch.tensor([10]), 4, 1)
    assert rows.tolist() == [[1, 2, 8, 9]] and kept.tolist() == [4] and vals.tolist() == [[5.0, 5.0, 9.0, 9.0]]
    rows, _, _ = oracle.select_cache_rows(w[:, :9], torch.tensor([9]), 8)
    assert rows.tolist() == [[0, 1, 2, 4, 5, 6, 7, 8]]          # the NaN goes
    rows, kept, _ = oracle.select_cache_rows(w, torch.tensor([3]), 4)
    assert rows.tolist() == [[0, 1, 2, -1]] and kept.tolist() == [3]


def test_compact_oracle():
    cache = torch.arange(4 * 2 * 8).view(4, 2, 1, 8).to(torch.bfloat16)
    table = torch.tensor([[2, 0], [3, 9]], dtype=torch.int32)
    rows, kept = torch.tensor([[1, 2], [1, 3]], dtype=torch.int32), torch.tensor([2, 2], dtype=torch.int32)
    got = oracle.compact_cache(cache, table, rows, kept)
    assert torch.equal(got[2, 0], cache[2, 1]) and torch.equal(got[2, 1], cache[0, 0])
    assert torch.equal(got[3, 0], cache[3, 1]) and (got[3, 1] == 0).all()       # page 9 does not exist
    assert torch.equal(got[0], cache[0]) and torch.equal(got[1], cache[1])


# ----------------------------------------------------------------------------- sums with room for rows appended later
def test_select_refuses_places_for_the_kept_weights(fm):
    w, lens = torch.zeros(2, 9), torch.zeros(2, dtype=torch.int32)
    for bad in (torch.zeros(2, 3), torch.zeros(1, 9), torch.zeros(2, 9, dtype=torch.float64), torch.zeros(18), w, w[:, :5]):
        with pytest.raises(ValueError):
            fm.mla_select_cache_rows(w, lens, 4, 1, kept_weights=bad)


@pytest.mark.parametrize("change,code", [
    (dict(kept_width=3), SMLA_EINVAL), (dict(kept_stride=7), SMLA_EINVAL), (dict(width=2, stride=2, kept_width=1), SMLA_EINVAL),
    (dict(vals=FAKE), SMLA_EINVAL), (dict(vals=FAKE + 4 * 40), SMLA_EINVAL), (dict(vals=FAKE - 4 * 40), SMLA_EINVAL),
    (dict(vals=FAKE + 4 * 7, stride=16, kept_stride=16), SMLA_EINVAL), (dict(vals=FAKE + 4 * 9, stride=16, kept_stride=16), SMLA_EINVAL),
    (dict(vals=FAKE - 4 * 7, stride=16, kept_stride=16), SMLA_EINVAL), (dict(vals=FAKE + 4 * 8, stride=16, kept_stride=15), SMLA_EINVAL),
    (dict(batch=0), SMLA_OK), (dict(budget=0), SMLA_EINVAL),
])
def test_select_into_c_refusals(abi, change, code):
    """weights [8, 8], kept_weights [8, 8] that are too narrow, the same, or partly the same."""
    a = dict(weights=FAKE, stride=8, width=8, lens=FAKE, batch=8, budget=4, recent=0, rows=FAKE, kept=FAKE, vals=FAKE + 4096, kept_stride=8,
             kept_width=8)
    a.update(change)
    assert abi.load().smla_select_cache_rows_into(a["weights"], a["stride"], a["width"], a["lens"], a["batch"], a["budget"], a["recent"],
                                                  a["rows"], a["kept"], a["vals"], a["kept_stride"], a["kept_width"], None) == code


def test_two_evictions_of_the_oracle_keep_the_newest_rows():
    """200 rows, 64 stay; 40 more; the second choice is among 104 and has the last 16, where the sums have room for them."""
    g = torch.Generator().manual_seed(2)
    sums = torch.rand(1, 320, generator=g)
    sums[:, 200:] = 0
    rows, kept, sums = oracle.select_cache_rows(sums, torch.tensor([200]), 64, 16, columns=320)
    assert sums.shape == (1, 320) and (sums[:, 64:] == 0).all()
    sums[:, :104] += torch.rand(1, 104, generator=g)
    rows, kept, sums = oracle.select_cache_rows(sums, torch.tensor([104]), 64, 16, columns=320)
    assert rows[0, -16:].tolist() == list(range(88, 104)) and kept.tolist() == [64]


@pytest.mark.parametrize("width,code", [(2 ** 31 - 1, SMLA_ETOOBIG), (2 ** 31 - 1024, SMLA_ETOOBIG)])
def test_row_weights_refuse_rows_that_a_tile_would_count_past_an_int(abi, width, code):
    """A tile of 256 rows and a piece of 1024 columns that begin in front of 2^31 must end there."""
    p = abi.SmlaRowWeightsParams()
    vals = dict(batch=1, seqlen_q=1, num_heads=4, head_dim=576, softmax_scale=0.1, q=FAKE, softmax_lse=FAKE, k_cache=FAKE,
                k_block_stride=16 * 1152, k_row_stride=1152, num_blocks=5, page_block_size=16, max_blocks_per_seq=2, block_table=FAKE,
                block_table_stride=2, cache_seqlens=FAKE, weights=FAKE, weights_stride=width, weights_width=width)
    for k, v in vals.items():
        setattr(p, k, v)
    assert abi.load().smla_cache_row_weights(ctypes.byref(p), None) == code
