"""CPU oracle for the sparse-MLA hot path.  TEST INFRASTRUCTURE, NOT PRODUCT.

This package restates, on the CPU, what the reference's fp32 torch oracle and
its byte-format helpers compute for sparse MLA attention over ``fp8_ds_mla`` /
``int8_ds_mla`` paged caches, for the int8 row quantizer, and for dense paged MLA
decode over bf16 caches.  Only the test
suite, the smoke check and the benchmark's CPU-baseline / reference arm may
import it; the product package never does (the product fails loudly when its
CUDA library is missing instead of falling back to this code).

Parity is pinned: ``tests/golden/*.npz`` hold inputs and outputs produced by the
reference's own Python code (its ``_ref`` / ``_fp32_ref`` oracles, cache packers
and ``quantize_int8_ds_mla_rows``), generated by ``tests/golden/make_golden.py``;
``tests/test_oracle_golden.py`` checks every function here against them.
"""
from .ds_mla_formats import (  # noqa: F401
    E4M3_LUT,
    bf16_bits_to_f32,
    f32_to_bf16_bits,
    dequant_fp8_ds_mla,
    dequant_int8_ds_mla,
    pack_fp8_ds_mla,
    pack_int8_inline528,
    quantize_int8_rows,
    quantize_int8_rows_writer,
    ue8m0_exponents,
    write_fp8_ds_mla,
    write_int8_inline528,
)
from .sparse_mla_ref import sparse_mla_attention, cos_diff  # noqa: F401
from .dense_mla_ref import dense_mla_decode  # noqa: F401
from .dense_prefill_ref import dense_mla_prefill  # noqa: F401
from .cache_eviction_ref import cache_row_weights, compact_cache, select_cache_rows, sequence_slots  # noqa: F401
