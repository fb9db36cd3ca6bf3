// Attention weight of each cached row for sm_100a: w[b, r] = sum over queries i and heads h of
// exp(scale q_bih . K_br - lse_bhi), over the paged bf16 latent cache of dense MLA decode.
//
// One warp per row: its dims stay in registers, the queries stream past.  Bound by instruction issue.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "smla_internal.h"

namespace smla {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__global__ void __launch_bounds__(256) row_weights_kernel(const smla_row_weights_params_t p) {
    const int lane = threadIdx.x & 31, b = blockIdx.y;
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= p.weights_width) return;
    const long long cap = static_cast<long long>(p.max_blocks_per_seq) * p.page_block_size;
    const int len = static_cast<int>(min(static_cast<long long>(max(p.cache_seqlens[b], 0)), cap));
    float *dst = p.weights + b * p.weights_stride + r;
    if (r >= len) {
        if (!p.accumulate && lane == 0) *dst = 0.0f;
        return;
    }
    const int page = p.block_table[b * p.block_table_stride + r / p.page_block_size];
    const int pairs = p.head_dim / 2;            // 288 or 256: nine or eight to a lane
    float2 k[9];
    const uint32_t *row = reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(p.k_cache) + page * p.k_block_stride +
                                                             (r % p.page_block_size) * p.k_row_stride);
    const bool real = page >= 0 && page < p.num_blocks;
#pragma unroll
    for (int e = 0; e < 9; ++e) {
        const uint32_t w = (real && e * 32 + lane < pairs) ? row[e * 32 + lane] : 0u;
        k[e] = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
    float sum = 0.0f;
    for (int i = 0; i < p.seqlen_q; ++i) {
        if (p.causal && r >= len - (p.seqlen_q - 1 - i)) continue;
        for (int h = 0; h < p.num_heads; ++h) {
            const uint32_t *q = static_cast<const uint32_t *>(p.q) +
                                ((static_cast<long long>(b) * p.seqlen_q + i) * p.num_heads + h) * pairs;
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < 9; ++e) {
                if (e * 32 + lane >= pairs) continue;
                const uint32_t w = q[e * 32 + lane];
                s = fmaf(k[e].x, __uint_as_float(w << 16), fmaf(k[e].y, __uint_as_float(w & 0xFFFF0000u), s));
            }
            for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            const float lse = p.softmax_lse[(static_cast<long long>(b) * p.num_heads + h) * p.seqlen_q + i];
            if (lse != -INFINITY) sum += exp2f((s * p.softmax_scale - lse) * kLog2e);
        }
    }
    if (lane == 0) *dst = p.accumulate ? *dst + sum : sum;
}

}  // namespace

int launch_row_weights(const smla_row_weights_params_t &p, int, cudaStream_t stream) {
    if (p.batch > 65535) return SMLA_ETOOBIG;
    row_weights_kernel<<<dim3(static_cast<unsigned>((p.weights_width + 7) / 8), static_cast<unsigned>(p.batch)), 256, 0, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace smla
