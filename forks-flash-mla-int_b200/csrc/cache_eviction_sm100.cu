// Choice of the rows of a sequence that stay in its cache, and their move to the front, for sm_100a.
//
// Selection.  Weights become 32-bit keys that order as they do (sign folded, -0 made 0, NaN made the lowest).
// Four passes of eight bits find the key T of the row that is last among the heaviest: a pass counts the
// digits of the keys that agree with T so far and takes the digit at which the count from above reaches the
// rows still wanted.  Rows above T stay, rows equal to T stay from the lowest on until the budget is full.
// One CTA per sequence.
//
// Move.  Rows are copied in ascending order, a block of rows at a time: all loads of a block precede its
// stores, so that in-place moves never overwrite a row that is still to be read (its source index is at
// least its target's).
#include <cuda_runtime.h>
#include <cstdint>

#include "smla_internal.h"

namespace smla {
namespace {

constexpr int kSelThreads = 1024;

__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);            // -0 + 0 = 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kSelThreads) select_rows_kernel(const float *weights, int64_t stride, int width,
                                                                  const int32_t *lens, int budget, int recent, int32_t *rows,
                                                                  int32_t *kept, float *kept_weights) {
    __shared__ unsigned hist[256];
    __shared__ unsigned s_prefix, s_want;
    __shared__ int s_cnt[2][33];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = min(max(lens[b], 0), width);
    const float *w = weights + b * stride;
    rows += static_cast<int64_t>(b) * budget;
    if (kept_weights) kept_weights += static_cast<int64_t>(b) * budget;
    if (tid == 0) kept[b] = min(len, budget);
    for (int j = min(len, budget) + tid; j < budget; j += kSelThreads) {
        rows[j] = -1;
        if (kept_weights) kept_weights[j] = 0.0f;
    }
    if (len <= budget) {
        for (int j = tid; j < len; j += kSelThreads) {
            rows[j] = j;
            if (kept_weights) kept_weights[j] = w[j];
        }
        return;
    }
    const int old = len - recent, want0 = budget - recent;
    for (int j = tid; j < recent; j += kSelThreads) {
        rows[want0 + j] = old + j;
        if (kept_weights) kept_weights[want0 + j] = w[old + j];
    }
    if (want0 == 0) return;
    unsigned prefix = 0, want = want0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < old; j += kSelThreads) {
            const uint32_t k = weight_key(w[j]);
            if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255;
            unsigned left = want;
            while (hist[d] < left) left -= hist[d--];
            s_prefix = (prefix << 8) | d;
            s_want = left;
        }
        __syncthreads();
        prefix = s_prefix;
        want = s_want;
        __syncthreads();
    }
    // rows above `prefix` stay, and the first `want` rows equal to it
    int out = 0, ties = 0;
    for (int j0 = 0; j0 < old; j0 += kSelThreads) {
        const int j = j0 + tid;
        const uint32_t k = j < old ? weight_key(w[j]) : 0u;
        const bool above = j < old && k > prefix, tie = j < old && k == prefix;
        const unsigned ba = __ballot_sync(0xffffffffu, above), bt = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) {
            s_cnt[0][warp] = __popc(ba);
            s_cnt[1][warp] = __popc(bt);
        }
        __syncthreads();
        int a = out, t = ties;
        for (int i = 0; i < warp; ++i) {
            a += s_cnt[0][i];
            t += s_cnt[1][i];
        }
        for (int i = 0; i < kSelThreads / 32; ++i) {
            out += s_cnt[0][i];
            ties += s_cnt[1][i];
        }
        const unsigned below = (1u << lane) - 1u;
        a += __popc(ba & below);
        t += __popc(bt & below);
        if (above || (tie && t < static_cast<int>(want))) {
            const int at = a + min(t, static_cast<int>(want));
            rows[at] = j;
            if (kept_weights) kept_weights[at] = w[j];
        }
        __syncthreads();
    }
}

__device__ __forceinline__ const uint8_t *row_at(const smla_compact_params_t &p, const int32_t *table, int columns, int row) {
    const int col = row / p.page_block_size;
    if (row < 0 || col >= columns) return nullptr;
    const int page = table[col];
    if (page < 0 || page >= p.num_blocks) return nullptr;
    return static_cast<const uint8_t *>(p.cache) + page * p.block_stride + (row - col * p.page_block_size) * p.row_stride;
}

constexpr int kMoveThreads = 256;
constexpr int kSlice = 128;                                  // bytes of a row that one CTA moves

__global__ void __launch_bounds__(kMoveThreads) compact_kernel(const smla_compact_params_t p) {
    const int b = blockIdx.y, n = min(max(p.kept[b], 0), p.budget);
    const int piece = threadIdx.x % (kSlice / 16);
    const int at = blockIdx.x * kSlice + piece * 16;
    const int32_t *rows = p.rows + static_cast<int64_t>(b) * p.budget;
    constexpr int kRows = kMoveThreads / (kSlice / 16);
    for (int j0 = 0; j0 < n; j0 += kRows) {
        const int j = j0 + threadIdx.x / (kSlice / 16);
        const bool mine = j < n && at < p.row_bytes;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (mine) {
            const uint8_t *src = row_at(p, p.block_table + b * p.block_table_stride, p.max_blocks_per_seq, rows[j]);
            if (src) x = *reinterpret_cast<const uint4 *>(src + at);
        }
        __syncthreads();
        if (mine) {
            uint8_t *dst = const_cast<uint8_t *>(row_at(p, p.out_block_table + b * p.out_block_table_stride, p.out_max_blocks_per_seq, j));
            if (dst) *reinterpret_cast<uint4 *>(dst + at) = x;
        }
        __syncthreads();
    }
}

}  // namespace

int launch_select_rows(const float *weights, int64_t weights_stride, int width, const int32_t *lens, int batch, int budget,
                       int recent, int32_t *rows, int32_t *kept, float *kept_weights, cudaStream_t stream) {
    select_rows_kernel<<<batch, kSelThreads, 0, stream>>>(weights, weights_stride, width, lens, budget, recent, rows, kept, kept_weights);
    return static_cast<int>(cudaGetLastError());
}

int launch_compact(const smla_compact_params_t &p, int, cudaStream_t stream) {
    if (p.batch > 65535) return SMLA_ETOOBIG;
    compact_kernel<<<dim3((p.row_bytes + kSlice - 1) / kSlice, p.batch), kMoveThreads, 0, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace smla
