// Attention weight of each cached row for sm_100a: w[b, r] = sum over query positions i and heads h that see row r of
// exp(scale q_bih . K_br - lse_bhi), over the paged bf16 latent cache of dense MLA decode.
//
// The (position, head) pairs of a sequence are columns c = i H + h of one matrix product: S^T = K Q^T with 128 cached
// rows as M (the lanes of tensor memory) and N columns.  A row's weight is then a sum along its own lane: no exchange
// between threads, and a fixed order (per block of columns, then block after block).  There is no running maximum: the
// lse is known, every term is at most 1.  Under the causal mask position i sees the rows r < len - (s_q - 1 - i), so a
// row is seen by the columns c >= max(0, r - len + s_q) H: one threshold per lane.
//
// Two forms, by the number of columns C = s_q H (both persistent, one CTA per SM, tiles of 128 rows in contiguous ranges):
//   C <= 128 (a decode step)  bound by reading the rows once.  K and Q slabs [rows][64 dims] stream through one ring of
//            stages; Q (N x 64 dims a stage) is fetched again for each tile, from L2: N / 128 of the rows' bytes.
//   C > 128 (a window)        bound by the tensor pipe.  The tile's rows stay in shared memory (147 KB) while the columns
//            pass in blocks of 256 through the ring; the next tile's slabs replace the rows as the last block leaves them.
// Roles (384 threads): warps 0-3 and 4-7 take turns at the score blocks (two accumulators), warp 8 issues the MMAs, warp
// 9 finds the tiles and loads.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "smla_internal.h"
#include "tensor_map.h"

namespace smla {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 384;
constexpr int kSlab = 128 * 128;                 // bytes of [128 rows][64 dims] of bf16
constexpr int kRecords = 4;

struct WeightsArgs {
    CUtensorMap q_map, k_map;
    const int32_t *table, *lens;
    int64_t table_stride;
    const float *lse;
    float *weights;
    int64_t w_stride;
    int width, accumulate, batch, s_q, heads, columns, causal, k_slabs;
    int num_blocks, page, box_rows, max_blocks;
    float scale_log2;
    int *status;
};

// RES: the rows stay while the columns pass.  N: columns of a score block.
template <bool RES, int N>
struct Smem {
    static constexpr int kQSlab = N * 128;
    static constexpr int kStage = RES ? kQSlab : kSlab + kQSlab;
    static constexpr int kStages = RES ? 2 : (208 * 1024 / kStage < 12 ? 208 * 1024 / kStage : 12);
    static constexpr int kResident = RES ? 9 : 0;
    static constexpr int kRingAt = kResident * kSlab;
    static constexpr int kLse = kRingAt + kStages * kStage;              // two buffers of N floats
    static constexpr int kSums = kLse + 2 * N * 4;                       // RES: the second group's sums of a tile
    static constexpr int kBars = kSums + 128 * 4;
    static constexpr int kBarFull = 0, kBarEmpty = kStages, kBarKFull = 2 * kStages, kBarKEmpty = kBarKFull + kResident,
                         kBarS = kBarKEmpty + kResident, kBarSFree = kBarS + 2, kBarRecFull = kBarSFree + 2,
                         kBarRecEmpty = kBarRecFull + kRecords, kNumBars = kBarRecEmpty + kRecords;
    static constexpr int kRecs = kBars + kNumBars * 8;                   // {valid, sequence, first row, length}
    static constexpr int kMisc = kRecs + kRecords * 16;
    static constexpr int kBytes = kMisc + 16;
    static constexpr int kTmemCols = 2 * N < 32 ? 32 : 2 * N;
};
static_assert(Smem<true, 256>::kBytes <= 232448 && Smem<false, 128>::kBytes <= 232448, "shared memory of one CTA");

__device__ __forceinline__ void give_up(volatile int *abort_flag, int *status, int bit) {
    *abort_flag = 1;
    atomicOr(status, bit);
}

// Rows of sequence b that take part.
__device__ __forceinline__ int rows_of(const WeightsArgs &a, int b, int *length = nullptr) {
    const int64_t cap = static_cast<int64_t>(a.max_blocks) * a.page;
    const int len = static_cast<int>(min(static_cast<int64_t>(max(__ldg(a.lens + b), 0)), cap));
    if (length) *length = len;
    return min(len, a.width);
}

// ------------------------------------------------------------------ loader
template <bool RES, int N>
__device__ __forceinline__ void loader_role(const WeightsArgs &a, uint8_t *smem, volatile int *abort_flag, int lane) {
    using L = Smem<RES, N>;
    const uint32_t bars = smem_u32(smem + L::kBars), ring = smem_u32(smem + L::kRingAt), ks = smem_u32(smem);
    // this CTA's range of the tiles of all sequences
    long long total = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32)
        total += __reduce_add_sync(0xffffffffu, b0 + lane < a.batch ? (rows_of(a, b0 + lane) + 127) >> 7 : 0);
    const long long first = total * blockIdx.x / gridDim.x, end = total * (blockIdx.x + 1) / gridDim.x;
    const int boxes = 128 / a.box_rows, blocks = RES ? (a.columns + N - 1) / N : 1;
    long long base = 0;                          // tiles in front of the 32 sequences at b0
    int b0 = 0, rec_i = 0;
    uint32_t st = 0, tile_n = 0, k_loads = 0;
    bool ok = true;
    for (long long idx = first; ok; ++idx, ++rec_i) {
        int b = -1, t = 0;
        while (idx < end && b0 < a.batch) {
            const int n = b0 + lane < a.batch ? (rows_of(a, b0 + lane) + 127) >> 7 : 0;
            int upto = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += x;
            }
            const long long r = idx - base;
            const unsigned hit = __ballot_sync(0xffffffffu, r >= upto - n && r < upto);
            if (hit != 0u) {
                const int src = __ffs(hit) - 1;
                b = b0 + src;
                t = static_cast<int>(r) - __shfl_sync(0xffffffffu, upto - n, src);
                break;
            }
            base += __shfl_sync(0xffffffffu, upto, 31);
            b0 += 32;
        }
        const int slot = rec_i % kRecords;
        if (!(ok = mbar_wait(bars + (L::kBarRecEmpty + slot) * 8, ((rec_i / kRecords) & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
            int *rec = reinterpret_cast<int *>(smem + L::kRecs) + slot * 4;
            int len = 0;
            if (b >= 0) rows_of(a, b, &len);
            rec[0] = b >= 0;
            rec[1] = b;
            rec[2] = t * 128;
            rec[3] = len;
            mbar_arrive(bars + (L::kBarRecFull + slot) * 8);
        }
        __syncwarp();
        if (b < 0) break;
        // the pages of the tile's boxes; one outside the table or the cache lies past the tensor's end: zeros
        int page = a.num_blocks, in_page = 0;
        if (lane < boxes) {
            const int row = t * 128 + lane * a.box_rows, col = row / a.page;
            in_page = row - col * a.page;
            if (col < a.max_blocks) page = __ldg(a.table + b * a.table_stride + col);
            if (page < 0 || page > a.num_blocks) page = a.num_blocks;
        }
        const int q_row = b * a.columns;
        for (int cb = 0; cb < blocks && ok; ++cb) {
            for (int s = 0; s < a.k_slabs; ++s, ++st) {
                if (RES && cb == 0) {
                    if (!(ok = mbar_wait(bars + (L::kBarKEmpty + s) * 8, (tile_n & 1) ^ 1, abort_flag))) break;
                    if (lane == 0) mbar_arrive_expect_tx(bars + (L::kBarKFull + s) * 8, kSlab);
                    __syncwarp();
                    if (lane < boxes)
                        tma_load_3d(ks + s * kSlab + lane * a.box_rows * 128, &a.k_map, bars + (L::kBarKFull + s) * 8, s * 64, in_page, page);
                    ++k_loads;
                }
                const uint32_t at = st % L::kStages, full = bars + (L::kBarFull + at) * 8, dst = ring + at * L::kStage;
                if (!(ok = mbar_wait(bars + (L::kBarEmpty + at) * 8, ((st / L::kStages) & 1) ^ 1, abort_flag))) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(full, L::kStage);
                    constexpr int kBox = N < 128 ? N : 128;
#pragma unroll
                    for (int x = 0; x < N / kBox; ++x)
                        tma_load_3d(dst + (RES ? 0 : kSlab) + x * kBox * 128, &a.q_map, full, s * 64, q_row + cb * N + x * kBox, 0);
                }
                __syncwarp();
                if (!RES && lane < boxes) tma_load_3d(dst + lane * a.box_rows * 128, &a.k_map, full, s * 64, in_page, page);
            }
        }
        if (ok) ++tile_n;
    }
    if (!ok) {
        // the copies in flight have to land before the CTA may end
        if (lane == 0) give_up(abort_flag, a.status, kStatusGatherWait);
        __syncwarp();
        int never = 0;
        for (uint32_t i = st > static_cast<uint32_t>(L::kStages) ? st - L::kStages : 0; i < st; ++i)
            mbar_wait(bars + (L::kBarFull + i % L::kStages) * 8, (i / L::kStages) & 1, &never);
        for (uint32_t i = k_loads > static_cast<uint32_t>(a.k_slabs) ? k_loads - a.k_slabs : 0; i < k_loads; ++i)
            mbar_wait(bars + (L::kBarKFull + i % a.k_slabs) * 8, (i / a.k_slabs) & 1, &never);
    }
}

// ------------------------------------------------------------------ MMA issue
template <bool RES, int N>
__device__ __forceinline__ void mma_role(const WeightsArgs &a, uint8_t *smem, uint32_t tmem, volatile int *abort_flag, int lane) {
    using L = Smem<RES, N>;
    const uint32_t bars = smem_u32(smem + L::kBars), ring = smem_u32(smem + L::kRingAt);
    const uint32_t go = elect_one();
    constexpr uint32_t idesc = umma_idesc_bf16(128, N, 0, 0);
    const uint64_t kd = umma_desc_sw128(RES ? smem_u32(smem) : ring, 16), qd = umma_desc_sw128(ring + (RES ? 0 : kSlab), 16);
    const int blocks = RES ? (a.columns + N - 1) / N : 1;
    uint32_t st = 0, n_blocks = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
        const int slot = it % kRecords;
        if (!(ok = mbar_wait(bars + (L::kBarRecFull + slot) * 8, (it / kRecords) & 1, abort_flag))) break;
        const int valid = reinterpret_cast<const volatile int *>(smem + L::kRecs)[slot * 4];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) break;
        for (int cb = 0; cb < blocks && ok; ++cb, ++n_blocks) {
            const int buf = n_blocks & 1;
            if (!(ok = mbar_wait(bars + (L::kBarSFree + buf) * 8, ((n_blocks >> 1) & 1) ^ 1, abort_flag))) break;
            for (int s = 0; s < a.k_slabs; ++s, ++st) {
                if (RES && cb == 0 && !(ok = mbar_wait(bars + (L::kBarKFull + s) * 8, it & 1, abort_flag))) break;
                const uint32_t at = st % L::kStages;
                if (!(ok = mbar_wait(bars + (L::kBarFull + at) * 8, (st / L::kStages) & 1, abort_flag))) break;
                tc_fence_after_sync();
                const uint64_t ka = kd + static_cast<uint64_t>((RES ? s * kSlab : at * L::kStage) >> 4);
                const uint64_t qb = qd + static_cast<uint64_t>((at * L::kStage) >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_bf16_ss_pred(tmem + buf * N, ka + 2 * k, qb + 2 * k, idesc, (s | k) != 0 ? 1u : 0u, go);
                umma_commit_pred(bars + (L::kBarEmpty + at) * 8, go);
                if (RES && cb + 1 == blocks) umma_commit_pred(bars + (L::kBarKEmpty + s) * 8, go);
            }
            if (ok) umma_commit_pred(bars + (L::kBarS + buf) * 8, go);
        }
    }
    if (!ok && lane == 0) give_up(abort_flag, a.status, kStatusMmaWait);
}

// ------------------------------------------------------------------ sums
// Sum of exp2(s c - lse2) over `kCols` columns of this lane; with MASK only the columns in [lo, hi).
template <int kCols, bool MASK>
__device__ __forceinline__ void add_columns(uint32_t taddr, const float *lse2, float c, int lo, int hi, uint64_t (&acc)[4]) {
    uint32_t s[kCols];
    if constexpr (kCols == 32) {
        tmem_ld_x32_nowait(taddr, s);
        tmem_ld_wait();
    } else {
        tmem_ld_x16(taddr, s);
    }
    const uint64_t c2 = pack2(c, c);
#pragma unroll
    for (int j = 0; j < kCols; j += 4) {
        const float4 z = *reinterpret_cast<const float4 *>(lse2 + j);    // negated
        float x[4];
        unpack2(fma2(pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), c2, pack2(z.x, z.y)), x[0], x[1]);
        unpack2(fma2(pack2(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])), c2, pack2(z.z, z.w)), x[2], x[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = fast_exp2(x[e]);
            if (MASK && (j + e < lo || j + e >= hi)) x[e] = 0.0f;
        }
        acc[(j >> 1) & 3] = add2(acc[(j >> 1) & 3], pack2(x[0], x[1]));
        acc[((j >> 1) & 3) + 1] = add2(acc[((j >> 1) & 3) + 1], pack2(x[2], x[3]));
    }
}

template <bool RES, int N>
__device__ __forceinline__ void sum_role(const WeightsArgs &a, uint8_t *smem, uint32_t tmem, volatile int *abort_flag, int warp, int lane) {
    using L = Smem<RES, N>;
    constexpr int kCols = N < 32 ? N : 32;
    const uint32_t bars = smem_u32(smem + L::kBars);
    const int group = warp >> 2, lane_row = (warp & 3) * 32 + lane;
    float *lse2 = reinterpret_cast<float *>(smem + L::kLse) + group * N;
    float *sums = reinterpret_cast<float *>(smem + L::kSums);
    const uint32_t t_addr = tmem + group * N + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int blocks = RES ? (a.columns + N - 1) / N : 1;
    uint32_t n_blocks = 0;
    bool failed = false;
    for (int it = 0;; ++it) {
        const int slot = it % kRecords;
        failed |= !mbar_wait(bars + (L::kBarRecFull + slot) * 8, (it / kRecords) & 1, abort_flag);
        // whoever meets at the barriers below leaves together
        if (RES ? named_bar_or(3, 256, failed) : named_bar_or(1 + group, 128, failed)) {
            if (lane == 0) give_up(abort_flag, a.status, kStatusSoftmaxWait);
            return;
        }
        const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * 4;
        const int valid = rec[0], b = rec[1], row = rec[2] + lane_row, len = rec[3];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) return;
        // columns below `from` do not see this row; the warp's last row sees the fewest
        const int from = a.causal ? max(0, row - len + a.s_q) * a.heads : 0;
        const int from_warp = a.causal ? max(0, row - lane + 31 - len + a.s_q) * a.heads : 0;
        float total = 0.0f, lost = 0.0f;         // compensated sum over the blocks
        for (int cb = 0; cb < blocks; ++cb, ++n_blocks) {
            if ((n_blocks & 1) != static_cast<uint32_t>(group)) continue;
            const int c0 = cb * N;
            for (int x = lane_row; x < N; x += 128) {
                const int c = c0 + x, i = c / a.heads, h = c - i * a.heads;
                float z = -INFINITY;
                if (c < a.columns) {
                    z = -__ldg(a.lse + (static_cast<int64_t>(b) * a.heads + h) * a.s_q + i) * kLog2e;
                    if (z == INFINITY) z = -INFINITY;            // a query that saw no row
                }
                lse2[x] = z;
            }
            failed |= !mbar_wait(bars + (L::kBarS + group) * 8, (n_blocks >> 1) & 1, abort_flag);
            named_bar_sync(1 + group, 128);
            tc_fence_after_sync();
            uint64_t acc[4] = {0, 0, 0, 0};
            if (from_warp <= c0 && c0 + N <= a.columns) {
#pragma unroll 2
                for (int j = 0; j < N; j += kCols) add_columns<kCols, false>(t_addr + j, lse2 + j, a.scale_log2, 0, 0, acc);
            } else {
                // columns of the block that count for this row (those past the last hold other queries' scores)
                const int lo = from - c0, hi = a.columns - c0;
                for (int j = 0; j < N; j += kCols) add_columns<kCols, true>(t_addr + j, lse2 + j, a.scale_log2, lo - j, hi - j, acc);
            }
            tc_fence_before_sync();
            named_bar_sync(1 + group, 128);      // the scores and the lse buffer have been read
            if ((warp & 3) == 0 && lane == 0) mbar_arrive(bars + (L::kBarSFree + group) * 8);
            const uint64_t both = add2(add2(acc[0], acc[1]), add2(acc[2], acc[3]));
            float x, y;
            unpack2(both, x, y);
            const float part = __fadd_rn(x, y), corrected = __fsub_rn(part, lost), sum = __fadd_rn(total, corrected);
            lost = __fsub_rn(__fsub_rn(sum, total), corrected);
            total = sum;
        }
        float *dst = a.weights + b * a.w_stride + row;
        const bool mine = row < min(len, a.width);
        if (RES) {
            if (group == 1) sums[lane_row] = total;
            named_bar_sync(3, 256);
            if (group == 0) {
                total += sums[lane_row];
                if (mine) *dst = a.accumulate ? *dst + total : total;
            }
            named_bar_sync(3, 256);
        } else if (((n_blocks - 1) & 1) == static_cast<uint32_t>(group) && mine) {
            *dst = a.accumulate ? *dst + total : total;
        }
    }
}

template <bool RES, int N>
__global__ void __launch_bounds__(kThreads, 1) row_weights_kernel(const __grid_constant__ WeightsArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using L = Smem<RES, N>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kMisc);
    const uint32_t bars = smem_u32(smem + L::kBars);
    if ((smem_u32(smem) & 1023u) != 0u) {
        if (tid == 0) atomicOr(a.status, kStatusSmemLayout);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(bars + (L::kBarFull + i) * 8, 1);
            mbar_init(bars + (L::kBarEmpty + i) * 8, 1);
        }
        for (int i = 0; i < L::kResident; ++i) {
            mbar_init(bars + (L::kBarKFull + i) * 8, 1);
            mbar_init(bars + (L::kBarKEmpty + i) * 8, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars + (L::kBarS + i) * 8, 1);
            mbar_init(bars + (L::kBarSFree + i) * 8, 1);
        }
        for (int i = 0; i < kRecords; ++i) {
            mbar_init(bars + (L::kBarRecFull + i) * 8, 1);
            mbar_init(bars + (L::kBarRecEmpty + i) * 8, 9);
        }
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 8) tmem_alloc(smem_u32(smem + L::kMisc + 8), L::kTmemCols);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::kMisc + 8);
    if (warp < 8) {
        sum_role<RES, N>(a, smem, tmem, abort_flag, warp, lane);
    } else if (warp == 8) {
        mma_role<RES, N>(a, smem, tmem, abort_flag, lane);
    } else if (warp == 9) {
        loader_role<RES, N>(a, smem, abort_flag, lane);
    } else if (!a.accumulate) {
        // the two warps left over clear what lies behind the sequences, 1024 columns at a time
        const int pieces = (a.width + 1023) >> 10;
        for (long long x = blockIdx.x * 2 + (warp - 10); x < static_cast<long long>(pieces) * a.batch; x += 2 * gridDim.x) {
            const int b = static_cast<int>(x / pieces), c0 = static_cast<int>(x % pieces) << 10, n = rows_of(a, b);
            float *dst = a.weights + b * a.w_stride;
            for (int c = max(c0, n) + lane; c < min(c0 + 1024, a.width); c += 32) dst[c] = 0.0f;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 8) {
        tmem_relinquish();
        tmem_dealloc(tmem, L::kTmemCols);
    }
}

template <bool RES, int N>
int launch(WeightsArgs &a, unsigned grid, cudaStream_t stream) {
    static KernelSetup setup;
    const int rc = setup.get(reinterpret_cast<const void *>(&row_weights_kernel<RES, N>), Smem<RES, N>::kBytes, &a.status);
    if (rc != 0) return rc;
    row_weights_kernel<RES, N><<<grid, kThreads, Smem<RES, N>::kBytes, stream>>>(a);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace

int launch_row_weights(const smla_row_weights_params_t &p, int sm_count, cudaStream_t stream) {
    WeightsArgs a = {};
    a.columns = p.seqlen_q * p.num_heads;
    const uint32_t q_box = a.columns <= 16 ? 16 : a.columns <= 32 ? 32 : a.columns <= 64 ? 64 : 128;
    a.box_rows = 8;                              // rows of a tile that surely lie in one page
    while (a.box_rows < 128 && p.page_block_size % (a.box_rows * 2) == 0) a.box_rows *= 2;
    if (!make_slab_map(&a.q_map, false, p.q, p.head_dim, static_cast<uint64_t>(p.batch) * a.columns, 1, p.head_dim * 2,
                       static_cast<uint64_t>(p.head_dim) * 2 * p.batch * a.columns, q_box))
        return SMLA_EINVAL;
    a.max_blocks = p.max_blocks_per_seq;
    a.num_blocks = p.num_blocks;
    if (!make_slab_map(&a.k_map, false, p.k_cache, p.head_dim, p.page_block_size, p.num_blocks, p.k_row_stride, p.k_block_stride, a.box_rows))
        return SMLA_EINVAL;
    a.table = p.block_table;
    a.table_stride = p.block_table_stride;
    a.lens = p.cache_seqlens;
    a.lse = p.softmax_lse;
    a.weights = p.weights;
    a.w_stride = p.weights_stride;
    a.width = p.weights_width;
    a.accumulate = p.accumulate ? 1 : 0;
    a.batch = p.batch;
    a.s_q = p.seqlen_q;
    a.heads = p.num_heads;
    a.causal = p.causal ? 1 : 0;
    a.k_slabs = p.head_dim / 64;
    a.page = p.page_block_size;
    a.scale_log2 = p.softmax_scale * kLog2e;
    const int64_t rows = std::min<int64_t>(p.weights_width, static_cast<int64_t>(p.max_blocks_per_seq) * p.page_block_size);
    const int64_t tiles = std::max<int64_t>(1, (rows + 127) / 128) * p.batch;
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(tiles, sm_count));
    if (a.columns <= 16) return launch<false, 16>(a, grid, stream);
    if (a.columns <= 32) return launch<false, 32>(a, grid, stream);
    if (a.columns <= 64) return launch<false, 64>(a, grid, stream);
    if (a.columns <= 128) return launch<false, 128>(a, grid, stream);
    return launch<true, 256>(a, grid, stream);
}

}  // namespace smla
