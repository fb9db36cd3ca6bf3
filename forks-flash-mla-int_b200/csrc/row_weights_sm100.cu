// Attention weight of each cached row for sm_100a: w[b, r] = sum over query positions i and heads h that see row r of
// exp(scale q_bih . K_br - lse_bhi), over the paged bf16 latent cache of dense MLA decode.
//
// The (position, head) pairs of a sequence are columns c = i H + h of one matrix product: S^T = K Q^T with 128 cached
// rows as M (the lanes of tensor memory) and N columns.  A row's weight is then a sum along its own lane: no exchange
// between threads, and a fixed order (per block of columns, then block after block).  There is no running maximum: the
// lse is known, every term is at most 1.  Under the causal mask position i sees the rows r < len - (s_q - 1 - i), so a
// row is seen by the columns c >= max(0, r - len + s_q) H: one threshold per lane.
//
// Two forms, by the number of columns C = s_q H (both persistent):
//   C <= 128 (a decode step)  one CTA per SM, tiles of 128 rows in contiguous ranges.  Bound by reading the rows once.  K and Q
//            slabs [rows][64 dims] stream through one ring of stages; Q (N x 64 dims a stage) is fetched again for each tile,
//            from L2: N / 128 of the rows' bytes.  128 sequences of 4096 rows, 16 columns: 107 us, 5.7 TB/s of rows.
//   C > 128 (a window)        pairs of CTAs that multiply as one (M = 256, half of the columns in each CTA's shared memory).
//            The rows of a pair's tile stay in shared memory (147 KB each) while the columns pass in blocks of 256 through the
//            ring; the next tile's slabs replace the rows as the last block leaves them.  With scratch the blocks of all tiles
//            are dealt out evenly, and tiles that are cut are joined by a second kernel.  8192 columns, 28939 rows: 216 us, 1.26
//            PFLOP/s (single CTAs with blocks of 128: 254 us).  Bound by the feed of columns: each pair takes 295 KB a block
//            from L2, 6 TB/s over all.  (Eight stages of 8 KB in place of four of 16 KB: 5 % slower.)
// Roles (384 threads): warps 0-3 and 4-7 take turns at the score blocks (two accumulators), warp 8 issues the MMAs, warp
// 9 finds the tiles and loads.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cmath>
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
    float start, turn;                           // B and 8/3 B, see Smem
    // RES with scratch: the blocks of columns of all tiles are dealt out, and a tile that is cut leaves its sums here, 2 slots
    // of 128 per CTA (the end of a tile begun by a CTA before, the begin of one ended by a CTA behind), each with {sequence,
    // first row, first block, end block}
    float *part;
    int4 *desc;
    int *status;
};

// RES: the rows stay while the columns pass.  N: columns of a score block.
// A score is a sum over nine (eight) slabs of 64 dims in 36 steps.  The tensor pipe rounds a step's sum toward zero, always
// to the side where it makes the score smaller: 4e-6 of a weight whose score is 6.
// Up to 32 columns: tensor memory has room for an accumulator for each slab or two, which the sum warps add up with proper
// rounding; their signs vary (one sequence, 16 columns: 4.5e-6 -> 3e-7).
// More: a score starts at B (the scale's sign), and after half of its steps 8/3 B is taken off, so that it goes on from -5/3 B.
// B = 1.125 2^j, with 2^j times the scale between 8 and 16: for scores up to 7, which have the weight, the sum then stays
// between 2^j and 2^(j+1) in size, and the errors that a step's sum makes are the same in both halves on average, with opposite
// signs.  What is left of a score, 2.7e-6, varies from column to column and averages out in the sums (64 query positions of 128
// heads, all rows: 3.7e-6 -> 2.3e-7).  Not turned is what does not follow the sum's sign: a row that all queries look at, whose
// products have one sign, stays 1.2e-6 to 1.6e-6 too light (64 to 512 columns, scores of 2 to 7, directions of random components),
// 4e-6 where the components are all of one size.  Scores beyond 7 fare as without B.  Both offsets are products of their own, of
// constant operands: 38 steps for 36.
template <bool RES, int N>
struct Smem {
    static constexpr bool kBalanced = N >= 64;
    static constexpr int kPerGroup = N == 16 ? 1 : N == 32 ? 2 : 9;      // slabs of an accumulator
    static constexpr int kGroups = (9 + kPerGroup - 1) / kPerGroup;
    static constexpr int kQSlab = (RES ? N / 2 : N) * 128;               // a CTA of a pair has half of the columns
    static constexpr int kStage = RES ? kQSlab : kSlab + kQSlab;
    static constexpr int kStages = RES ? 4 : (208 * 1024 / kStage < 12 ? 208 * 1024 / kStage : 12);
    static constexpr int kResident = RES ? 9 : 0;
    static constexpr int kRingAt = kResident * kSlab;
    static constexpr int kOnes = kRingAt + kStages * kStage;             // kBalanced: [128 rows][16 dims], 1 in two dims of each row
    static constexpr int kStart = kOnes + (kBalanced ? 128 * 32 : 0);    // ... and as many columns as a slab of Q: start / 2 there
    static constexpr int kTurn = kStart + (kBalanced ? kQSlab / 4 : 0);  // ... -turn / 2 there
    static constexpr int kLse = kTurn + (kBalanced ? kQSlab / 4 : 0);    // two buffers of N floats
    static constexpr int kSums = kLse + 2 * N * 4;                       // RES: the second group's sums of a tile
    static constexpr int kBars = kSums + 128 * 4;
    static constexpr int kBarFull = 0, kBarEmpty = kStages, kBarKFull = 2 * kStages, kBarKEmpty = kBarKFull + kResident,
                         kBarS = kBarKEmpty + kResident, kBarSFree = kBarS + 2, kBarRecFull = kBarSFree + 2,
                         kBarRecEmpty = kBarRecFull + kRecords, kNumBars = kBarRecEmpty + kRecords;
    static constexpr int kRecs = kBars + kNumBars * 8;                   // {valid, sequence, first row, length, first block, end block}
    static constexpr int kMisc = kRecs + kRecords * 32;
    static constexpr int kBytes = kMisc + 16;
    static constexpr int kTmemCols = 512;
    static_assert(2 * N * kGroups <= kTmemCols, "two score blocks in tensor memory");
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
    // This CTA's (pair's) range of the tiles of all sequences, or of their blocks of columns.
    constexpr int kRows = RES ? 256 : 128;       // rows of a tile: 128 in each CTA
    const int blocks = RES ? (a.columns + N - 1) / N : 1, per_tile = RES && a.part != nullptr ? blocks : 1;
    long long total = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32)
        total += __reduce_add_sync(0xffffffffu, b0 + lane < a.batch ? (rows_of(a, b0 + lane) + kRows - 1) / kRows : 0);
    total *= per_tile;
    const unsigned team = RES ? blockIdx.x >> 1 : blockIdx.x, teams = RES ? gridDim.x >> 1 : gridDim.x;
    const int rank = RES ? static_cast<int>(cluster_rank()) : 0;
    const long long end = total * (team + 1) / teams;
    const int boxes = 128 / a.box_rows;
    if (RES && a.part != nullptr && lane < 2) a.desc[2 * blockIdx.x + lane] = make_int4(-1, 0, 0, 0);
    __syncwarp();
    long long base = 0;                          // tiles in front of the 32 sequences at b0
    int b0 = 0, rec_i = 0;
    uint32_t st = 0, tile_n = 0, k_loads = 0;
    bool ok = true;
    for (long long at_unit = total * team / teams; ok; ++rec_i) {
        int b = -1, t = 0;
        const long long idx = at_unit / per_tile;
        const int cb0 = static_cast<int>(at_unit - idx * per_tile);
        const int cb1 = per_tile == 1 ? blocks : static_cast<int>(min(static_cast<long long>(blocks), end - idx * per_tile));
        while (at_unit < end && b0 < a.batch) {
            const int n = b0 + lane < a.batch ? (rows_of(a, b0 + lane) + kRows - 1) / kRows : 0;
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
        at_unit = (idx + 1) * per_tile;
        const int slot = rec_i % kRecords;
        if (!(ok = mbar_wait(bars + (L::kBarRecEmpty + slot) * 8, ((rec_i / kRecords) & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
            int *rec = reinterpret_cast<int *>(smem + L::kRecs) + slot * 8;
            int len = 0;
            if (b >= 0) rows_of(a, b, &len);
            rec[0] = b >= 0;
            rec[1] = b;
            rec[2] = t * kRows + rank * 128;
            rec[3] = len;
            rec[4] = cb0;
            rec[5] = cb1;
            mbar_arrive(bars + (L::kBarRecFull + slot) * 8);
        }
        __syncwarp();
        if (b < 0) break;
        // the pages of the tile's boxes; one outside the table or the cache lies past the tensor's end: zeros
        int page = a.num_blocks, in_page = 0;
        if (lane < boxes) {
            const int row = t * kRows + rank * 128 + lane * a.box_rows, col = row / a.page;
            in_page = row - col * a.page;
            if (col < a.max_blocks) page = __ldg(a.table + b * a.table_stride + col);
            if (page < 0 || page > a.num_blocks) page = a.num_blocks;
        }
        const int q_row = b * a.columns;
        for (int cb = cb0; cb < cb1 && ok; ++cb) {
            for (int s = 0; s < a.k_slabs; ++s, ++st) {
                if (RES && cb == cb0) {
                    if (!(ok = mbar_wait(bars + (L::kBarKEmpty + s) * 8, (tile_n & 1) ^ 1, abort_flag))) break;
                    const uint32_t full = bars + (L::kBarKFull + s) * 8;
                    if (lane == 0 && rank == 0) mbar_arrive_expect_tx(full, 2 * kSlab);
                    __syncwarp();
                    if (lane < boxes)
                        tma_load_3d_pair(ks + s * kSlab + lane * a.box_rows * 128, &a.k_map, map_rank(full, 0), s * 64, in_page, page);
                    ++k_loads;
                }
                const uint32_t at = st % L::kStages, full = bars + (L::kBarFull + at) * 8, dst = ring + at * L::kStage;
                if (!(ok = mbar_wait(bars + (L::kBarEmpty + at) * 8, ((st / L::kStages) & 1) ^ 1, abort_flag))) break;
                if constexpr (RES) {
                    if (lane == 0) {
                        if (rank == 0) mbar_arrive_expect_tx(full, 2 * L::kStage);
                        tma_load_3d_pair(dst, &a.q_map, map_rank(full, 0), s * 64, q_row + cb * N + rank * (N / 2), 0);
                    }
                    __syncwarp();
                } else {
                    if (lane == 0) {
                        mbar_arrive_expect_tx(full, L::kStage);
                        tma_load_3d(dst + kSlab, &a.q_map, full, s * 64, q_row, 0);
                    }
                    __syncwarp();
                    if (lane < boxes) tma_load_3d(dst + lane * a.box_rows * 128, &a.k_map, full, s * 64, in_page, page);
                }
            }
        }
        if (ok) ++tile_n;
    }
    // What the products still signal to this CTA has to have come before it may end.
    for (uint32_t i = st > static_cast<uint32_t>(L::kStages) ? st - L::kStages : 0; ok && i < st; ++i)
        ok = mbar_wait(bars + (L::kBarEmpty + i % L::kStages) * 8, (i / L::kStages) & 1, abort_flag);
    if (RES && tile_n > 0)
        for (int s = 0; ok && s < a.k_slabs; ++s) ok = mbar_wait(bars + (L::kBarKEmpty + s) * 8, (tile_n - 1) & 1, abort_flag);
    if (!ok) {
        // The copies in flight have to land before the CTA may end.  Those of a pair are counted on the even CTA's barriers,
        // which wait for both CTAs' bytes; the odd one stays until the even one has seen them (cluster barrier at the end).
        if (lane == 0) give_up(abort_flag, a.status, kStatusGatherWait);
        __syncwarp();
        int never = 0;
        if (rank == 0) {
            for (uint32_t i = st > static_cast<uint32_t>(L::kStages) ? st - L::kStages : 0; i < st; ++i)
                mbar_wait(bars + (L::kBarFull + i % L::kStages) * 8, (i / L::kStages) & 1, &never);
            for (uint32_t i = k_loads > static_cast<uint32_t>(a.k_slabs) ? k_loads - a.k_slabs : 0; i < k_loads; ++i)
                mbar_wait(bars + (L::kBarKFull + i % a.k_slabs) * 8, (i / a.k_slabs) & 1, &never);
        }
    }
}

// ------------------------------------------------------------------ MMA issue
template <bool RES, int N>
__device__ __forceinline__ void mma_role(const WeightsArgs &a, uint8_t *smem, uint32_t tmem, volatile int *abort_flag, int lane) {
    using L = Smem<RES, N>;
    const uint32_t bars = smem_u32(smem + L::kBars), ring = smem_u32(smem + L::kRingAt);
    const uint32_t go = elect_one();
    constexpr uint32_t idesc = umma_idesc_bf16(RES ? 256 : 128, N, 0, 0);
    const auto multiply = [&](uint32_t d, uint64_t x, uint64_t y, uint32_t add) {
        if constexpr (RES) umma_ss_pair_pred(d, x, y, idesc, add, 1u);
        else umma_bf16_ss_pred(d, x, y, idesc, add, 1u);
    };
    const auto commit = [&](uint32_t bar) {
        if constexpr (RES) umma_commit_pair_pred(bar, go);
        else umma_commit_pred(bar, go);
    };
    const uint64_t kd = umma_desc_sw128(RES ? smem_u32(smem) : ring, 16), qd = umma_desc_sw128(ring + (RES ? 0 : kSlab), 16);
    // constant operands: all groups of 8 elements are alike
    const uint64_t ones = umma_desc(smem_u32(smem + L::kOnes), 128, 256), start = umma_desc(smem_u32(smem + L::kStart), 128, 256),
                   turn = umma_desc(smem_u32(smem + L::kTurn), 128, 256);
    uint32_t st = 0, n_blocks = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
        const int slot = it % kRecords;
        if (!(ok = mbar_wait(bars + (L::kBarRecFull + slot) * 8, (it / kRecords) & 1, abort_flag))) break;
        const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * 8;
        const int valid = rec[0], cb0 = rec[4], cb1 = rec[5];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) break;
        for (int cb = cb0; cb < cb1 && ok; ++cb, ++n_blocks) {
            const int buf = n_blocks & 1;
            const uint32_t s_free = bars + (L::kBarSFree + buf) * 8, s_phase = ((n_blocks >> 1) & 1) ^ 1;
            if (!(ok = mbar_wait(s_free, s_phase, abort_flag))) break;
            tc_fence_after_sync();
            const uint32_t d0 = tmem + buf * L::kGroups * N;
            if (L::kBalanced && go) multiply(d0, ones, start, 0u);
            for (int s = 0; s < a.k_slabs; ++s, ++st) {
                if (RES && cb == cb0 && !(ok = mbar_wait(bars + (L::kBarKFull + s) * 8, it & 1, abort_flag))) break;
                const uint32_t at = st % L::kStages;
                if (!(ok = mbar_wait(bars + (L::kBarFull + at) * 8, (st / L::kStages) & 1, abort_flag))) break;
                tc_fence_after_sync();
                const uint64_t ka = kd + static_cast<uint64_t>((RES ? s * kSlab : at * L::kStage) >> 4);
                const uint64_t qb = qd + static_cast<uint64_t>((at * L::kStage) >> 4);
                if (go) {
                    const uint32_t d = d0 + s / L::kPerGroup * N;
                    const int half = 2 * a.k_slabs - 4 * s;      // products of this slab before the turn, where it is among them
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (L::kBalanced && (k == 0 || k == 2) && half == k) multiply(d, ones, turn, 1u);
                        multiply(d, ka + 2 * k, qb + 2 * k, L::kBalanced || s % L::kPerGroup || k ? 1u : 0u);
                    }
                }
                commit(bars + (L::kBarEmpty + at) * 8);
                if (RES && cb + 1 == cb1) commit(bars + (L::kBarKEmpty + s) * 8);
            }
            if (ok) commit(bars + (L::kBarS + buf) * 8);
        }
    }
    if (!ok && lane == 0) give_up(abort_flag, a.status, kStatusMmaWait);
}

// ------------------------------------------------------------------ sums
// Sum of exp2((s + offset) c - lse2) over kCols columns of this lane, each the sum of `groups` accumulators N columns apart; with
// MASK only the columns in [lo, hi).
template <int kCols, int N, int kGroups, bool MASK>
__device__ __forceinline__ void add_columns(uint32_t taddr, int groups, const float *lse2, float c, float offset, int lo, int hi,
                                            uint64_t (&acc)[4]) {
    uint32_t s[kCols];
    const auto load = [](uint32_t at, uint32_t (&r)[kCols]) {
        if constexpr (kCols == 32) {
            tmem_ld_x32_nowait(at, r);
            tmem_ld_wait();
        } else {
            tmem_ld_x16(at, r);
        }
    };
    load(taddr, s);
    if constexpr (kGroups > 1) {
#pragma unroll 1
        for (int g = 1; g < groups; ++g) {
            uint32_t x[kCols];
            load(taddr + g * N, x);
#pragma unroll
            for (int j = 0; j < kCols; ++j) s[j] = __float_as_uint(__uint_as_float(s[j]) + __uint_as_float(x[j]));
        }
    }
    const uint64_t c2 = pack2(c, c), offset2 = pack2(offset, offset);
    const auto score = [&](int j) {
        const uint64_t v = pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1]));
        return kGroups == 1 ? add2(v, offset2) : v;
    };
#pragma unroll
    for (int j = 0; j < kCols; j += 4) {
        const float4 z = *reinterpret_cast<const float4 *>(lse2 + j);    // negated
        float x[4];
        unpack2(fma2(score(j), c2, pack2(z.x, z.y)), x[0], x[1]);
        unpack2(fma2(score(j + 2), c2, pack2(z.z, z.w)), x[2], x[3]);
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
    const uint32_t t_addr = tmem + group * N * L::kGroups + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int blocks = RES ? (a.columns + N - 1) / N : 1, groups = (a.k_slabs + L::kPerGroup - 1) / L::kPerGroup;
    const float offset = a.turn - a.start;       // exact
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
        const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * 8;
        const int valid = rec[0], b = rec[1], rec_row = rec[2], row = rec_row + lane_row, len = rec[3], cb0 = rec[4], cb1 = rec[5];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) return;
        // columns below `from` do not see this row; the warp's last row sees the fewest
        const int from = a.causal ? max(0, row - len + a.s_q) * a.heads : 0;
        const int from_warp = a.causal ? max(0, row - lane + 31 - len + a.s_q) * a.heads : 0;
        float total = 0.0f, lost = 0.0f;         // compensated sum over the blocks
        for (int cb = cb0; cb < cb1; ++cb, ++n_blocks) {
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
                for (int j = 0; j < N; j += kCols) add_columns<kCols, N, L::kGroups, false>(t_addr + j, groups, lse2 + j, a.scale_log2, offset, 0, 0, acc);
            } else {
                // columns of the block that count for this row (those past the last hold other queries' scores)
                const int lo = from - c0, hi = a.columns - c0;
                for (int j = 0; j < N; j += kCols) add_columns<kCols, N, L::kGroups, true>(t_addr + j, groups, lse2 + j, a.scale_log2, offset, lo - j, hi - j, acc);
            }
            tc_fence_before_sync();
            named_bar_sync(1 + group, 128);      // the scores and the lse buffer have been read
            if ((warp & 3) == 0 && lane == 0) {
                const uint32_t s_free = bars + (L::kBarSFree + group) * 8;
                if constexpr (RES) mbar_arrive_remote(map_rank(s_free, 0));      // the even CTA issues for both
                else mbar_arrive(s_free);
            }
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
                if (cb0 == 0 && cb1 == blocks) {
                    if (mine) *dst = a.accumulate ? *dst + total : total;
                } else {
                    const int place = 2 * blockIdx.x + (cb0 == 0 ? 1 : 0);
                    a.part[place * 128 + lane_row] = total;
                    if (lane_row == 0) a.desc[place] = make_int4(b, rec_row, cb0, cb1);
                }
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
    const bool issues = !RES || cluster_rank() == 0;         // the products of a pair are issued by its even CTA
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
            mbar_init(bars + (L::kBarSFree + i) * 8, RES ? 2 : 1);
        }
        for (int i = 0; i < kRecords; ++i) {
            mbar_init(bars + (L::kBarRecFull + i) * 8, 1);
            mbar_init(bars + (L::kBarRecEmpty + i) * 8, issues ? 9 : 8);
        }
        *abort_flag = 0;
        mbar_init_fence();
    }
    if constexpr (L::kBalanced) {
        const uint32_t half = __float_as_uint(0.5f * a.start) >> 16, minus = __float_as_uint(-0.5f * a.turn) >> 16;   // exact in bf16
        for (int x = L::kOnes + tid * 16; x < L::kLse; x += kThreads * 16)
            *reinterpret_cast<uint4 *>(smem + x) = make_uint4(x < L::kStart ? 0x3F80u : x < L::kTurn ? half : minus, 0, 0, 0);
        fence_async_smem();
    }
    if (warp == 8) {
        if constexpr (RES) tmem_alloc_pair(smem_u32(smem + L::kMisc + 8), L::kTmemCols);
        else tmem_alloc(smem_u32(smem + L::kMisc + 8), L::kTmemCols);
    }
    tc_fence_before_sync();
    if constexpr (RES) cluster_sync_all();       // also: the other CTA's barriers are there
    else __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::kMisc + 8);
    if (warp < 8) {
        sum_role<RES, N>(a, smem, tmem, abort_flag, warp, lane);
    } else if (warp == 8) {
        if (issues) mma_role<RES, N>(a, smem, tmem, abort_flag, lane);
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
    __syncwarp();
    if constexpr (RES) cluster_sync_all();       // nothing of this CTA's is used by the other any more
    else __syncthreads();
    if (warp == 8) {
        if constexpr (RES) {
            tmem_free_pair(tmem, L::kTmemCols);
        } else {
            tmem_relinquish();
            tmem_dealloc(tmem, L::kTmemCols);
        }
    }
}

// The tiles that were cut: the block of the CTA that has a tile's first columns adds up its pieces, in the order of the CTAs.
__global__ void __launch_bounds__(128) row_weights_join_kernel(const WeightsArgs a, int blocks, int ctas) {
    const int4 d = a.desc[2 * blockIdx.x + 1];
    if (d.x < 0) return;
    float total = a.part[(2 * blockIdx.x + 1) * 128 + threadIdx.x];
    int end = d.w;
    for (int c = blockIdx.x + 2; end < blocks && c < ctas; c += 2) {     // the same half of the next pair
        const int4 e = a.desc[2 * c];
        if (e.x < 0) continue;                   // a CTA without a share
        if (e.x != d.x || e.y != d.y || e.z != end) break;
        total += a.part[2 * c * 128 + threadIdx.x];
        end = e.w;
    }
    const int row = d.y + threadIdx.x;
    if (row >= rows_of(a, d.x)) return;
    float *dst = a.weights + d.x * a.w_stride + row;
    *dst = a.accumulate ? *dst + total : total;
}

template <bool RES, int N>
int launch(WeightsArgs &a, unsigned grid, cudaStream_t stream) {
    static KernelSetup setup;
    const int rc = setup.get(reinterpret_cast<const void *>(&row_weights_kernel<RES, N>), Smem<RES, N>::kBytes, &a.status);
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<RES, N>::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = RES ? 2 : 1;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = RES ? 1 : 0;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, row_weights_kernel<RES, N>, a));
}

}  // namespace

size_t row_weights_workspace(int seqlen_q, int num_heads, int sm_count) {
    return static_cast<int64_t>(seqlen_q) * num_heads <= 128 ? 0 : static_cast<size_t>(sm_count) * 2 * (128 * sizeof(float) + sizeof(int4));
}

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
    const float range = 8.0f / std::fabs(p.softmax_scale);
    if (range > 0.0f && range < INFINITY) {      // a scale of 0, or one as good as that, needs no offsets
        const float base = std::ldexp(1.0f, std::min(100, std::max(-100, static_cast<int>(std::ceil(std::log2(range))))));
        a.start = std::copysign(1.125f * base, p.softmax_scale);
        a.turn = std::copysign(3.0f * base, p.softmax_scale);
    }
    const int64_t rows = std::min<int64_t>(p.weights_width, static_cast<int64_t>(p.max_blocks_per_seq) * p.page_block_size);
    const int64_t tiles = std::max<int64_t>(1, (rows + 127) / 128) * p.batch;
    if (a.columns > 128) {
        // With scratch every SM gets a share, down to a block of columns; else whole tiles are dealt out.
        const int blocks = (a.columns + 255) / 256;
        const int64_t pair_tiles = std::max<int64_t>(1, (rows + 255) / 256) * p.batch;
        int64_t grid = 2 * std::min<int64_t>(pair_tiles, sm_count / 2);
        const bool split = p.workspace != nullptr && p.workspace_bytes >= row_weights_workspace(p.seqlen_q, p.num_heads, sm_count);
        if (split) {
            if (reinterpret_cast<uintptr_t>(p.workspace) & 15u) return SMLA_EALIGN;
            grid = 2 * std::min<int64_t>(pair_tiles * blocks, sm_count / 2);
            a.desc = static_cast<int4 *>(p.workspace);
            a.part = reinterpret_cast<float *>(a.desc + 2 * grid);
        }
        const int rc = launch<true, 256>(a, static_cast<unsigned>(grid), stream);
        if (rc != 0 || !split) return rc;
        row_weights_join_kernel<<<static_cast<unsigned>(grid), 128, 0, stream>>>(a, blocks, static_cast<int>(grid));
        return static_cast<int>(cudaGetLastError());
    }
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(tiles, sm_count));
    if (a.columns <= 16) return launch<false, 16>(a, grid, stream);
    if (a.columns <= 32) return launch<false, 32>(a, grid, stream);
    if (a.columns <= 64) return launch<false, 64>(a, grid, stream);
    return launch<false, 128>(a, grid, stream);
}

}  // namespace smla
