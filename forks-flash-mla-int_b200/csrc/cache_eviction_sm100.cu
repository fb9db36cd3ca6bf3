// Choice of the rows of a sequence that stay in its cache, and their move to the front, for sm_100a.
//
// Selection.  Weights become 32-bit keys that order as they do (sign folded, -0 made 0, NaN made the lowest).
// Four passes of eight bits find the key T of the row that is last among the heaviest: a pass counts the
// digits of the keys that agree with T so far and takes the digit at which the count from above reaches the
// rows still wanted (and stops where a digit's rows are wanted all).  Rows above T stay, rows equal to T stay from
// the lowest on until the budget is full, and all are written in row order by counting from the front.
// Counts are integers, so nothing depends on the order of the atomics.
//
// A cluster of CTAs takes a sequence.  Each holds its part of the keys in shared memory, so the weights are read
// once, and the counts of a pass are added up through distributed shared memory.  What bounds it is latency: the
// passes (two to four), each a count, a cluster barrier and a search, one after the other, and in the first one adds that
// wait for one another: the top eight bits of a key are the sign and seven bits of the exponent, of which such sums have a handful
// (and zeros), so many lanes of a warp add to one word.  64 sequences of 32768 rows, two
// CTAs each: 19 us, of which reading the weights (8 MB) would be 1.3; of 15 in the kernel the first pass takes 4, the second 3,
// counting what stays 1.6 and writing it 4.5.  Four sequences of 2048 rows: 8 us back to back, 4 of them in the kernel.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>

#include "smla_internal.h"
#include "tensor_map.h"

namespace smla {
namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kMaxKeys = 48 * 1024;              // keys a CTA holds (192 KB); the rest is read again in each pass

__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);            // -0 + 0 = 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// The weight of a key that is neither a zero's nor a NaN's.
__device__ __forceinline__ float key_weight(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

__global__ void __launch_bounds__(kSelThreads, 1) select_rows_kernel(const float *weights, int64_t stride, int width, const int32_t *lens,
                                                                     int budget, int recent, int held, int32_t *rows, int32_t *kept,
                                                                     float *kept_weights, int64_t kept_stride, int kept_width) {
    extern __shared__ __align__(16) uint32_t keys[];         // `held` of this CTA's keys, a multiple of 4
    __shared__ unsigned hist[2][256];
    __shared__ unsigned total[256];              // digit d at (255 - d) % 8 * 32 + (255 - d) / 8
    __shared__ int s_digit, s_left, s_all;
    __shared__ int s_warp[2][kSelWarps];
    __shared__ int s_sum[2];                     // this CTA's rows above T, and equal to it
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int b = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = min(max(lens[b], 0), width), stay = min(len, budget);
    const float *w = weights + b * stride;
    rows += static_cast<int64_t>(b) * budget;
    if (kept_weights) kept_weights += b * kept_stride;
    const int all = rank * kSelThreads + tid, step = ranks * kSelThreads;
    if (all == 0) kept[b] = stay;
    // (a budget, a width or a length may be up to 2^31 - 1, so what is counted up to them in steps is 64 bits wide)
    for (int64_t j = static_cast<int64_t>(stay) + all; j < budget; j += step) rows[j] = -1;
    if (kept_weights)
        for (int64_t j = static_cast<int64_t>(stay) + all; j < kept_width; j += step) kept_weights[j] = 0.0f;
    const int old = len - recent, want0 = budget - recent;   // of the `old` first rows `want0` stay
    const bool whole = len <= budget;
    if (whole || want0 == 0) {                   // (the whole cluster takes the same way)
        const int first = whole ? 0 : old;
        for (int64_t j = all; j < stay; j += step) {
            rows[j] = static_cast<int>(first + j);
            if (kept_weights) kept_weights[j] = w[first + j];
        }
        return;
    }
    // this CTA's part: whole multiples of 32 rows, in rank order
    const int part = ((old - 1) / ranks + 32) & ~31;
    const int lo = min(rank * part, old), n = min(part, old - lo);
    const float *mine = w + lo;
    const auto key_at = [&](int j) { return j < held ? keys[j] : weight_key(__ldg(mine + j)); };
    if (tid < 256) hist[0][tid] = hist[1][tid] = 0;
    __syncthreads();
    unsigned prefix = 0, want = want0;
    int shift = 24;
    for (int pass = 0;; ++pass, shift -= 8) {
        unsigned *h = hist[pass & 1];
        if (pass == 0) {
#pragma unroll 8
            for (int j = tid; j < n; j += kSelThreads) {
                const uint32_t k = weight_key(__ldg(mine + j));
                if (j < held) keys[j] = k;
                atomicAdd(&h[k >> 24], 1u);
            }
        } else {
            const auto count = [&](uint32_t k) {
                if ((k >> (shift + 8)) == prefix) atomicAdd(&h[(k >> shift) & 255], 1u);
            };
            const int there = min(n, held) & ~3;
#pragma unroll 2
            for (int j = tid * 4; j < there; j += kSelThreads * 4) {
                const uint4 k = *reinterpret_cast<const uint4 *>(keys + j);
                count(k.x);
                count(k.y);
                count(k.z);
                count(k.w);
            }
            for (int j = there + tid; j < n; j += kSelThreads) count(key_at(j));
        }
        if (ranks > 1) cluster.sync();
        else __syncthreads();
        if (tid < 256) {
            unsigned sum = 0;
            for (int r = 0; r < ranks; ++r) sum += *cluster.map_shared_rank(&h[tid], r);
            total[((255 - tid) & 7) * 32 + ((255 - tid) >> 3)] = sum;
            hist[(pass & 1) ^ 1][tid] = 0;       // the other ranks have read it: they are past this pass's barrier
        }
        __syncthreads();
        if (warp == 0) {
            // lane l has the digits 255 - 8 l down to 248 - 8 l; `above`: rows with larger digits than those
            unsigned c[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += c[e] = total[e * 32 + lane];
            unsigned upto = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const unsigned x = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += x;
            }
            unsigned above = upto - sum;
            if (above < want && want <= upto) {  // one lane: the counts add up to at least `want`
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (above < want && want <= above + c[e]) {
                        s_digit = 255 - 8 * lane - e;
                        s_left = static_cast<int>(want - above);
                        s_all = want - above == c[e];
                    }
                    above += c[e];
                }
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | static_cast<unsigned>(s_digit);
        want = static_cast<unsigned>(s_left);
        if (shift == 0 || s_all) break;
    }
    // Rows whose key, without the bits not looked at, is above the prefix stay, and the first `want` that equal it: keys above
    // `high`, and those from `low` on.  A warp takes consecutive rows.
    const uint32_t low = prefix << shift, high = low | ((1u << shift) - 1u);
    const int warp_part = ((n + kSelWarps - 1) / kSelWarps + 127) & ~127;
    const int w_lo = min(warp * warp_part, n), w_hi = min(w_lo + warp_part, n), w_held = min(w_hi, held);
    int above = 0, equal = 0;
    int j_rest = w_lo;
    for (; j_rest + 128 <= w_held; j_rest += 128) {
        const uint4 k = *reinterpret_cast<const uint4 *>(keys + j_rest + lane * 4);
        above += (k.x > high) + (k.y > high) + (k.z > high) + (k.w > high);
        equal += (k.x >= low) + (k.y >= low) + (k.z >= low) + (k.w >= low);
    }
    for (int j = j_rest + lane; j < w_hi; j += 32) {
        const uint32_t k = key_at(j);
        above += k > high;
        equal += k >= low;
    }
    equal -= above;
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) {
        s_warp[0][warp] = above;
        s_warp[1][warp] = equal;
    }
    __syncthreads();
    if (warp == 0) {
        const int a = s_warp[0][lane], t = s_warp[1][lane];
        int ua = a, ut = t;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, ua, d), y = __shfl_up_sync(0xffffffffu, ut, d);
            if (lane >= d) {
                ua += x;
                ut += y;
            }
        }
        s_warp[0][lane] = ua - a;
        s_warp[1][lane] = ut - t;
        if (lane == 31) {
            s_sum[0] = ua;
            s_sum[1] = ut;
        }
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    above = s_warp[0][warp];
    equal = s_warp[1][warp];
    for (int r = 0; r < rank; ++r) {
        above += *cluster.map_shared_rank(&s_sum[0], r);
        equal += *cluster.map_shared_rank(&s_sum[1], r);
    }
    const int ties = static_cast<int>(want);
    const unsigned before = (1u << lane) - 1u;
    for (int j0 = w_lo; j0 < w_hi; j0 += 128) {
        uint32_t k[4];
        unsigned up[4], tie[4];                  // lanes with a row above, equal
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = j0 + e * 32 + lane;
            const bool there = j < w_hi;
            k[e] = j < w_held ? keys[j] : there ? key_at(j) : 0u;
            up[e] = __ballot_sync(0xffffffffu, k[e] > high);
            tie[e] = __ballot_sync(0xffffffffu, there && k[e] >= low) & ~up[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int t = equal;
            bool stays = k[e] > high;
            if (tie[e]) {
                t += __popc(tie[e] & before);
                stays |= ((tie[e] >> lane) & 1u) && t < ties;
                equal += __popc(tie[e]);
            }
            if (stays) {
                const int at = above + __popc(up[e] & before) + min(t, ties), j = j0 + e * 32 + lane;
                rows[at] = lo + j;
                // out of the key: reading it again costs the latency of memory
                if (kept_weights) kept_weights[at] = k[e] == 0u || k[e] == 0x80000000u ? __ldg(mine + j) : key_weight(k[e]);
            }
            above += __popc(up[e]);
        }
    }
    for (int64_t j = all; j < recent; j += step) {
        rows[want0 + j] = static_cast<int>(old + j);
        if (kept_weights) kept_weights[want0 + j] = w[old + j];
    }
    if (ranks > 1) cluster.sync();               // no CTA may end while another reads its sums
}

// ------------------------------------------------------------------ move
__device__ __forceinline__ const uint8_t *row_at(const smla_compact_params_t &p, const int32_t *table, int columns, int row) {
    const int col = row / p.page_block_size;
    if (row < 0 || col >= columns) return nullptr;
    const int page = __ldg(table + col);
    if (page < 0 || page >= p.num_blocks) return nullptr;
    return static_cast<const uint8_t *>(p.cache) + page * p.block_stride + (row - col * p.page_block_size) * p.row_stride;
}

// This block's sequence; the grid's last two dimensions count them.
__device__ __forceinline__ int sequence_of_block() { return static_cast<int>(blockIdx.z * gridDim.y + blockIdx.y); }
dim3 sequence_grid(int64_t blocks, int batch) {
    constexpr int most = 65535;
    return dim3(static_cast<unsigned>(blocks), std::min(batch, most), (batch - 1) / most + 1);
}

// Rows of sequence b that have a place to go to.
__device__ __forceinline__ int rows_to_move(const smla_compact_params_t &p, int b) {
    const int64_t places = static_cast<int64_t>(p.out_max_blocks_per_seq) * p.page_block_size;
    return static_cast<int>(min(static_cast<int64_t>(min(max(__ldg(p.kept + b), 0), p.budget)), places));
}

// Inside their own pages: a CTA takes 64 bytes of all rows of a sequence (slices of a row do not touch one another) and
// moves 512 rows at a time, all their loads in front of all their stores.  A row's source index is at least its target's,
// so what a later turn reads has not been written yet.  Bound by the latency of a turn, three loads that depend on one another
// and two barriers: 16 sequences x 4096 rows 55 us, one of 32768 rows 276 us (18 CTAs, 64 turns).
constexpr int kSlice = 64, kTurnRows = 512;
template <int THREADS>
__device__ __forceinline__ void move_slice_in_place(const smla_compact_params_t &p, int b, int n, int slice) {
    constexpr int kStep = THREADS / (kSlice / 16), kPieces = kTurnRows / kStep;
    const int at = slice * kSlice + (threadIdx.x % (kSlice / 16)) * 16;
    const int32_t *rows = p.rows + static_cast<int64_t>(b) * p.budget, *table = p.block_table + b * p.block_table_stride,
                  *out_table = p.out_block_table + b * p.out_block_table_stride;
    for (int64_t j0 = 0; j0 < n; j0 += kTurnRows) {            // (n may be near 2^31)
        uint4 x[kPieces];
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
            const int64_t j = j0 + e * kStep + threadIdx.x / (kSlice / 16);
            x[e] = make_uint4(0, 0, 0, 0);
            if (j < n && at < p.row_bytes) {
                const uint8_t *src = row_at(p, table, p.max_blocks_per_seq, __ldg(rows + j));
                if (src) x[e] = *reinterpret_cast<const uint4 *>(src + at);
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
            const int64_t j = j0 + e * kStep + threadIdx.x / (kSlice / 16);
            if (j < n && at < p.row_bytes) {
                uint8_t *dst = const_cast<uint8_t *>(row_at(p, out_table, p.out_max_blocks_per_seq, static_cast<int>(j)));
                if (dst) *reinterpret_cast<uint4 *>(dst + at) = x[e];
            }
        }
        __syncthreads();                         // the next turn's loads come behind these stores of the whole CTA
    }
}

constexpr int kSliceThreads = 512;
__global__ void __launch_bounds__(kSliceThreads) move_rows_in_place_kernel(const smla_compact_params_t p) {
    const int b = sequence_of_block();
    if (b < p.batch) move_slice_in_place<kSliceThreads>(p, b, rows_to_move(p, b), blockIdx.x);
}

// To other pages: a warp takes four rows, works out their addresses once and has all their pieces in flight together (three
// of 16 bytes a lane and row: 1152 bytes are 2.25).  Bound by HBM, 2 x row_bytes a row: 16 sequences x 4096 rows 29 us, 5.2 TB/s.
// A sequence whose target table names some of the source's pages in their own place (a copy of the table, or a table that
// goes on with new pages) moves in place there: its rows are taken in order, by the first CTAs.
constexpr int kMoveWarps = 8, kMoveRows = 4, kMoveTurn = 3;
__global__ void __launch_bounds__(kMoveWarps * 32) move_rows_kernel(const smla_compact_params_t p) {
    const int b = sequence_of_block(), lane = threadIdx.x & 31, slices = (p.row_bytes + kSlice - 1) / kSlice;
    if (b >= p.batch) return;
    const int32_t *table = p.block_table + b * p.block_table_stride, *out_table = p.out_block_table + b * p.out_block_table_stride;
    // the first pages are compared while the count of rows is on its way
    const int places = min(min(p.max_blocks_per_seq, p.out_max_blocks_per_seq), (p.budget - 1) / p.page_block_size + 1);
    const auto same_page = [&](int c) {
        const int page = __ldg(out_table + c);
        return page == __ldg(table + c) && page >= 0 && page < p.num_blocks;
    };
    bool own = static_cast<int>(threadIdx.x) < places && same_page(threadIdx.x);
    const int n = rows_to_move(p, b), j0 = (blockIdx.x * kMoveWarps + (threadIdx.x >> 5)) * kMoveRows;
    if (n == 0 || (blockIdx.x >= slices && blockIdx.x * static_cast<int64_t>(kMoveWarps * kMoveRows) >= n)) return;
    const uint8_t *src = nullptr;
    uint8_t *dst = nullptr;
    if (lane < kMoveRows && j0 < n && j0 + lane < n) {
        const int row = __ldg(p.rows + static_cast<int64_t>(b) * p.budget + j0 + lane);
        src = row_at(p, table, p.max_blocks_per_seq, row);
        dst = const_cast<uint8_t *>(row_at(p, out_table, p.out_max_blocks_per_seq, j0 + lane));
    }
    const int columns = min(places, (n - 1) / p.page_block_size + 1);
    own &= static_cast<int>(threadIdx.x) < columns;
    for (int c = threadIdx.x + kMoveWarps * 32; c < columns; c += kMoveWarps * 32) own |= same_page(c);
    const uint8_t *from[kMoveRows];
    uint8_t *to[kMoveRows];
#pragma unroll
    for (int r = 0; r < kMoveRows; ++r) {
        from[r] = reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), r));
        to[r] = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
    }
    uint4 x[kMoveRows][kMoveTurn];
    const auto load = [&](int at) {
#pragma unroll
        for (int r = 0; r < kMoveRows; ++r)
#pragma unroll
            for (int e = 0; e < kMoveTurn; ++e) {
                x[r][e] = make_uint4(0, 0, 0, 0);
                if (from[r] && at + e * 512 < p.row_bytes) x[r][e] = __ldcs(reinterpret_cast<const uint4 *>(from[r] + at + e * 512));
            }
    };
    load(lane * 16);                             // in flight while the CTA learns whether they may be stored
    if (__syncthreads_or(own)) {
        if (blockIdx.x < slices) move_slice_in_place<kMoveWarps * 32>(p, b, n, blockIdx.x);
        return;
    }
    for (int at = lane * 16; at < p.row_bytes;) {
#pragma unroll
        for (int r = 0; r < kMoveRows; ++r)
#pragma unroll
            for (int e = 0; e < kMoveTurn; ++e)
                if (to[r] && at + e * 512 < p.row_bytes) *reinterpret_cast<uint4 *>(to[r] + at + e * 512) = x[r][e];
        at += kMoveTurn * 512;
        if (at < p.row_bytes) load(at);
    }
}

}  // namespace

int launch_select_rows(const float *weights, int64_t weights_stride, int width, const int32_t *lens, int batch, int budget,
                       int recent, int32_t *rows, int32_t *kept, float *kept_weights, int64_t kept_stride, int kept_width, int sm_count,
                       cudaStream_t stream) {
    // As many CTAs to a sequence as leave each at least 4096 rows and do not ask for more than one per SM (up to 8, the
    // portable cluster size); more than 8 x 48 K rows are partly read from L2 in each pass.
    int ranks = 1;
    while (ranks < 8 && width / (ranks * 2) >= 4096 && static_cast<int64_t>(batch) * ranks * 2 <= sm_count) ranks *= 2;
    while (ranks < 8 && width / ranks > kMaxKeys) ranks *= 2;
    const int part = (std::max(width - 1, 0) / ranks + 32) & ~31, held = std::min(part, kMaxKeys);
    if (static_cast<int64_t>(batch) * ranks > 0x7FFFFFFFLL) return SMLA_ETOOBIG;
    static KernelSetup setup;
    int *status;                                 // (this kernel waits for nothing that could fail to come)
    const int rc = setup.get(reinterpret_cast<const void *>(&select_rows_kernel), kMaxKeys * 4, &status);
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(batch) * ranks);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(held) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(ranks);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, select_rows_kernel, weights, weights_stride, width, lens, budget, recent, held, rows, kept, kept_weights,
                                               kept_stride, kept_width));
}

int launch_compact(const smla_compact_params_t &p, cudaStream_t stream) {
    if (p.out_block_table == p.block_table && (p.batch <= 1 || p.out_block_table_stride == p.block_table_stride)) {
        move_rows_in_place_kernel<<<sequence_grid((p.row_bytes + kSlice - 1) / kSlice, p.batch), kSliceThreads, 0, stream>>>(p);
    } else {
        constexpr int per_block = kMoveWarps * kMoveRows;
        const int64_t blocks = std::max<int64_t>((static_cast<int64_t>(p.budget) + per_block - 1) / per_block, (p.row_bytes + kSlice - 1) / kSlice);
        move_rows_kernel<<<sequence_grid(blocks, p.batch), kMoveWarps * 32, 0, stream>>>(p);
    }
    return static_cast<int>(cudaGetLastError());
}

}  // namespace smla
