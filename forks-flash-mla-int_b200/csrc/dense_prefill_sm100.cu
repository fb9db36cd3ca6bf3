// Dense MLA prefill for sm_100a: attention of packed prompts over keys and values expanded to heads.
//
//   s_ij = scale q_i . k_j   (j < nk - (nq - 1 - i) with the causal mask),   lse_i = log sum_j exp s_ij,
//   out_i = sum_j exp(s_ij - lse_i) v_j
//
// One pass over the keys with a running reference m and sum l of the softmax: weights are exp(s - m), and where the
// reference moves from m to m', l and the accumulated output are scaled by exp(m - m').  The reference need not be the
// maximum, only near it: it moves when a score exceeds it by more than 2^8 in weight, so on ordinary data it moves in
// the first block of keys and hardly ever again.  Weights are rounded to the input type for the second product (the
// tensor pipe multiplies 16-bit operands); the sum l takes them unrounded, in fp32.
//
// Work is cut into items: 256 query rows of one head, for a pair of CTAs (a cluster, persistent) that multiplies as one
// with M = 256: each CTA has 128 of the rows, in the lanes of its tensor memory, and half of every key block.  The items'
// key blocks of 128 form one sequence of tiles that runs on across items:
//   S(g) = Q K(g)^T  -> one of three buffers of 128 columns in tensor memory
//   P(g) = exp(S(g) - m)  -> 16-bit, written over S(g) (64 columns)
//   O += P(g) V(g)  -> 128 columns
// Three tiles are scored ahead of the output, so the weights of a tile have the time of two tiles' products to be computed
// in, and two warpgroups take turns at the tiles: a weight computation (about 2100 cycles for a tile, one row per thread)
// may take nearly twice as long as the products of a tile (1280 cycles at 192 dims).
// What bounds it: tensor work, at 91 % while a long item runs (1280 of 1400 cycles a tile: the chain weights - output - score of the
// tile three on takes a little longer than three tiles' products), and the power limit in long runs.  From item to item the
// output takes about 4000 cycles (last product, read, first product), of which half is hidden: two tiles an item.  8192 causal tokens of 37
// heads: 573 to 616 us with 192 dims, from GPU to GPU (1.39 to 1.29 PFLOP/s), 502 to 541 us with 128 (1.27 to 1.18).  Measured
// against the former: one CTA per item, S in one buffer
// for each half of the rows, 675 and 580 us; weights in buffers of their own beside S (a fourth wait and narrower stores)
// 660 and 587; weights handed over in two pieces 602 and 530; the rows' reference through mbarriers in place of named ones
// 600 and 542; the output written by the softmax warpgroup that had the last tile 577 and 509.
// K and V arrive by TMA as slabs of 64 dims with the 128-byte swizzle: of K the rows of 64 keys (its half of N), of V all
// 128 keys of 64 of the dims (its half of N there).  A slab read K-major gives K for the first product, MN-major V for the
// second.  Sharing B halves the fills: with both operands from shared memory one CTA's products alone (M = N = 128) take all
// of its 128 bytes a cycle.
//
// Roles (512 threads): warps 0-3 and 4-7 are the two softmax warpgroups, warp 8 (of the even CTA) issues the products, warp 9
// finds the items and loads Q and K, warp 10 loads V, warps 12-15 write the output.  Item records go through a ring of four in shared memory.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "smla_internal.h"
#include "tensor_map.h"

namespace smla {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kThreads = 512;
constexpr int kSlab = 128 * 128;                 // bytes of [128 rows][64 dims] of 16-bit elements
constexpr int kHalfSlab = kSlab / 2;             // [64 rows][64 dims]
constexpr int kRecords = 4;
constexpr int kRecInts = 12;
constexpr int kBuffers = 3;                      // of S
constexpr uint32_t kTmemO = kBuffers * 128;
// Registers: 128 a thread at launch (the most that 512 threads can have); the softmax warps hold a row of 128 scores.
constexpr int kRegsLaunch = 128, kRegsSoftmax = 200, kRegsOther = 56;
static_assert(256 * kRegsSoftmax + 256 * kRegsOther <= kThreads * kRegsLaunch, "shares of the launch's registers");

struct PrefillArgs {
    CUtensorMap q_map, k_map, v_map;
    void *out;
    int64_t o_ts, o_hs;                          // elements
    float *lse;
    int64_t lse_hs;
    const int32_t *cu_q, *cu_k;
    int total_q, total_k, batch, heads, group, causal;
    float scale_log2;                            // |scale| log2 e
    int negate;                                  // scale < 0
    int *status;
};

template <int DQK>
struct Smem {
    static constexpr int kDSlabs = DQK / 64;
    static constexpr int kQBytes = kDSlabs * kSlab, kKBytes = kDSlabs * kHalfSlab;     // of this CTA
    static constexpr int kSlots = DQK == 192 ? 3 : 4;                    // K blocks, and V blocks, in flight
    static constexpr int kQ = 0;                                         // two: the next item's is loaded early
    static constexpr int kK = 2 * kQBytes;
    static constexpr int kV = kK + kSlots * kKBytes;
    static constexpr int kBars = kV + kSlots * kSlab;
    static constexpr int kBarQFull = 0, kBarQEmpty = 2, kBarKFull = 4, kBarKEmpty = kBarKFull + kSlots, kBarVFull = kBarKEmpty + kSlots,
                         kBarVEmpty = kBarVFull + kSlots, kBarS = kBarVEmpty + kSlots, kBarP = kBarS + kBuffers, kBarPv = kBarP + kBuffers,
                         kBarO = kBarPv + 4, kBarRead = kBarO + 1, kBarSums = kBarRead + 8, kBarSumsEmpty = kBarSums + 8,
                         kBarTail = kBarSumsEmpty + 8, kBarRecFull = kBarTail + 1,
                         kBarRecEmpty = kBarRecFull + kRecords, kNumBars = kBarRecEmpty + kRecords;
    static constexpr int kRecs = kBars + kNumBars * 8;
    static constexpr int kRef = kRecs + kRecords * kRecInts * 4;         // the rows' reference
    static constexpr int kSums = kRef + 128 * 4;                         // {reference, sum} of each warpgroup at an item's end, of two items
    static constexpr int kQueue = kSums + 4 * 128 * 8;                   // eight items {blocks, keys} with scores not yet added
    static constexpr int kTurn = kQueue + 8 * 8;                         // [kRecords][4] whether the warps of a quarter go on
    static constexpr int kMisc = kTurn + kRecords * 4 * 4;               // abort flag, tensor memory address
    static constexpr int kOut = (kMisc + 16 + 127) & ~127;               // [4][32 rows][16 columns] of output on their way
    static constexpr int kBytes = kOut + 4 * 1024;
};
static_assert(Smem<192>::kBytes <= 232448 && Smem<128>::kBytes <= 232448, "shared memory of one CTA");

enum { kRecValid, kRecQRow, kRecRows, kRecHead, kRecKRow, kRecNk, kRecOff, kRecN };

__device__ __forceinline__ void give_up(volatile int *abort_flag, int *status, int bit) {
    *abort_flag = 1;
    atomicOr(status, bit);
}

// ------------------------------------------------------------------ items
// A sequence with nq queries and nk keys has ceil(nq / 256) items per head.  Item j of a causal sequence costs about as
// many steps as its last key, so items are dealt out in falling order of level = (level of the last) - (items behind
// it).  Levels are gathered into at most 32 buckets of two or more; inside a bucket the order is sequence, head, level, so
// that items which read the same keys run at the same time and the keys come from HBM once (512 queries with 8192 keys and 301
// with 4999, 64 heads: 259 us; level before head: 282).
struct Seq {
    int q0, nq, k0, nk, blocks, top;             // top: level of the last item
};
__device__ __forceinline__ Seq seq_of(const PrefillArgs &a, int b) {
    Seq s;
    s.q0 = min(max(__ldg(a.cu_q + b), 0), a.total_q);
    s.nq = min(max(__ldg(a.cu_q + b + 1), s.q0), a.total_q) - s.q0;
    s.k0 = min(max(__ldg(a.cu_k + b), 0), a.total_k);
    s.nk = min(max(__ldg(a.cu_k + b + 1), s.k0), a.total_k) - s.k0;
    s.blocks = (s.nq + 255) >> 8;
    s.top = max((s.nk + 255) >> 8, s.blocks);
    return s;
}

struct Walk {                                    // uniform over the loader warp
    int high, shift;                             // highest level of the bucket
    int b0;                                      // first of the 32 sequences looked at
    long long base;                              // items in front of theirs
};
// Items (per head) of sequence s in a bucket.
__device__ __forceinline__ int in_bucket(const Seq &s, const Walk &w) {
    const int lo = max(w.high - (1 << w.shift) + 1, s.top - s.blocks + 1), hi = min(w.high, s.top);
    return max(0, hi - lo + 1);
}
__device__ __forceinline__ void start_walk(const PrefillArgs &a, Walk &w, int lane) {
    int top = 0;
    for (int b = lane; b < a.batch; b += 32) {
        const Seq s = seq_of(a, b);
        if (s.blocks > 0) top = max(top, s.top);
    }
    w.high = __reduce_max_sync(0xffffffffu, top);
    w.shift = 1;
    while ((w.high >> w.shift) >= 32) ++w.shift;
    w.b0 = 0;
    w.base = 0;
}
// Item `idx` (not below any asked for before) as a record; false behind the last.
__device__ __forceinline__ bool find_item(const PrefillArgs &a, Walk &w, long long idx, int lane, int *rec) {
    for (; w.high > 0; w.high -= 1 << w.shift, w.b0 = 0) {
        for (; w.b0 < a.batch; w.b0 += 32) {
            Seq s = {};
            int n = 0;
            if (w.b0 + lane < a.batch) {
                s = seq_of(a, w.b0 + lane);
                n = s.blocks > 0 ? in_bucket(s, w) : 0;
            }
            int upto = n;                        // inclusive prefix sum over the lanes
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += x;
            }
            const long long here = static_cast<long long>(__shfl_sync(0xffffffffu, upto, 31)) * a.heads;
            if (idx < w.base + here) {
                // head after head, whose items are neighbours (they read the same keys); levels fall, from the highest that the
                // sequence has in the bucket
                const int local = static_cast<int>(idx - w.base) - (upto - n) * a.heads;  // (all items are fewer than 2^31)
                if (local >= 0 && local < n * a.heads) {                                 // one lane
                    const int head = local / n, level = min(w.high, s.top) - (local - head * n);
                    const int m0 = (s.blocks - 1 - (s.top - level)) << 8;
                    const int rows = min(256, s.nq - m0), off = m0 + s.nk - s.nq;
                    const int see = a.causal ? min(s.nk, max(0, off + rows)) : s.nk;     // keys that the item's last row sees
                    rec[kRecValid] = 1;
                    rec[kRecQRow] = s.q0 + m0;
                    rec[kRecRows] = rows;
                    rec[kRecHead] = head;
                    rec[kRecKRow] = s.k0;
                    rec[kRecNk] = s.nk;
                    rec[kRecOff] = off;
                    rec[kRecN] = (see + 127) >> 7;
                }
                return true;
            }
            w.base += here;
        }
    }
    return false;
}

// ------------------------------------------------------------------ loaders
// Records, Q and K.  Bytes of both CTAs are counted on the even one's barriers, whose products read them.
template <int DQK>
__device__ __forceinline__ void qk_loader_role(const PrefillArgs &a, uint8_t *smem, volatile int *abort_flag, int rank, int lane) {
    using L = Smem<DQK>;
    const uint32_t bars = smem_u32(smem + L::kBars), qs = smem_u32(smem + L::kQ), ks = smem_u32(smem + L::kK);
    const unsigned team = blockIdx.x >> 1, teams = gridDim.x >> 1;
    Walk w;
    start_walk(a, w, lane);
    uint32_t block = 0, nq = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
        const int slot = it % kRecords;
        int *rec = reinterpret_cast<int *>(smem + L::kRecs) + slot * kRecInts;
        if (!(ok = mbar_wait(bars + (L::kBarRecEmpty + slot) * 8, ((it / kRecords) & 1) ^ 1, abort_flag))) break;
        // back and forth over the pairs: the one with the largest item of a round gets the smallest of the next
        const unsigned turn = (it & 1) ? teams - 1 - team : team;
        const bool more = find_item(a, w, static_cast<long long>(it) * teams + turn, lane, rec);
        if (!more && lane == 0) rec[kRecValid] = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecFull + slot) * 8);
        if (!more) break;
        const volatile int *vr = rec;
        const int n = vr[kRecN], head = vr[kRecHead], krow = vr[kRecKRow] + rank * 64, qrow = vr[kRecQRow] + rank * 128;
        const int kv_head = head / a.group;
        if (n == 0) continue;
        const uint32_t qb = nq & 1;
        if (!(ok = mbar_wait(bars + (L::kBarQEmpty + qb) * 8, ((nq >> 1) & 1) ^ 1, abort_flag))) break;
        ++nq;
        if (lane == 0) {
            const uint32_t full = bars + (L::kBarQFull + qb) * 8;
            if (rank == 0) mbar_arrive_expect_tx(full, 2 * L::kQBytes);
            for (int s = 0; s < L::kDSlabs; ++s)
                tma_load_3d_pair(qs + qb * L::kQBytes + s * kSlab, &a.q_map, map_rank(full, 0), s * 64, qrow, head);
        }
        __syncwarp();
        for (int t = 0; t < n; ++t, ++block) {
            const uint32_t at = block % L::kSlots, full = bars + (L::kBarKFull + at) * 8;
            if (!(ok = mbar_wait(bars + (L::kBarKEmpty + at) * 8, ((block / L::kSlots) & 1) ^ 1, abort_flag))) break;
            if (lane == 0) {
                if (rank == 0) mbar_arrive_expect_tx(full, 2 * L::kKBytes);
                for (int s = 0; s < L::kDSlabs; ++s)
                    tma_load_3d_pair(ks + at * L::kKBytes + s * kHalfSlab, &a.k_map, map_rank(full, 0), s * 64, krow + t * 128, kv_head);
            }
            __syncwarp();
        }
    }
    // What the products still signal to this CTA has to have come before it may end.
    for (uint32_t i = block > static_cast<uint32_t>(L::kSlots) ? block - L::kSlots : 0; ok && i < block; ++i)
        ok = mbar_wait(bars + (L::kBarKEmpty + i % L::kSlots) * 8, (i / L::kSlots) & 1, abort_flag);
    for (uint32_t i = nq > 2 ? nq - 2 : 0; ok && i < nq; ++i) ok = mbar_wait(bars + (L::kBarQEmpty + (i & 1)) * 8, (i >> 1) & 1, abort_flag);
    if (!ok) {
        // Another role gave up, or this one.  The copies in flight have to land before the CTA may end; the odd CTA's are
        // counted by the even one, for which it waits at the end.
        if (lane == 0) give_up(abort_flag, a.status, kStatusGatherWait);
        __syncwarp();
        int never = 0;
        if (rank == 0) {
            for (uint32_t i = block > static_cast<uint32_t>(L::kSlots) ? block - L::kSlots : 0; i < block; ++i)
                mbar_wait(bars + (L::kBarKFull + i % L::kSlots) * 8, (i / L::kSlots) & 1, &never);
            for (uint32_t i = nq > 2 ? nq - 2 : 0; i < nq; ++i) mbar_wait(bars + (L::kBarQFull + (i & 1)) * 8, (i >> 1) & 1, &never);
        }
    }
}

template <int DQK>
__device__ __forceinline__ void v_loader_role(const PrefillArgs &a, uint8_t *smem, volatile int *abort_flag, int rank, int lane) {
    using L = Smem<DQK>;
    const uint32_t bars = smem_u32(smem + L::kBars), vs = smem_u32(smem + L::kV), tail = bars + L::kBarTail * 8;
    uint32_t block = 0, tails = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
        const int slot = it % kRecords;
        if (!(ok = mbar_wait(bars + (L::kBarRecFull + slot) * 8, (it / kRecords) & 1, abort_flag))) break;
        const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * kRecInts;
        const int valid = rec[kRecValid], n = rec[kRecN], nk = rec[kRecNk], krow = rec[kRecKRow], head = rec[kRecHead];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) break;
        const int kv_head = head / a.group;
        for (int t = 0; t < n; ++t, ++block) {
            const uint32_t at = block % L::kSlots, full = bars + (L::kBarVFull + at) * 8, dst = vs + at * kSlab;
            if (!(ok = mbar_wait(bars + (L::kBarVEmpty + at) * 8, ((block / L::kSlots) & 1) ^ 1, abort_flag))) break;
            const int left = nk - t * 128;
            if (left >= 128 || (left & 15) == 0) {
                if (lane == 0) {
                    const uint32_t both = map_rank(full, 0);
                    mbar_arrive_expect_tx_cluster(both, kSlab);
                    tma_load_3d_pair(dst, &a.v_map, both, rank * 64, krow + t * 128, kv_head);
                }
                __syncwarp();
            } else {
                // The last 16 rows that are multiplied reach past the sequence: what lies there (another sequence's rows,
                // NaN) has weight 0, and 0 x NaN is NaN.  They are cleared before the block is given to the products.
                if (lane == 0) {
                    mbar_arrive_expect_tx(tail, kSlab);
                    tma_load_3d(dst, &a.v_map, tail, rank * 64, krow + t * 128, kv_head);
                }
                __syncwarp();
                if (!(ok = mbar_wait(tail, tails++ & 1, abort_flag))) break;
                const int r0 = left, r1 = (left + 15) & ~15;
                for (int x = lane; x < (r1 - r0) * 8; x += 32)
                    asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(dst + (r0 + (x >> 3)) * 128 + (x & 7) * 16), "r"(0) : "memory");
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(map_rank(full, 0));
            }
        }
    }
    for (uint32_t i = block > static_cast<uint32_t>(L::kSlots) ? block - L::kSlots : 0; ok && i < block; ++i)      // as the other loader
        ok = mbar_wait(bars + (L::kBarVEmpty + i % L::kSlots) * 8, (i / L::kSlots) & 1, abort_flag);
    if (!ok) {
        if (lane == 0) give_up(abort_flag, a.status, kStatusGatherWait);
        __syncwarp();
        int never = 0;
        if (tails > 0) mbar_wait(tail, (tails - 1) & 1, &never);
        if (rank == 0)
            for (uint32_t i = block > static_cast<uint32_t>(L::kSlots) ? block - L::kSlots : 0; i < block; ++i)
                mbar_wait(bars + (L::kBarVFull + i % L::kSlots) * 8, (i / L::kSlots) & 1, &never);
    }
}

// ------------------------------------------------------------------ products (the even CTA, for both)
// Two barriers, looked at together first: a look takes this warp over 100 cycles, but they overlap.
__device__ __forceinline__ bool wait_both(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1, volatile int *abort_flag) {
    const bool x = mbar_test_wait(b0, p0), y = mbar_test_wait(b1, p1);
    return (x && y) || (mbar_wait(b0, p0, abort_flag) && mbar_wait(b1, p1, abort_flag));
}
template <int DQK, bool FP16>
__device__ __forceinline__ void mma_role(const PrefillArgs &a, uint8_t *smem, uint32_t tmem, volatile int *abort_flag, int lane) {
    using L = Smem<DQK>;
    const uint32_t bars = smem_u32(smem + L::kBars);
    const uint32_t go = elect_one();
    constexpr uint32_t idesc_qk = umma_idesc_16(FP16, 256, 128, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_16(FP16, 256, 128, 0, 1);
    const uint64_t qd = umma_desc_sw128(smem_u32(smem + L::kQ), 16), kd = umma_desc_sw128(smem_u32(smem + L::kK), 16),
                   vd = umma_desc_sw128(smem_u32(smem + L::kV), 16);
    volatile int2 *queue = reinterpret_cast<volatile int2 *>(smem + L::kQueue);
    // Two cursors over the items' tiles: the scores run ahead of the output by up to three.  Items pass from one to the other
    // through a queue, and records are given back at once.
    int s_it = 0, s_left = 0, o_n = 0, o_t = 0, o_nk = 0;
    uint32_t scored = 0, added = 0, items_in = 0, items_out = 0;         // tiles; items with keys
    bool ok = true, more = true;                 // more: there may be tiles to score

    // Finds the next tile to score and waits for its operands.  While output is outstanding the next record may depend on it:
    // it is then looked for, not waited for.
    const auto find_tile = [&] {
        while (more && s_left == 0) {
            const int slot = s_it % kRecords;
            const uint32_t rec_bar = bars + (L::kBarRecFull + slot) * 8, rec_phase = (s_it / kRecords) & 1;
            if (scored != added) {
                if (!__all_sync(0xffffffffu, mbar_test_wait(rec_bar, rec_phase))) return false;
            } else if (!(ok = mbar_wait(rec_bar, rec_phase, abort_flag))) {
                return false;
            }
            const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * kRecInts;
            more = rec[kRecValid] != 0;
            const int nk = rec[kRecNk];
            s_left = more ? rec[kRecN] : 0;
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
                if (s_left > 0) {
                    queue[items_in % 8].x = s_left;
                    queue[items_in % 8].y = nk;
                }
            }
            __syncwarp();
            ++s_it;
            if (s_left > 0) {
                if (!(ok = mbar_wait(bars + (L::kBarQFull + (items_in & 1)) * 8, (items_in >> 1) & 1, abort_flag))) return false;
                ++items_in;
            }
        }
        if (!more || !(ok = mbar_wait(bars + (L::kBarKFull + scored % L::kSlots) * 8, (scored / L::kSlots) & 1, abort_flag))) return false;
        tc_fence_after_sync();
        return true;
    };
    // S(scored) = Q K^T, into the buffer of the tile three before, whose product into O has been issued
    const auto score = [&] {
        const uint32_t at = scored % L::kSlots, buf = scored % kBuffers, qb = (items_in - 1) & 1;
        const uint64_t qa = qd + static_cast<uint64_t>((qb * L::kQBytes) >> 4), kb = kd + static_cast<uint64_t>((at * L::kKBytes) >> 4);
        if (go) {
#pragma unroll
            for (int s = 0; s < L::kDSlabs; ++s)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_ss_pair_pred(tmem + buf * 128, qa + ((s * kSlab) >> 4) + 2 * k, kb + ((s * kHalfSlab) >> 4) + 2 * k, idesc_qk,
                                      (s | k) ? 1u : 0u, 1u);
        }
        umma_commit_pair_pred(bars + (L::kBarS + buf) * 8, go);
        umma_commit_pair_pred(bars + (L::kBarKEmpty + at) * 8, go);
        if (--s_left == 0) umma_commit_pair_pred(bars + (L::kBarQEmpty + qb) * 8, go);
        ++scored;
    };
    // Three tiles are scored ahead, the next one right behind the product into O that frees its buffer.
    while (scored < static_cast<uint32_t>(kBuffers) && find_tile()) score();
    uint32_t at = 0, buf = 0, v_phase = 0, p_phase = 0;      // of tile `added`
    while (ok && scored != added) {
        if (o_t == o_n) {
            o_n = queue[items_out % 8].x;
            o_nk = queue[items_out % 8].y;
            ++items_out;
            o_t = 0;
        }
        // O += P V of the next tile
        const int left = o_nk - o_t * 128;
        const uint64_t v = vd + static_cast<uint64_t>((at * kSlab) >> 4);
        const uint32_t p = tmem + buf * 128, acc = o_t > 0 ? 1u : 0u;
        // V, and the weights of both CTAs in tensor memory; O has been moved to a new reference where one was needed, and the last
        // item's output has been read
        if (!(ok = wait_both(bars + (L::kBarVFull + at) * 8, v_phase, bars + (L::kBarP + buf) * 8, p_phase, abort_flag))) break;
        tc_fence_after_sync();
        if (left > 112) {
            if (go) {
#pragma unroll
                for (int k = 0; k < 8; ++k) umma_ts_pair_pred(tmem + kTmemO, p + k * 8, v + k * 128, idesc_pv, k ? 1u : acc, 1u);
            }
        } else {
            for (int k = 0; k * 16 < left; ++k) umma_ts_pair_pred(tmem + kTmemO, p + k * 8, v + k * 128, idesc_pv, k ? 1u : acc, go);
        }
        ++added;
        if (++o_t == o_n) umma_commit_pair_pred(bars + L::kBarO * 8, go);
        if (find_tile()) score();
        if (!ok) break;
        umma_commit_pair_pred(bars + (L::kBarPv + ((added - 1) & 3)) * 8, go);
        umma_commit_pair_pred(bars + (L::kBarVEmpty + at) * 8, go);
        if (++at == L::kSlots) {
            at = 0;
            v_phase ^= 1;
        }
        if (++buf == kBuffers) {
            buf = 0;
            p_phase ^= 1;
        }
        // the last tiles of an item whose successor was not there yet
        while (scored - added < static_cast<uint32_t>(kBuffers) && find_tile()) score();
    }
    if (!ok && lane == 0) give_up(abort_flag, a.status, kStatusMmaWait);
}

// ------------------------------------------------------------------ softmax and output
template <bool FP16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    uint32_t r;
    if constexpr (FP16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Weights are 2^kLift times exp(s - m).  A weight may be 2^8 before the reference moves, and fp16 holds 2^15: what is above
// that is given to the small ones, which fp16 drops below 2^-25.  A key far below the row's largest adds next to nothing,
// but 10^5 of them at 2^-26 are 0.2 % of the output, and the sum counts them.  bf16 has the exponents of fp32.
template <bool FP16>
constexpr float kLift = FP16 ? 7.0f : 0.0f;

// Warpgroup `side` takes the tiles g with g % 2 == side of a CTA's sequence; its thread is a row (lane of tensor memory).  The
// row's reference passes from tile to tile through shared memory; each warpgroup keeps its own part of the sum.
template <int DQK, bool FP16>
__device__ __forceinline__ void softmax_role(const PrefillArgs &a, uint8_t *smem, uint32_t tmem, volatile int *abort_flag, int rank, int warp, int lane) {
    using L = Smem<DQK>;
    const uint32_t bars = smem_u32(smem + L::kBars);
    const int side = warp >> 2, quarter = warp & 3, lane_row = quarter * 32 + lane, row = rank * 128 + lane_row;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16), o_addr = t_lane + kTmemO;
    float *ref_at = reinterpret_cast<float *>(smem + L::kRef) + lane_row;
    const uint32_t p_bar = map_rank(bars + L::kBarP * 8, 0);  // the even CTA's
    float2 *sums = reinterpret_cast<float2 *>(smem + L::kSums) + side * 128 + lane_row;
    const float c = a.scale_log2;
    uint32_t tile = 0, n_items = 0;              // tiles; items with keys
    bool failed = false;
    // The two softmax warps of a quarter meet at barriers that know no time limit, so they have to take the same items.  Whichever
    // comes to an item first decides, for both, whether they take it or one of them has given up.
    int *turns = reinterpret_cast<int *>(smem + L::kTurn) + quarter;
    const auto go_on = [&](int it, bool mine) {
        int v = 0;
        if (lane == 0) {
            int *turn = turns + it % kRecords * 4;
            const int want = (it + 1) * 2 + (mine ? 1 : 0), old = *const_cast<volatile int *>(turn);
            v = (old >> 1) == it + 1 ? old : atomicCAS(turn, old, want);
            if (v == old && (old >> 1) != it + 1) v = want;
        }
        return (__shfl_sync(0xffffffffu, v, 0) & 1) != 0;
    };
    for (int it = 0;; ++it) {
        const int slot = it % kRecords;
        failed |= !mbar_wait(bars + (L::kBarRecFull + slot) * 8, (it / kRecords) & 1, abort_flag);
        failed = __any_sync(0xffffffffu, failed);
        if (!go_on(it, !failed)) {
            failed = true;
            break;
        }
        const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * kRecInts;
        const int valid = rec[kRecValid], n = rec[kRecN], nk = rec[kRecNk], off = rec[kRecOff];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) break;
        const int lim = a.causal ? min(nk, off + row + 1) : nk;                        // keys that this row sees
        const int lim_warp = a.causal ? min(nk, off + row - lane + 1) : nk;            // ... and the warp's first row
        float m = -INFINITY;                     // the reference, in log2 units
        uint64_t l2 = 0;                         // two partial sums
        for (int t = 0; t < n; ++t, ++tile) {
            if ((tile & 1) != static_cast<uint32_t>(side)) continue;
            const uint32_t buf = tile % kBuffers, s_addr = t_lane + buf * 128;
            // The output's barriers take turns over four tiles, and a parity tells only neighbouring phases apart: a wait for the
            // product of tile - 1 (below) needs to know that the one of tile - 5 has arrived.  So every tile's warp sees the product
            // of tile - 4 first: it came before these scores in the tensor pipe (no delay), tile's own cannot have come, and the
            // warp before saw the one of tile - 5 ahead of its arrival at the named barrier.
            failed |= !mbar_wait(bars + (L::kBarPv + (tile & 3)) * 8, ((tile >> 2) & 1) ^ 1, abort_flag);
            failed |= !mbar_wait(bars + (L::kBarS + buf) * 8, (tile / kBuffers) & 1, abort_flag);
            tc_fence_after_sync();
            uint32_t s[128];
#pragma unroll
            for (int j = 0; j < 4; ++j) tmem_ld_x32_nowait(s_addr + j * 32, s + j * 32);
            tmem_ld_wait();
            if (a.negate) {
#pragma unroll
                for (int j = 0; j < 128; ++j) s[j] ^= 0x80000000u;
            }
            if (t * 128 + 128 > lim_warp) {
                const int see = lim - t * 128;
#pragma unroll
                for (int j = 0; j < 128; j += 32) {
                    const uint32_t hidden = see >= j + 32 ? 0u : see <= j ? ~0u : ~0u << (see - j);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if ((hidden >> e) & 1u) s[j + e] = 0xFF800000u;
                }
            }
            float mx[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(__uint_as_float(s[e]), __uint_as_float(s[4 + e]));
#pragma unroll
            for (int j = 8; j < 128; j += 8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], fmaxf(__uint_as_float(s[j + e]), __uint_as_float(s[j + 4 + e])));
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
            // the reference as the tile before left it
            if (tile > 0) named_bar_sync(6 + quarter * 2 - side, 64);
            const float now = t > 0 ? *ref_at : -INFINITY, to = top > now + 8.0f ? top : now;
            if (t == 0 || __any_sync(0xffffffffu, to != m)) {
                // (the warpgroup's first tile of an item, or one of the last two tiles moved a reference)
                if (t > 0 && __any_sync(0xffffffffu, to != now)) {
                    // everything before this tile has to be in O, nothing behind it can be
                    failed |= !mbar_wait(bars + (L::kBarPv + ((tile - 1) & 3)) * 8, ((tile - 1) >> 2) & 1, abort_flag);
                    tc_fence_after_sync();
                    const float f = to == now ? 1.0f : fast_exp2(now - to);
#pragma unroll 1
                    for (int j = 0; j < 128; j += 8) {
                        uint32_t o[8];
                        tmem_ld_x8(o_addr + j, o);
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_x8(o_addr + j, o);
                    }
                }
                *ref_at = to;
                const float f = to == m ? 1.0f : fast_exp2(m - to);      // 0 for the warpgroup's first keys
                l2 = mul2(l2, pack2(f, f));
                m = to;
                __syncwarp();
            }
            named_bar_arrive(5 + quarter * 2 + side, 64);    // the warp with the next tile's rows waits there
            const float ref = m == -INFINITY ? 0.0f : kLift<FP16> - m;
            const uint64_t c2 = pack2(c, c), ref2 = pack2(ref, ref);
            uint64_t la = l2, lb = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float x, y;
                    unpack2(fma2(pack2(__uint_as_float(s[j * 32 + 2 * e]), __uint_as_float(s[j * 32 + 2 * e + 1])), c2, ref2), x, y);
                    x = fast_exp2(x);
                    y = fast_exp2(y);
                    if (e & 1) lb = add2(lb, pack2(x, y));
                    else la = add2(la, pack2(x, y));
                    w[e] = pack16<FP16>(x, y);
                }
                tmem_st_x16(s_addr + j * 16, w);
            }
            l2 = add2(la, lb);
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            // The last item's output (k - 1) has been read before the product that overwrites it can start.  Two barriers in
            // turn: what item k - 3 signalled on this one is known to have come.  Either items k - 1 and k - 2 have a tile each, and
            // this warpgroup waited for k - 3 with the one of k - 2; or they have three, and this tile's scores came behind the
            // product of a tile of k - 2, which waited for it.
            if (t == 0 && n_items > 0) {
                const uint32_t last = n_items - 1;
                failed |= !mbar_wait(bars + (L::kBarRead + (last & 1) * 4 + quarter) * 8, (last >> 1) & 1, abort_flag);
            }
            if (lane == 0) mbar_arrive_remote(p_bar + buf * 8);
        }
        if (n == 0) continue;
        float lx, ly;
        unpack2(l2, lx, ly);
        const uint32_t sums_at = (n_items & 1) * 4 + quarter;
        failed |= !mbar_wait(bars + (L::kBarSumsEmpty + sums_at) * 8, ((n_items >> 1) & 1) ^ 1, abort_flag);
        sums[(n_items & 1) * 256] = make_float2(m, lx + ly);
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarSums + sums_at) * 8);
        ++n_items;
    }
    if (tile > 0 && (tile & 1) == static_cast<uint32_t>(side)) {
        named_bar_sync(6 + quarter * 2 - side, 64);          // the last arrival's
        for (uint32_t i = tile > 4 ? tile - 4 : 0; !failed && i < tile; ++i)           // and the last products'
            failed = !mbar_wait(bars + (L::kBarPv + (i & 3)) * 8, (i >> 2) & 1, abort_flag);
    }
    if (failed && lane == 0) give_up(abort_flag, a.status, kStatusSoftmaxWait);
}

// The output of an item, while the softmax warps go on with the next one, whose first weights they hand over when this output
// has been read.  A thread is a row.
template <int DQK, bool FP16>
__device__ __forceinline__ void output_role(const PrefillArgs &a, uint8_t *smem, uint32_t tmem, volatile int *abort_flag, int rank, int quarter, int lane) {
    using L = Smem<DQK>;
    const uint32_t bars = smem_u32(smem + L::kBars), o_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + kTmemO;
    const int row = rank * 128 + quarter * 32 + lane;
    const float2 *sums = reinterpret_cast<const float2 *>(smem + L::kSums) + quarter * 32 + lane;
    // A warp's rows go through shared memory 16 columns at a time, so that two lanes store 32 consecutive bytes: 16 bytes of
    // each row at a time, straight from the lanes, take 32 cycles of the load and store unit per instruction.  The loop is not
    // unrolled: the instruction cache holds the softmax, and a whole row in registers first (88 of them) took 40 % longer
    // where items are one tile.
    uint8_t *stage = smem + L::kOut + quarter * 1024;
    uint4 *put[2] = {reinterpret_cast<uint4 *>(stage + lane * 32 + (lane >> 2 & 1) * 16), reinterpret_cast<uint4 *>(stage + lane * 32 + (~lane >> 2 & 1) * 16)};
    const uint4 *get = reinterpret_cast<const uint4 *>(stage + (lane >> 1) * 32 + ((lane ^ (lane >> 3)) & 1) * 16);
    const int first = rank * 128 + quarter * 32 + (lane >> 1);
    uint32_t n_items = 0;
    bool ok = true;
    for (int it = 0;; ++it) {
        const int slot = it % kRecords;
        if (!(ok = mbar_wait(bars + (L::kBarRecFull + slot) * 8, (it / kRecords) & 1, abort_flag))) break;
        const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * kRecInts;
        const int valid = rec[kRecValid], n = rec[kRecN], rows = rec[kRecRows], head = rec[kRecHead], qrow = rec[kRecQRow];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) break;
        float top = -INFINITY, l = 0.0f;
        if (n > 0) {
            // the sums of both warpgroups, under the later of their references (it only rises)
            const uint32_t sums_at = (n_items & 1) * 4 + quarter;
            if (!(ok = mbar_wait(bars + (L::kBarSums + sums_at) * 8, (n_items >> 1) & 1, abort_flag))) break;
            const float2 s0 = sums[(n_items & 1) * 256], s1 = sums[(n_items & 1) * 256 + 128];
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + (L::kBarSumsEmpty + sums_at) * 8);
            top = fmaxf(s0.x, s1.x);
            l = top == -INFINITY ? s0.y + s1.y : s0.y * fast_exp2(s0.x - top) + s1.y * fast_exp2(s1.x - top);      // 0, or NaN from NaN
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (row < rows && a.lse != nullptr) a.lse[head * a.lse_hs + qrow + row] = l == 0.0f ? -INFINITY : (top - kLift<FP16> + log2f(l)) * kLn2;
        if (n > 0) {
            if (!(ok = mbar_wait(bars + L::kBarO * 8, n_items & 1, abort_flag))) break;
            tc_fence_after_sync();
        }
        uint16_t *dst = static_cast<uint16_t *>(a.out) + (qrow + first) * a.o_ts + head * a.o_hs + (lane & 1) * 8;
#pragma unroll 1
        for (int j = 0; j < 128; j += 16) {
            uint4 w[2] = {};
            if (n > 0) {
                uint32_t o[16];
                tmem_ld_x16(o_addr + j, o);
                if (j == 112) {
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bars + (L::kBarRead + (n_items & 1) * 4 + quarter) * 8);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)      // a row without keys: zeros (the accumulator may hold anything)
                        x[i] = l == 0.0f ? 0u : pack16<FP16>(__uint_as_float(o[e * 8 + 2 * i]) * inv, __uint_as_float(o[e * 8 + 2 * i + 1]) * inv);
                    *put[e] = make_uint4(x[0], x[1], x[2], x[3]);
                }
                __syncwarp();
                w[0] = get[0];
                w[1] = get[32];
                __syncwarp();
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (first + e * 16 < rows) *reinterpret_cast<uint4 *>(dst + e * 16 * a.o_ts + j) = w[e];
        }
        if (n > 0) ++n_items;
    }
    if (!ok && lane == 0) give_up(abort_flag, a.status, kStatusSoftmaxWait);
}

template <int DQK, bool FP16>
__global__ void __launch_bounds__(kThreads, 1) dense_prefill_kernel(const __grid_constant__ PrefillArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using L = Smem<DQK>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = static_cast<int>(cluster_rank());
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kMisc);
    const uint32_t bars = smem_u32(smem + L::kBars);
    if ((smem_u32(smem) & 1023u) != 0u) {        // the swizzled slabs need it
        if (tid == 0) atomicOr(a.status, kStatusSmemLayout);
        return;
    }
    if (tid == 0) {
        const auto init = [&](int first, int n, int count) {
            for (int i = 0; i < n; ++i) mbar_init(bars + (first + i) * 8, count);
        };
        init(L::kBarQFull, 4, 1);                // and kBarQEmpty
        init(L::kBarKFull, 2 * L::kSlots, 1);    // and kBarKEmpty
        init(L::kBarVFull, L::kSlots, 2);        // both CTAs' loaders
        init(L::kBarVEmpty, L::kSlots, 1);
        init(L::kBarS, kBuffers, 1);
        init(L::kBarP, kBuffers, 8);             // four warps of each CTA
        init(L::kBarPv, 4, 1);
        init(L::kBarO, 1, 1);
        init(L::kBarRead, 8, 1);
        init(L::kBarSums, 8, 2);                 // a warp of each softmax warpgroup
        init(L::kBarSumsEmpty, 8, 1);
        init(L::kBarTail, 1, 1);
        init(L::kBarRecFull, kRecords, 1);
        init(L::kBarRecEmpty, kRecords, rank == 0 ? 14 : 13);
        for (int i = 0; i < kRecords * 4; ++i) reinterpret_cast<int *>(smem + L::kTurn)[i] = 0;
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 8) tmem_alloc_pair(smem_u32(smem + L::kMisc + 8), 512);
    tc_fence_before_sync();
    cluster_sync_all();                          // also: the other CTA's barriers are there
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::kMisc + 8);
    if (warp < 8) {
        regs_inc<kRegsSoftmax>();
        softmax_role<DQK, FP16>(a, smem, tmem, abort_flag, rank, warp, lane);
    } else {
        regs_dec<kRegsOther>();
        if (warp == 8 && rank == 0) mma_role<DQK, FP16>(a, smem, tmem, abort_flag, lane);
        else if (warp == 9) qk_loader_role<DQK>(a, smem, abort_flag, rank, lane);
        else if (warp == 10) v_loader_role<DQK>(a, smem, abort_flag, rank, lane);
        else if (warp >= 12) output_role<DQK, FP16>(a, smem, tmem, abort_flag, rank, warp & 3, lane);
    }
    tc_fence_before_sync();
    __syncwarp();
    cluster_sync_all();                          // nothing of this CTA's is used by the other any more
    if (warp == 8) tmem_free_pair(tmem, 512);
}

template <int DQK, bool FP16>
int launch(PrefillArgs &a, unsigned grid, cudaStream_t stream) {
    static KernelSetup setup;
    const int rc = setup.get(reinterpret_cast<const void *>(&dense_prefill_kernel<DQK, FP16>), Smem<DQK>::kBytes, &a.status, kRegsLaunch);
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<DQK>::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, dense_prefill_kernel<DQK, FP16>, a));
}

}  // namespace

int launch_dense_prefill(const smla_prefill_params_t &p, int sm_count, cudaStream_t stream) {
    PrefillArgs a = {};
    const bool fp16 = p.dtype == 1;
    if (!make_slab_map(&a.q_map, fp16, p.q, p.head_dim, p.total_q, p.num_heads, p.q_token_stride * 2, p.q_head_stride * 2, 128))
        return SMLA_EINVAL;
    // without keys no item has a key block, and the maps of k and v are never used
    if (p.total_k > 0 &&
        (!make_slab_map(&a.k_map, fp16, p.k, p.head_dim, p.total_k, p.num_kv_heads, p.k_token_stride * 2, p.k_head_stride * 2, 64) ||
         !make_slab_map(&a.v_map, fp16, p.v, 128, p.total_k, p.num_kv_heads, p.v_token_stride * 2, p.v_head_stride * 2, 128)))
        return SMLA_EINVAL;
    a.out = p.out;
    a.o_ts = p.out_token_stride;
    a.o_hs = p.out_head_stride;
    a.lse = p.softmax_lse;
    a.lse_hs = p.lse_head_stride;
    a.cu_q = p.cu_seqlens_q;
    a.cu_k = p.cu_seqlens_k;
    a.total_q = static_cast<int>(p.total_q);
    a.total_k = static_cast<int>(p.total_k);
    a.batch = p.batch;
    a.heads = p.num_heads;
    a.group = p.num_heads / p.num_kv_heads;
    a.causal = p.causal ? 1 : 0;
    const float c = p.softmax_scale * kLog2e;
    a.negate = c < 0.0f;
    // a scale of 0 makes all scores equal; a factor too small to matter does the same and keeps -inf x factor defined
    a.scale_log2 = std::max(c < 0.0f ? -c : c, 1e-35f);
    // each sequence adds at most one item that is not full
    const int64_t items = (p.total_q / 256 + p.batch) * p.num_heads;
    const unsigned grid = 2 * static_cast<unsigned>(std::min<int64_t>(items, sm_count / 2));
    if (p.head_dim == 192) return fp16 ? launch<192, true>(a, grid, stream) : launch<192, false>(a, grid, stream);
    return fp16 ? launch<128, true>(a, grid, stream) : launch<128, false>(a, grid, stream);
}

}  // namespace smla
