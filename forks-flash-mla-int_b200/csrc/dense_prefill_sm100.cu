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
// Work is cut into items: 256 query rows of one head, as two halves of 128 (the lanes of tensor memory).  A CTA
// (persistent, one per SM) holds the item's Q (2 x 128 x d) in shared memory and walks the keys in blocks of 128:
//   S_i = Q_i K^T  -> tensor memory, 128 columns of fp32 per half (both operands by descriptor from shared memory)
//   P_i = exp(S_i - m)  -> 16-bit, written over S_i in tensor memory (64 columns)
//   O_i += P_i V  -> tensor memory, 128 columns per half (P_i read from tensor memory, V from shared memory)
// S0 | S1 | O0 | O1 take all 512 columns.  While one half's weights are computed the tensor pipe works on the other's.
// K and V arrive by TMA as [128 rows][64 dims] slabs with the 128-byte swizzle in one ring; a slab read K-major gives
// K for the first product and MN-major gives V for the second.
//
// Roles (384 threads): warps 0-3 and 4-7 are the softmax of the two halves (one row per thread), warp 8 issues the
// MMAs, warp 9 finds the items and loads.  Item records go through a ring of four in shared memory.
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
constexpr int kThreads = 384;
constexpr int kSlab = 128 * 128;                 // bytes of [128 rows][64 dims] of 16-bit elements
constexpr int kSlabs = 14;                       // Q and ring together
constexpr int kRecords = 4;
// Registers: 168 a thread at launch (the most that 384 threads can have); the softmax warps hold a row of 128 scores.
constexpr int kRegsLaunch = 168, kRegsSoftmax = 208, kRegsOther = 88;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther <= kThreads * kRegsLaunch, "shares of the launch's registers");
constexpr int kRecInts = 12;

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
    static constexpr int kDSlabs = DQK / 64;                 // slabs of a 128-row tile of Q or K
    static constexpr int kRing = kSlabs - 2 * kDSlabs;       // 8 slabs at 192 dims, 10 at 128
    static constexpr int kQ = 0;
    static constexpr int kRingAt = 2 * kDSlabs * kSlab;
    static constexpr int kBars = kSlabs * kSlab;
    static constexpr int kBarFull = 0, kBarEmpty = kRing, kBarQFull = 2 * kRing, kBarQEmpty = kBarQFull + 1, kBarS = kBarQFull + 2,
                         kBarP = kBarQFull + 4, kBarO = kBarQFull + 6, kBarRecFull = kBarQFull + 8, kBarRecEmpty = kBarRecFull + kRecords,
                         kNumBars = kBarRecEmpty + kRecords;
    static constexpr int kRecs = kBars + kNumBars * 8;
    static constexpr int kMisc = kRecs + kRecords * kRecInts * 4;        // abort flag, tensor memory address
    static constexpr int kBytes = kMisc + 16;
};
static_assert(Smem<192>::kBytes <= 232448 && Smem<128>::kBytes <= 232448, "shared memory of one CTA");

enum { kRecValid, kRecQRow, kRecRows, kRecHead, kRecKRow, kRecNk, kRecOff, kRecN0, kRecN1 };

__device__ __forceinline__ void give_up(volatile int *abort_flag, int *status, int bit) {
    *abort_flag = 1;
    atomicOr(status, bit);
}

// ------------------------------------------------------------------ items
// A sequence with nq queries and nk keys has ceil(nq / 256) items per head.  Item j of a causal sequence costs about as
// many steps as its last key, so items are dealt out in falling order of level = (level of the last) - (items behind
// it); levels are gathered into at most 32 buckets, inside a bucket the order is sequence, level, head.
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
    int bucket, shift;
    long long base;                              // items in the buckets above
};
// Items (per head) of sequence s in a bucket.
__device__ __forceinline__ int in_bucket(const Seq &s, int bucket, int shift) {
    const int lo = max(bucket << shift, s.top - s.blocks + 1), hi = min(((bucket + 1) << shift) - 1, s.top);
    return max(0, hi - lo + 1);
}
__device__ __forceinline__ void start_walk(const PrefillArgs &a, Walk &w, int lane) {
    int top = 0;
    for (int b = lane; b < a.batch; b += 32) {
        const Seq s = seq_of(a, b);
        if (s.blocks > 0) top = max(top, s.top);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    w.shift = 0;
    while ((top >> w.shift) >= 32) ++w.shift;
    w.bucket = top >> w.shift;
    w.base = 0;
}
// Item `idx` (not below any asked for before) as a record; false behind the last.
__device__ __forceinline__ bool find_item(const PrefillArgs &a, Walk &w, long long idx, int lane, int *rec) {
    for (; w.bucket >= 0; --w.bucket) {
        int r = -1;                              // rank of the item among those of the bucket, without the head
        if (idx >= w.base) r = static_cast<int>(min((idx - w.base) / a.heads, 0x7FFFFFFFll));
        const int head = static_cast<int>((idx - w.base) % a.heads);
        int before = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 32) {
            Seq s = {};
            int n = 0;
            if (b0 + lane < a.batch) {
                s = seq_of(a, b0 + lane);
                n = s.blocks > 0 ? in_bucket(s, w.bucket, w.shift) : 0;
            }
            int upto = n;                        // inclusive prefix sum over the lanes
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += x;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, r >= before + upto - n && r < before + upto);
            if (hit != 0u) {
                const int src = __ffs(hit) - 1;
                // levels fall inside the bucket: rank 0 is the highest level that the sequence has there
                const int level = min(((w.bucket + 1) << w.shift) - 1, s.top) - (r - (before + upto - n));
                const int m0 = (s.blocks - 1 - (s.top - level)) << 8;
                const int rows = min(256, s.nq - m0), off = m0 + s.nk - s.nq;
                int n0 = s.nk, n1 = s.nk;
                if (a.causal) {
                    n0 = min(s.nk, max(0, off + min(rows, 128)));
                    n1 = min(s.nk, max(0, off + rows));
                }
                if (lane == src) {
                    rec[kRecValid] = 1;
                    rec[kRecQRow] = s.q0 + m0;
                    rec[kRecRows] = rows;
                    rec[kRecHead] = head;
                    rec[kRecKRow] = s.k0;
                    rec[kRecNk] = s.nk;
                    rec[kRecOff] = off;
                    rec[kRecN0] = (n0 + 127) >> 7;
                    rec[kRecN1] = rows > 128 ? (n1 + 127) >> 7 : 0;
                }
                return true;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        w.base += static_cast<long long>(before) * a.heads;
    }
    return false;
}

// ------------------------------------------------------------------ loader
template <int DQK>
__device__ __forceinline__ void loader_role(const PrefillArgs &a, uint8_t *smem, volatile int *abort_flag, int lane) {
    using L = Smem<DQK>;
    const uint32_t bars = smem_u32(smem + L::kBars), ring = smem_u32(smem + L::kRingAt), qs = smem_u32(smem + L::kQ);
    Walk w;
    start_walk(a, w, lane);
    uint32_t slab = 0, nq_loads = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
        const int slot = it % kRecords;
        int *rec = reinterpret_cast<int *>(smem + L::kRecs) + slot * kRecInts;
        if (!(ok = mbar_wait(bars + (L::kBarRecEmpty + slot) * 8, ((it / kRecords) & 1) ^ 1, abort_flag))) break;
        // back and forth over the CTAs: the one with the largest item of a round gets the smallest of the next
        const unsigned turn = (it & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
        const bool more = find_item(a, w, static_cast<long long>(it) * gridDim.x + turn, lane, rec);
        if (!more && lane == 0) rec[kRecValid] = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecFull + slot) * 8);
        if (!more) break;
        const volatile int *vr = rec;
        const int n0 = vr[kRecN0], n1 = vr[kRecN1], n = max(n0, n1), head = vr[kRecHead], krow = vr[kRecKRow], qrow = vr[kRecQRow];
        const int kv_head = head / a.group;
        if (n == 0) continue;
        if (!(ok = mbar_wait(bars + L::kBarQEmpty * 8, (nq_loads & 1) ^ 1, abort_flag))) break;
        ++nq_loads;
        if (lane == 0) {
            mbar_arrive_expect_tx(bars + L::kBarQFull * 8, ((n0 > 0) + (n1 > 0)) * L::kDSlabs * kSlab);
            for (int i = 0; i < 2; ++i) {
                if ((i ? n1 : n0) == 0) continue;
                for (int s = 0; s < L::kDSlabs; ++s)
                    tma_load_3d(qs + (i * L::kDSlabs + s) * kSlab, &a.q_map, bars + L::kBarQFull * 8, s * 64, qrow + i * 128, head);
            }
        }
        for (int t = 0; t < n && ok; ++t) {
            for (int s = 0; s < L::kDSlabs + 2; ++s, ++slab) {
                const uint32_t at = slab % L::kRing;
                if (!(ok = mbar_wait(bars + (L::kBarEmpty + at) * 8, ((slab / L::kRing) & 1) ^ 1, abort_flag))) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(bars + (L::kBarFull + at) * 8, kSlab);
                    if (s < L::kDSlabs)
                        tma_load_3d(ring + at * kSlab, &a.k_map, bars + (L::kBarFull + at) * 8, s * 64, krow + t * 128, kv_head);
                    else
                        tma_load_3d(ring + at * kSlab, &a.v_map, bars + (L::kBarFull + at) * 8, (s - L::kDSlabs) * 64, krow + t * 128, kv_head);
                }
                __syncwarp();
            }
        }
    }
    if (!ok) {
        // another role gave up, or this one: the copies in flight have to land before the CTA may end
        if (lane == 0) give_up(abort_flag, a.status, kStatusGatherWait);
        __syncwarp();
        int never = 0;
        const uint32_t first = slab > static_cast<uint32_t>(L::kRing) ? slab - L::kRing : 0;
        for (uint32_t i = first; i < slab; ++i) mbar_wait(bars + (L::kBarFull + i % L::kRing) * 8, (i / L::kRing) & 1, &never);
        if (nq_loads > 0) mbar_wait(bars + L::kBarQFull * 8, (nq_loads - 1) & 1, &never);
    }
}

// ------------------------------------------------------------------ MMA issue
template <int DQK, bool FP16>
__device__ __forceinline__ void mma_role(const PrefillArgs &a, uint8_t *smem, uint32_t tmem, volatile int *abort_flag, int lane) {
    using L = Smem<DQK>;
    const uint32_t bars = smem_u32(smem + L::kBars), ring = smem_u32(smem + L::kRingAt);
    const uint32_t go = elect_one();
    constexpr uint32_t idesc_qk = umma_idesc_16(FP16, 128, 128, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_16(FP16, 128, 128, 0, 1);
    constexpr uint32_t idesc_pv64 = umma_idesc_16(FP16, 128, 64, 0, 1);
    const uint64_t qd = umma_desc_sw128(smem_u32(smem + L::kQ), 16), kd = umma_desc_sw128(ring, 16), vd = umma_desc_sw128(ring, kSlab);
    constexpr int kPer = L::kDSlabs + 2;
    uint32_t base = 0, nq_loads = 0, np[2] = {0, 0};
    bool ok = true;

    for (int it = 0; ok; ++it) {
        const int slot = it % kRecords;
        if (!(ok = mbar_wait(bars + (L::kBarRecFull + slot) * 8, (it / kRecords) & 1, abort_flag))) break;
        const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * kRecInts;
        const int valid = rec[kRecValid], n0 = rec[kRecN0], n1 = rec[kRecN1], nk = rec[kRecNk];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) break;
        const int n = max(n0, n1);
        if (n == 0) continue;
        if (!(ok = mbar_wait(bars + L::kBarQFull * 8, nq_loads & 1, abort_flag))) break;
        ++nq_loads;

        // S_i = Q_i K(t)^T; the last user of the tile gives its slabs back, the last use of Q the Q tile
        const auto qk = [&](int i, int t) {
            const bool last = i == 1 || t >= n1;
            for (int s = 0; s < L::kDSlabs; ++s) {
                const uint32_t idx = base + t * kPer + s, at = idx % L::kRing;
                if (!mbar_wait(bars + (L::kBarFull + at) * 8, (idx / L::kRing) & 1, abort_flag)) return false;
                tc_fence_after_sync();
                const uint64_t qa = qd + static_cast<uint64_t>(((i * L::kDSlabs + s) * kSlab) >> 4), kb = kd + static_cast<uint64_t>((at * kSlab) >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_bf16_ss_pred(tmem + i * 128, qa + 2 * k, kb + 2 * k, idesc_qk, (s | k) != 0 ? 1u : 0u, go);
                if (last) umma_commit_pred(bars + (L::kBarEmpty + at) * 8, go);
            }
            umma_commit_pred(bars + (L::kBarS + i) * 8, go);
            return true;
        };
        // O_i += P_i V(t)
        const auto pv = [&](int i, int t) {
            const bool first = i == 0 || t >= n0, last = i == 1 || t >= n1;
            const uint32_t idx = base + t * kPer + L::kDSlabs;
            const uint32_t at0 = idx % L::kRing, at1 = (idx + 1) % L::kRing;
            if (!mbar_wait(bars + (L::kBarFull + at0) * 8, (idx / L::kRing) & 1, abort_flag)) return false;
            if (!mbar_wait(bars + (L::kBarFull + at1) * 8, ((idx + 1) / L::kRing) & 1, abort_flag)) return false;
            const int left = nk - t * 128, steps = left >= 128 ? 8 : (left + 15) >> 4;
            if (first && left < 128 && (left & 15) != 0) {
                // the last 16 rows that are multiplied reach past the sequence: what lies there (another sequence's
                // rows, NaN) has weight 0, and 0 x NaN is NaN
                const int r0 = left, r1 = (left + 15) & ~15;
                for (int x = lane; x < (r1 - r0) * 16; x += 32) {
                    const uint32_t dst = ring + ((x & 8) ? at1 : at0) * kSlab + (r0 + (x >> 4)) * 128 + (x & 7) * 16;
                    asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(dst), "r"(0) : "memory");
                }
                fence_async_smem();
                __syncwarp();
            }
            tc_fence_after_sync();
            const uint64_t v0 = vd + static_cast<uint64_t>((at0 * kSlab) >> 4), v1 = vd + static_cast<uint64_t>((at1 * kSlab) >> 4);
            const uint32_t o = tmem + 256 + i * 128, p = tmem + i * 128;
            if (at1 == at0 + 1) {
                for (int k = 0; k < steps; ++k) umma_f16_ts_pred(o, p + k * 8, v0 + k * 128, idesc_pv, (t | k) != 0 ? 1u : 0u, go);
            } else {                             // the pair lies at the two ends of the ring
                for (int k = 0; k < steps; ++k) {
                    umma_f16_ts_pred(o, p + k * 8, v0 + k * 128, idesc_pv64, (t | k) != 0 ? 1u : 0u, go);
                    umma_f16_ts_pred(o + 64, p + k * 8, v1 + k * 128, idesc_pv64, (t | k) != 0 ? 1u : 0u, go);
                }
            }
            if (last) {
                umma_commit_pred(bars + (L::kBarEmpty + at0) * 8, go);
                umma_commit_pred(bars + (L::kBarEmpty + at1) * 8, go);
            }
            return true;
        };
        for (int i = 0; i < 2 && ok; ++i)
            if ((i ? n1 : n0) > 0) {
                ok = qk(i, 0);
                if (n == 1 && (i == 1 || n1 == 0)) umma_commit_pred(bars + L::kBarQEmpty * 8, go);
            }
        for (int t = 0; t < n && ok; ++t) {
            for (int i = 0; i < 2 && ok; ++i) {
                const int ni = i ? n1 : n0;
                if (t >= ni) continue;
                // the half's weights are in tensor memory (and its last item's output has been read)
                if (!(ok = mbar_wait(bars + (L::kBarP + i) * 8, np[i] & 1, abort_flag))) break;
                ++np[i];
                if (!(ok = pv(i, t))) break;
                if (t + 1 < ni) {
                    if (!(ok = qk(i, t + 1))) break;
                    if (t + 2 == n && (i == 1 || t + 1 >= n1)) umma_commit_pred(bars + L::kBarQEmpty * 8, go);
                } else {
                    umma_commit_pred(bars + (L::kBarO + i) * 8, go);
                }
            }
        }
        base += n * kPer;
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

template <int DQK, bool FP16>
__device__ __forceinline__ void softmax_role(const PrefillArgs &a, uint8_t *smem, uint32_t tmem, volatile int *abort_flag, int warp, int lane) {
    using L = Smem<DQK>;
    const uint32_t bars = smem_u32(smem + L::kBars);
    const int half = warp >> 2, lane0 = (warp & 3) * 32;
    const uint32_t s_addr = tmem + half * 128 + (static_cast<uint32_t>(lane0) << 16);
    const uint32_t o_addr = s_addr - half * 128 + 256 + half * 128;
    const int row = half * 128 + lane0 + lane;   // of the item
    const float c = a.scale_log2;
    uint32_t ns = 0, no = 0;
    for (int it = 0;; ++it) {
        const int slot = it % kRecords;
        if (!mbar_wait(bars + (L::kBarRecFull + slot) * 8, (it / kRecords) & 1, abort_flag)) break;
        const volatile int *rec = reinterpret_cast<const int *>(smem + L::kRecs) + slot * kRecInts;
        const int valid = rec[kRecValid], n = rec[half ? kRecN1 : kRecN0], nk = rec[kRecNk], off = rec[kRecOff], rows = rec[kRecRows],
                  head = rec[kRecHead], qrow = rec[kRecQRow];
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + (L::kBarRecEmpty + slot) * 8);
        if (!valid) return;
        const int lim = a.causal ? min(nk, off + row + 1) : nk;                    // keys that this row sees
        const int lim_warp = a.causal ? min(nk, off + half * 128 + lane0 + 1) : nk; // ... and the warp's first row
        float m = -INFINITY;                     // the reference, in log2 units
        uint64_t l2 = 0;                         // two partial sums
        for (int t = 0; t < n; ++t, ++ns) {
            if (!mbar_wait(bars + (L::kBarS + half) * 8, ns & 1, abort_flag)) {
                if (lane == 0) give_up(abort_flag, a.status, kStatusSoftmaxWait);
                return;
            }
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
                for (int j = 0; j < 128; ++j)
                    if (j >= see) s[j] = 0xFF800000u;
            }
            float mx[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) mx[j] = __uint_as_float(s[j]);
#pragma unroll
            for (int j = 4; j < 128; j += 8) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mx[e] = fmaxf(mx[e], j + 4 + e < 128 ? fmaxf(__uint_as_float(s[j + e]), __uint_as_float(s[j + 4 + e])) : __uint_as_float(s[j + e]));
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
            const bool move = top > m + 8.0f;
            if (__any_sync(0xffffffffu, move)) {
                const float to = move ? top : m;
                const float f = move ? fast_exp2(m - to) : 1.0f;         // 0 for the row's first keys
                m = to;
                l2 = mul2(l2, pack2(f, f));
                if (t > 0) {
                    // every earlier product into O_i is complete: the scores of this block were issued behind them
#pragma unroll 1
                    for (int j = 0; j < 128; j += 8) {
                        uint32_t o[8];
                        tmem_ld_x8(o_addr + j, o);
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_x8(o_addr + j, o);
                    }
                }
            }
            const float ref = m == -INFINITY ? 0.0f : -m;
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
            if (lane == 0) mbar_arrive(bars + (L::kBarP + half) * 8);
        }
        float lx, ly;
        unpack2(l2, lx, ly);
        const float l = lx + ly;
        const bool mine = row < rows;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (mine && a.lse != nullptr) a.lse[head * a.lse_hs + qrow + row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
        uint16_t *dst = static_cast<uint16_t *>(a.out) + (qrow + row) * a.o_ts + head * a.o_hs;
        if (n > 0) {
            if (!mbar_wait(bars + (L::kBarO + half) * 8, no & 1, abort_flag)) {
                if (lane == 0) give_up(abort_flag, a.status, kStatusEpilogueWait);
                return;
            }
            ++no;
            tc_fence_after_sync();
        }
#pragma unroll
        for (int j = 0; j < 128; j += 32) {
            uint32_t o[32];
            if (n > 0) {
                tmem_ld_x32_nowait(o_addr + j, o);
                tmem_ld_wait();
            }
            if (mine) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x)      // a row without keys: zeros (the accumulator may hold anything)
                        w[x] = l == 0.0f ? 0u : pack16<FP16>(__uint_as_float(o[e + 2 * x]) * inv, __uint_as_float(o[e + 2 * x + 1]) * inv);
                    *reinterpret_cast<uint4 *>(dst + j + e) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        tc_fence_before_sync();                  // the next item's first product comes behind this warp's next arrival
    }
}

template <int DQK, bool FP16>
__global__ void __launch_bounds__(kThreads, 1) dense_prefill_kernel(const __grid_constant__ PrefillArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using L = Smem<DQK>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kMisc);
    const uint32_t bars = smem_u32(smem + L::kBars);
    if ((smem_u32(smem) & 1023u) != 0u) {        // the swizzled slabs need it
        if (tid == 0) atomicOr(a.status, kStatusSmemLayout);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < L::kRing; ++i) {
            mbar_init(bars + (L::kBarFull + i) * 8, 1);
            mbar_init(bars + (L::kBarEmpty + i) * 8, 1);
        }
        mbar_init(bars + L::kBarQFull * 8, 1);
        mbar_init(bars + L::kBarQEmpty * 8, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars + (L::kBarS + i) * 8, 1);
            mbar_init(bars + (L::kBarP + i) * 8, 4);
            mbar_init(bars + (L::kBarO + i) * 8, 1);
        }
        for (int i = 0; i < kRecords; ++i) {
            mbar_init(bars + (L::kBarRecFull + i) * 8, 1);
            mbar_init(bars + (L::kBarRecEmpty + i) * 8, 9);
        }
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 8) tmem_alloc(smem_u32(smem + L::kMisc + 8), 512);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::kMisc + 8);
    if (warp < 8) {
        regs_inc<kRegsSoftmax>();
        softmax_role<DQK, FP16>(a, smem, tmem, abort_flag, warp, lane);
    } else {
        regs_dec<kRegsOther>();
        if (warp == 8) mma_role<DQK, FP16>(a, smem, tmem, abort_flag, lane);
        else if (warp == 9) loader_role<DQK>(a, smem, abort_flag, lane);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 8) {
        tmem_relinquish();
        tmem_dealloc(tmem, 512);
    }
}

template <int DQK, bool FP16>
int launch(PrefillArgs &a, unsigned grid, cudaStream_t stream) {
    static KernelSetup setup;
    const int rc = setup.get(reinterpret_cast<const void *>(&dense_prefill_kernel<DQK, FP16>), Smem<DQK>::kBytes, &a.status, kRegsLaunch);
    if (rc != 0) return rc;
    dense_prefill_kernel<DQK, FP16><<<grid, kThreads, Smem<DQK>::kBytes, stream>>>(a);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace

int launch_dense_prefill(const smla_prefill_params_t &p, int sm_count, cudaStream_t stream) {
    PrefillArgs a = {};
    const bool fp16 = p.dtype == 1;
    if (!make_slab_map(&a.q_map, fp16, p.q, p.head_dim, p.total_q, p.num_heads, p.q_token_stride * 2, p.q_head_stride * 2, 128))
        return SMLA_EINVAL;
    // without keys no item has a key block, and the maps of k and v are never used
    if (p.total_k > 0 &&
        (!make_slab_map(&a.k_map, fp16, p.k, p.head_dim, p.total_k, p.num_kv_heads, p.k_token_stride * 2, p.k_head_stride * 2, 128) ||
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
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(items, sm_count));
    if (p.head_dim == 192) return fp16 ? launch<192, true>(a, grid, stream) : launch<192, false>(a, grid, stream);
    return fp16 ? launch<128, true>(a, grid, stream) : launch<128, false>(a, grid, stream);
}

}  // namespace smla
