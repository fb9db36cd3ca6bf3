// Dense MLA prefill for sm_100a: attention of packed prompts over keys and values expanded to heads.
//
//   s_ij = scale q_i . k_j   (j <= i + nk - nq with the causal mask),   lse_i = log sum_j exp s_ij,
//   out_i = sum_j exp(s_ij - lse_i) v_j
//
// One pass over the keys with the running maximum m and sum l of the softmax: a block of keys with maximum m'
// turns (m, l, o) into (M, l e^(m-M) + sum e^(s-M), o e^(m-M) + sum e^(s-M) v), M = max(m, m').
//
// One warp per (query, head), 32 keys at a time: a lane scores one key, then owns four of the 128 output dims.
// Bound by instruction issue (no tensor cores).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "smla_internal.h"

namespace smla {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T> __device__ __forceinline__ float2 to_f2(uint32_t w);
template <> __device__ __forceinline__ float2 to_f2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 to_f2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

template <typename T>
__global__ void __launch_bounds__(128) dense_prefill_kernel(const smla_prefill_params_t p) {
    const int lane = threadIdx.x & 31;
    const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (item >= p.total_q * p.num_heads) return;
    const int row = static_cast<int>(item / p.num_heads), h = static_cast<int>(item % p.num_heads);
    // the sequence whose query rows hold `row`
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.cu_seqlens_q[mid] <= row) lo = mid; else hi = mid;
    }
    const int q0 = p.cu_seqlens_q[lo], q1 = p.cu_seqlens_q[lo + 1];
    if (row < q0 || row >= q1) return;
    const int tk = static_cast<int>(p.total_k);
    const int k0 = min(max(p.cu_seqlens_k[lo], 0), tk), k1 = min(max(p.cu_seqlens_k[lo + 1], k0), tk);
    const int nk = k1 - k0;
    const int see = p.causal ? min(nk, max(0, nk - (q1 - 1 - row))) : nk;
    const int hk = h / (p.num_heads / p.num_kv_heads);
    const T *q = static_cast<const T *>(p.q) + row * p.q_token_stride + h * p.q_head_stride;
    const T *k = static_cast<const T *>(p.k) + k0 * p.k_token_stride + hk * p.k_head_stride;
    const T *v = static_cast<const T *>(p.v) + k0 * p.v_token_stride + hk * p.v_head_stride;
    const float c = p.softmax_scale * kLog2e;
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = 0; j0 < see; j0 += 32) {
        float s = -INFINITY;
        if (j0 + lane < see) {
            const uint4 *kr = reinterpret_cast<const uint4 *>(k + (j0 + lane) * p.k_token_stride);
            const uint4 *qr = reinterpret_cast<const uint4 *>(q);
            s = 0.0f;
            for (int d = 0; d < p.head_dim / 8; ++d) {
                const uint4 a = kr[d], b = qr[d];
                const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = to_f2<T>(aw[e]), y = to_f2<T>(bw[e]);
                    s = fmaf(x.x, y.x, s);
                    s = fmaf(x.y, y.y, s);
                }
            }
            s *= c;
        }
        float mx = s;
        for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float M = fmaxf(m, mx);
        const float base = M == -INFINITY ? 0.0f : M;
        const float w = exp2f(s - base), f = exp2f(m - base);
        float sum = w;
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l = l * f + sum;
        m = M;
        for (int e = 0; e < 4; ++e) o[e] *= f;
        const int n = min(32, see - j0);
        for (int j = 0; j < n; ++j) {
            const float pj = __shfl_sync(0xffffffffu, w, j);
            const uint2 a = *reinterpret_cast<const uint2 *>(v + (j0 + j) * p.v_token_stride + lane * 4);
            const float2 x = to_f2<T>(a.x), y = to_f2<T>(a.y);
            o[0] = fmaf(pj, x.x, o[0]);
            o[1] = fmaf(pj, x.y, o[1]);
            o[2] = fmaf(pj, y.x, o[2]);
            o[3] = fmaf(pj, y.y, o[3]);
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    T *out = static_cast<T *>(p.out) + row * p.out_token_stride + h * p.out_head_stride + lane * 4;
    for (int e = 0; e < 4; ++e) out[e] = static_cast<T>(o[e] * inv);
    if (p.softmax_lse && lane == 0) p.softmax_lse[h * p.lse_head_stride + row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace

int launch_dense_prefill(const smla_prefill_params_t &p, int, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>((p.total_q * p.num_heads + 3) / 4);
    if (p.dtype == 0) dense_prefill_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(p);
    else dense_prefill_kernel<__half><<<grid, 128, 0, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace smla
