// Score-modified attention on plain FFMA: the kernels that take every type, every head dimension up
// to 256 and every stride.  float32 tensors and layouts that TMA cannot describe run here; 16-bit
// tensors otherwise run on the tensor-core kernels.
//
// One warp owns one output row.  Forward and grad_q walk the row's keys in chunks of 32: lane t
// forms the whole score of key t (its K row is contiguous, so the 32 rows stream through L1), the
// warp keeps one running maximum and sum, and for the second product each lane owns every 32nd
// column while the chunk's 32 weights go round by shuffle.  grad_k and grad_v are the same with the
// roles of queries and keys exchanged, over every query head that shares the key head, so no two
// warps add into one place and sums run in a fixed order.  A key outside the row's range is never
// multiplied in, whatever it holds.
//
// 4 (forward) to 14 (gradients, which form every score twice) head_dim operations per score at FFMA rate, with every
// operand re-read from L1/L2 by each warp: bound by load issue, not by HBM.

#include <math_constants.h>

#include "score_attention.h"

namespace sm120 {

constexpr int SIMT_WARPS = 4;
constexpr int SIMT_MAX_D = 256;
constexpr int SIMT_COLS = SIMT_MAX_D / 32;     // columns per lane

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float x, float* y) { *y = x; }
__device__ __forceinline__ void from_f(float x, __half* y) { *y = __float2half_rn(x); }
__device__ __forceinline__ void from_f(float x, __nv_bfloat16* y) { *y = __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ float dot_row(const float* a, const T* b, int d) {
    float s = 0.0f;
    for (int c = 0; c < d; ++c) s = fmaf(a[c], to_f(b[c]), s);
    return s;
}

// z of a raw product; `curve` gets tanh(x / softcap) (0 without a cap, so that 1 - curve^2 is the derivative's factor)
__device__ __forceinline__ float modified_score(float dot, const ScoreParams& p, float slope, int distance, float& curve) {
    float z = dot * p.scale;
    curve = 0.0f;
    if (p.softcap > 0.0f) {
        curve = tanhf(z / p.softcap);
        z = curve * p.softcap;
    }
    return z - slope * static_cast<float>(distance);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// out row (b, h, i).  TOKEN: the single-token form, keys [shared prefix | own cache].
template <typename T, bool TOKEN>
__global__ void __launch_bounds__(SIMT_WARPS * 32)
sa_simt_forward_kernel(const ScoreParams p) {
    __shared__ float q_s[SIMT_WARPS][SIMT_MAX_D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * SIMT_WARPS + warp;
    if (row >= static_cast<int64_t>(p.batch) * p.heads * p.seq_q) return;
    const int i = static_cast<int>(row % p.seq_q);
    const int64_t bh = row / p.seq_q;
    const int h = static_cast<int>(bh % p.heads), b = static_cast<int>(bh / p.heads), kvh = h / p.group;
    const T* q = static_cast<const T*>(p.q) + b * p.q_st[0] + h * p.q_st[1] + i * p.q_st[2];
    const T* k = static_cast<const T*>(p.k) + b * p.k_st[0] + kvh * p.k_st[1];
    const T* v = static_cast<const T*>(p.v) + b * p.v_st[0] + kvh * p.v_st[1];
    const T* pk = TOKEN ? static_cast<const T*>(p.prefix_k) + kvh * p.pk_st[0] : nullptr;
    const T* pv = TOKEN ? static_cast<const T*>(p.prefix_v) + kvh * p.pv_st[0] : nullptr;
    int lo, hi, pos;
    if (TOKEN) {
        lo = 0;
        hi = p.prefix_len + min(max(p.key_lengths[b], 0), p.seq_k);
        pos = hi - 1;
    } else {
        sa_row_range(p, b, i, lo, hi);
        pos = i + p.seq_k - p.seq_q;
    }
    for (int c = lane; c < p.head_dim; c += 32) q_s[warp][c] = to_f(q[c]);
    __syncwarp();
    const float slope = p.slopes != nullptr ? p.slopes[h] : 0.0f;
    float m = -CUDART_INF_F, l = 0.0f, acc[SIMT_COLS];
#pragma unroll
    for (int t = 0; t < SIMT_COLS; ++t) acc[t] = 0.0f;
    for (int j0 = lo; j0 < hi; j0 += 32) {
        const int j = j0 + lane;
        float z = -CUDART_INF_F, curve;
        if (j < hi) {
            const T* kr = TOKEN && j < p.prefix_len ? pk + j * p.pk_st[1] : k + (TOKEN ? j - p.prefix_len : j) * p.k_st[2];
            z = modified_score(dot_row(q_s[warp], kr, p.head_dim), p, slope, abs(pos - j), curve);
        }
        const float m_new = fmaxf(m, warp_max(z)), m_use = m_new == -CUDART_INF_F ? 0.0f : m_new;
        const float w = j < hi ? expf(z - m_use) : 0.0f, fade = expf(m - m_use);
        l = l * fade + warp_sum(w);
#pragma unroll
        for (int t = 0; t < SIMT_COLS; ++t) acc[t] *= fade;
        const int n = min(32, hi - j0);
        for (int s = 0; s < n; ++s) {
            const float ws = __shfl_sync(0xFFFFFFFFu, w, s);
            const int js = j0 + s;
            const T* vr = TOKEN && js < p.prefix_len ? pv + js * p.pv_st[1] : v + (TOKEN ? js - p.prefix_len : js) * p.v_st[2];
#pragma unroll
            for (int t = 0; t < SIMT_COLS; ++t)
                if (lane + 32 * t < p.head_dim) acc[t] = fmaf(ws, to_f(vr[lane + 32 * t]), acc[t]);
        }
        m = m_new;
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);      // a NaN sum stays one
    T* out = static_cast<T*>(p.out) + b * p.o_st[0] + h * p.o_st[1] + i * p.o_st[2];
#pragma unroll
    for (int t = 0; t < SIMT_COLS; ++t)
        if (lane + 32 * t < p.head_dim) from_f(acc[t] * inv, out + lane + 32 * t);
    if (p.lse != nullptr && lane == 0) p.lse[row] = l == 0.0f ? -CUDART_INF_F : m + logf(l);
}

// neg_lse, neg_delta and ranges of one row per warp, rows behind seq_q included.  One pass over out and grad_out.
template <typename T>
__global__ void __launch_bounds__(SIMT_WARPS * 32)
sa_grad_prepare_kernel(const ScoreParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * SIMT_WARPS + warp;
    if (row >= static_cast<int64_t>(p.batch) * p.heads * p.seq_q_pad) return;
    const int i = static_cast<int>(row % p.seq_q_pad);
    const int64_t bh = row / p.seq_q_pad;
    const int h = static_cast<int>(bh % p.heads), b = static_cast<int>(bh / p.heads);
    float neg_lse = -CUDART_INF_F, neg_delta = 0.0f;
    int2 range = make_int2(0, 0);
    if (i < p.seq_q) {
        const T* o = static_cast<const T*>(p.out) + b * p.o_st[0] + h * p.o_st[1] + i * p.o_st[2];
        const T* g = static_cast<const T*>(p.grad_out) + b * p.go_st[0] + h * p.go_st[1] + i * p.go_st[2];
        float d = 0.0f;
        for (int c = lane; c < p.head_dim; c += 32) d = fmaf(to_f(o[c]), to_f(g[c]), d);
        d = warp_sum(d);
        sa_row_range(p, b, i, range.x, range.y);
        const float lse = p.lse[bh * p.seq_q + i];
        if (range.x < range.y && lse != -CUDART_INF_F) {
            neg_lse = -lse * SA_LOG2E;
            neg_delta = -d;
        }
    }
    if (lane == 0) {
        p.neg_lse[row] = neg_lse;
        p.neg_delta[row] = neg_delta;
        if (h == 0) p.ranges[static_cast<int64_t>(b) * p.seq_q_pad + i] = range;
    }
}

// dx (the gradient of the scaled product) and P of one score
__device__ __forceinline__ float score_grad(float dot, float dp, float neg_lse, float neg_delta, const ScoreParams& p, float slope, int distance, float& prob) {
    float curve;
    const float z = modified_score(dot, p, slope, distance, curve);
    prob = exp2f(z * SA_LOG2E + neg_lse);
    return prob * (dp + neg_delta) * (1.0f - curve * curve);
}

template <typename T>
__global__ void __launch_bounds__(SIMT_WARPS * 32)
sa_simt_grad_q_kernel(const ScoreParams p) {
    __shared__ float q_s[SIMT_WARPS][SIMT_MAX_D], g_s[SIMT_WARPS][SIMT_MAX_D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * SIMT_WARPS + warp;
    if (row >= static_cast<int64_t>(p.batch) * p.heads * p.seq_q) return;
    const int i = static_cast<int>(row % p.seq_q);
    const int64_t bh = row / p.seq_q;
    const int h = static_cast<int>(bh % p.heads), b = static_cast<int>(bh / p.heads), kvh = h / p.group;
    const T* q = static_cast<const T*>(p.q) + b * p.q_st[0] + h * p.q_st[1] + i * p.q_st[2];
    const T* g = static_cast<const T*>(p.grad_out) + b * p.go_st[0] + h * p.go_st[1] + i * p.go_st[2];
    const T* k = static_cast<const T*>(p.k) + b * p.k_st[0] + kvh * p.k_st[1];
    const T* v = static_cast<const T*>(p.v) + b * p.v_st[0] + kvh * p.v_st[1];
    const int2 range = p.ranges[static_cast<int64_t>(b) * p.seq_q_pad + i];
    const float neg_lse = p.neg_lse[bh * p.seq_q_pad + i], neg_delta = p.neg_delta[bh * p.seq_q_pad + i];
    const int pos = i + p.seq_k - p.seq_q;
    for (int c = lane; c < p.head_dim; c += 32) {
        q_s[warp][c] = to_f(q[c]);
        g_s[warp][c] = to_f(g[c]);
    }
    __syncwarp();
    const float slope = p.slopes != nullptr ? p.slopes[h] : 0.0f;
    float acc[SIMT_COLS];
#pragma unroll
    for (int t = 0; t < SIMT_COLS; ++t) acc[t] = 0.0f;
    if (neg_lse != -CUDART_INF_F) {
        for (int j0 = range.x; j0 < range.y; j0 += 32) {
            const int j = j0 + lane;
            float dx = 0.0f, prob;
            if (j < range.y)
                dx = score_grad(dot_row(q_s[warp], k + j * p.k_st[2], p.head_dim), dot_row(g_s[warp], v + j * p.v_st[2], p.head_dim), neg_lse,
                                neg_delta, p, slope, abs(pos - j), prob);
            const int n = min(32, range.y - j0);
            for (int s = 0; s < n; ++s) {
                const float ws = __shfl_sync(0xFFFFFFFFu, dx, s);
                const T* kr = k + (j0 + s) * p.k_st[2];
#pragma unroll
                for (int t = 0; t < SIMT_COLS; ++t)
                    if (lane + 32 * t < p.head_dim) acc[t] = fmaf(ws, to_f(kr[lane + 32 * t]), acc[t]);
            }
        }
    }
    T* gq = static_cast<T*>(p.grad_q) + b * p.gq_st[0] + h * p.gq_st[1] + i * p.gq_st[2];
#pragma unroll
    for (int t = 0; t < SIMT_COLS; ++t)
        if (lane + 32 * t < p.head_dim) from_f(acc[t] * p.scale, gq + lane + 32 * t);
}

template <typename T>
__global__ void __launch_bounds__(SIMT_WARPS * 32)
sa_simt_grad_kv_kernel(const ScoreParams p) {
    __shared__ float k_s[SIMT_WARPS][SIMT_MAX_D], v_s[SIMT_WARPS][SIMT_MAX_D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * SIMT_WARPS + warp;
    if (row >= static_cast<int64_t>(p.batch) * p.kv_heads * p.seq_k) return;
    const int j = static_cast<int>(row % p.seq_k);
    const int64_t bh = row / p.seq_k;
    const int kvh = static_cast<int>(bh % p.kv_heads), b = static_cast<int>(bh / p.kv_heads);
    const T* k = static_cast<const T*>(p.k) + b * p.k_st[0] + kvh * p.k_st[1] + j * p.k_st[2];
    const T* v = static_cast<const T*>(p.v) + b * p.v_st[0] + kvh * p.v_st[1] + j * p.v_st[2];
    for (int c = lane; c < p.head_dim; c += 32) {
        k_s[warp][c] = to_f(k[c]);
        v_s[warp][c] = to_f(v[c]);
    }
    __syncwarp();
    const int2* ranges = p.ranges + static_cast<int64_t>(b) * p.seq_q_pad;
    float dk[SIMT_COLS], dv[SIMT_COLS];
#pragma unroll
    for (int t = 0; t < SIMT_COLS; ++t) dk[t] = dv[t] = 0.0f;
    for (int h = kvh * p.group; h < (kvh + 1) * p.group; ++h) {
        const T* q = static_cast<const T*>(p.q) + b * p.q_st[0] + h * p.q_st[1];
        const T* g = static_cast<const T*>(p.grad_out) + b * p.go_st[0] + h * p.go_st[1];
        const int64_t stat_row = (static_cast<int64_t>(b) * p.heads + h) * p.seq_q_pad;
        const float slope = p.slopes != nullptr ? p.slopes[h] : 0.0f;
        for (int i0 = 0; i0 < p.seq_q; i0 += 32) {
            const int i = i0 + lane;
            bool sees = false;
            float dx = 0.0f, prob = 0.0f;
            if (i < p.seq_q) {
                const int2 range = ranges[i];
                const float neg_lse = p.neg_lse[stat_row + i];
                sees = range.x <= j && j < range.y && neg_lse != -CUDART_INF_F;
                if (sees)
                    dx = score_grad(dot_row(k_s[warp], q + i * p.q_st[2], p.head_dim), dot_row(v_s[warp], g + i * p.go_st[2], p.head_dim), neg_lse,
                                    p.neg_delta[stat_row + i], p, slope, abs(i + p.seq_k - p.seq_q - j), prob);
            }
            unsigned left = __ballot_sync(0xFFFFFFFFu, sees);
            while (left != 0u) {
                const int s = __ffs(left) - 1;
                left &= left - 1;
                const float ds = __shfl_sync(0xFFFFFFFFu, dx, s), ps = __shfl_sync(0xFFFFFFFFu, prob, s);
                const T* qr = q + (i0 + s) * p.q_st[2];
                const T* gr = g + (i0 + s) * p.go_st[2];
#pragma unroll
                for (int t = 0; t < SIMT_COLS; ++t)
                    if (lane + 32 * t < p.head_dim) {
                        dk[t] = fmaf(ds, to_f(qr[lane + 32 * t]), dk[t]);
                        dv[t] = fmaf(ps, to_f(gr[lane + 32 * t]), dv[t]);
                    }
            }
        }
    }
    T* gk = static_cast<T*>(p.grad_k) + b * p.gk_st[0] + kvh * p.gk_st[1] + j * p.gk_st[2];
    T* gv = static_cast<T*>(p.grad_v) + b * p.gv_st[0] + kvh * p.gv_st[1] + j * p.gv_st[2];
#pragma unroll
    for (int t = 0; t < SIMT_COLS; ++t)
        if (lane + 32 * t < p.head_dim) {
            from_f(dk[t] * p.scale, gk + lane + 32 * t);
            from_f(dv[t], gv + lane + 32 * t);
        }
}

// one warp per row; the launch functions have checked that the block counts fit
static unsigned row_blocks(int64_t rows) { return static_cast<unsigned>((rows + SIMT_WARPS - 1) / SIMT_WARPS); }

#define SA_BY_TYPE(KERNEL_OF, ROWS)                                                                       \
    do {                                                                                                  \
        const int64_t rows_ = (ROWS);                                                                     \
        if (rows_ == 0) break;                                                                            \
        const unsigned blocks_ = row_blocks(rows_);                                                       \
        if (p.dtype == SM120_DTYPE_FLOAT32) KERNEL_OF(float)<<<blocks_, SIMT_WARPS * 32, 0, stream>>>(p); \
        else if (p.dtype == SM120_DTYPE_FLOAT16) KERNEL_OF(__half)<<<blocks_, SIMT_WARPS * 32, 0, stream>>>(p); \
        else KERNEL_OF(__nv_bfloat16)<<<blocks_, SIMT_WARPS * 32, 0, stream>>>(p);                        \
    } while (0)

cudaError_t sa_simt_forward(const ScoreParams& p, cudaStream_t stream) {
#define SA_K(T) sa_simt_forward_kernel<T, false>
    SA_BY_TYPE(SA_K, static_cast<int64_t>(p.batch) * p.heads * p.seq_q);
#undef SA_K
    return cudaGetLastError();
}

cudaError_t sa_simt_decode(const ScoreParams& p, cudaStream_t stream) {
#define SA_K(T) sa_simt_forward_kernel<T, true>
    SA_BY_TYPE(SA_K, static_cast<int64_t>(p.batch) * p.heads);
#undef SA_K
    return cudaGetLastError();
}

cudaError_t sa_simt_grad(const ScoreParams& p, cudaStream_t stream) {
#define SA_K(T) sa_grad_prepare_kernel<T>
    SA_BY_TYPE(SA_K, static_cast<int64_t>(p.batch) * p.heads * p.seq_q_pad);
#undef SA_K
#define SA_K(T) sa_simt_grad_q_kernel<T>
    SA_BY_TYPE(SA_K, static_cast<int64_t>(p.batch) * p.heads * p.seq_q);
#undef SA_K
#define SA_K(T) sa_simt_grad_kv_kernel<T>
    SA_BY_TYPE(SA_K, static_cast<int64_t>(p.batch) * p.kv_heads * p.seq_k);
#undef SA_K
    return cudaGetLastError();
}

}  // namespace sm120
