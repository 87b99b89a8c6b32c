// Internal declarations of the score-modified attention (sm120_launch_score_attention and its
// gradient and single-token forms): the resolved parameters that every kernel family takes, the
// row's key range, and the launch functions.  The mathematics is stated with
// SM120ScoreAttentionDesc in the public header.
#pragma once

#include "gemm_common.h"

namespace sm120 {

constexpr float SA_LOG2E = 1.4426950408889634f;
constexpr float SA_LN2 = 0.69314718055994531f;
constexpr int SA_ROW_PAD = 128;      // per-row arrays in the workspace are padded to a whole number of tiles

struct ScoreParams {
    int batch, heads, kv_heads, group;         // group = heads / kv_heads
    int seq_q, seq_k, head_dim, dtype;
    int seq_q_pad;                             // seq_q rounded up to SA_ROW_PAD
    int causal, num_documents;
    float scale, softcap;                      // softcap 0 = none
    const float* slopes;
    const int32_t* document_offsets;
    const int32_t* prefix_lengths;
    const void *q, *k, *v;
    void* out;
    float* lse;
    int64_t q_st[3], k_st[3], v_st[3], o_st[3];
    const void* grad_out;
    void *grad_q, *grad_k, *grad_v;
    int64_t go_st[3], gq_st[3], gk_st[3], gv_st[3];
    const int32_t* key_lengths;
    const void *prefix_k, *prefix_v;
    int prefix_len;
    int64_t pk_st[2], pv_st[2];
    // gradient workspace
    float2* stats;                             // [batch * heads][seq_q_pad]: {lse in log2 units, D}; +inf marks rows without keys
    int2* ranges;                              // [batch][seq_q_pad]: the keys [x, y) that a row sees
};

// Key range [lo, hi) of query row i of entry b.  Both ends never decrease with i, so the keys that
// consecutive rows see are one range as well, from the first row's lo to the last row's hi.
__device__ __forceinline__ void sa_row_range(const ScoreParams& p, int b, int i, int& lo, int& hi) {
    const int pos = i + p.seq_k - p.seq_q;
    lo = 0;
    hi = p.seq_k;
    if (p.num_documents > 0) {
        const int32_t* offs = p.document_offsets + static_cast<int64_t>(b) * (p.num_documents + 1);
        // first entry behind pos: documents may be empty, their repeated offsets are skipped
        int first = 0, last = p.num_documents + 1;
        while (first < last) {
            const int mid = (first + last) >> 1;
            if (__ldg(offs + mid) <= pos) first = mid + 1;
            else last = mid;
        }
        lo = __ldg(offs + max(first - 1, 0));
        hi = __ldg(offs + min(first, p.num_documents));
        lo = min(max(lo, 0), p.seq_k);
        hi = min(max(hi, lo), p.seq_k);        // outside every document both are the same offset: no key
    }
    if (p.causal) {
        int limit = pos + 1;
        if (p.prefix_lengths != nullptr) limit = max(limit, __ldg(p.prefix_lengths + b));
        hi = max(min(hi, limit), lo);
    }
}

// shared by the two kernel families (score_attention_simt.cu): fills stats and ranges
cudaError_t sa_grad_prepare_launch(const ScoreParams& p, cudaStream_t stream);

// Plain FFMA kernels: any type, head dimension up to 256, any strides.
cudaError_t sa_simt_forward(const ScoreParams& p, cudaStream_t stream);
cudaError_t sa_simt_grad(const ScoreParams& p, cudaStream_t stream);
cudaError_t sa_simt_decode(const ScoreParams& p, cudaStream_t stream);

// Tensor-core forward (score_attention_tcgen05.cuh): 16-bit types, head dimension a multiple of 8 up to 128, operands that TMA can address.
bool sa_tc_forward_supported(const ScoreParams& p);
cudaError_t sa_tc_forward(const ScoreParams& p, int device, cudaStream_t stream);

// Launcher state shared with launcher.cu: the current device (compute capability 10.x), the wait limit, and the
// bookkeeping behind sm120_get_launch_count / sm120_get_last_kernel_name.
cudaError_t current_device(int* device, int* sm_count);
uint64_t launch_wait_limit_ns();
void note_launches(const char* name, int count);

}  // namespace sm120
