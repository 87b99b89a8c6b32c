// Internal declarations of the score-modified attention (sm120_launch_score_attention and its
// gradient and single-token forms): the resolved parameters that every kernel family takes, the
// row's key range, and the launch functions.  The mathematics is stated with
// SM120ScoreAttentionDesc in the public header.
#pragma once

#include "gemm_common.h"

namespace sm120 {

constexpr float SA_LOG2E = 1.4426950408889634f;
constexpr float SA_LN2 = 0.69314718055994531f;
constexpr int SA_ROW_PAD = 128;      // per-row arrays in the workspace have rows behind the last: a copy of SA_GRAD_TILE rows from any row stays inside
constexpr int SA_GRAD_TILE = 64;     // streamed rows per tile of the gradient kernels

struct ScoreParams {
    int batch, heads, kv_heads, group;         // group = heads / kv_heads
    int seq_q, seq_k, head_dim, dtype;
    int seq_q_pad;                             // seq_q + SA_GRAD_TILE rounded up to SA_ROW_PAD
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
    float* neg_lse;                            // [batch * heads][seq_q_pad]: -lse in log2 units; -inf (P = 0) for rows without keys and behind seq_q
    float* neg_delta;                          // [batch * heads][seq_q_pad]: -<grad_out, out>
    int2* ranges;                              // [batch][seq_q_pad]: the keys [x, y) that a row sees
};

// The document of entry b that holds position pos, as clamped key positions.  A position outside every document gets an empty
// range at the nearest end, so both ends never decrease with pos.
__device__ __forceinline__ void sa_document(const ScoreParams& p, int b, int pos, int& lo, int& hi) {
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
    hi = min(max(hi, lo), p.seq_k);
}

// Key range [lo, hi) of query row i of entry b.  Both ends never decrease with i, so the keys that
// consecutive rows see are one range as well, from the first row's lo to the last row's hi.
__device__ __forceinline__ void sa_row_range(const ScoreParams& p, int b, int i, int& lo, int& hi) {
    const int pos = i + p.seq_k - p.seq_q;
    lo = 0;
    hi = p.seq_k;
    if (p.num_documents > 0) sa_document(p, b, pos, lo, hi);
    if (p.causal) {
        int limit = pos + 1;
        if (p.prefix_lengths != nullptr) limit = max(limit, __ldg(p.prefix_lengths + b));
        hi = max(min(hi, limit), lo);
    }
}

// Query rows [first, end) of entry b that see any of the keys [j0, j1): one range, by the same argument.
__device__ __forceinline__ void sa_query_range(const ScoreParams& p, int b, int j0, int j1, int& first, int& end) {
    const int first_pos = p.seq_k - p.seq_q;
    int from = 0, to = p.seq_q;
    if (p.num_documents > 0) {
        int lo, hi, other;
        sa_document(p, b, j0, lo, other);
        sa_document(p, b, j1 - 1, other, hi);
        from = max(from, lo - first_pos);
        to = min(to, hi - first_pos);
    }
    if (p.causal && !(p.prefix_lengths != nullptr && j0 < __ldg(p.prefix_lengths + b))) from = max(from, j0 - first_pos);
    first = from;
    end = max(to, from);
}

// Plain FFMA kernels: any type, head dimension up to 256, any strides.
cudaError_t sa_simt_forward(const ScoreParams& p, cudaStream_t stream);
cudaError_t sa_simt_grad(const ScoreParams& p, cudaStream_t stream);      // three launches
cudaError_t sa_simt_decode(const ScoreParams& p, cudaStream_t stream);

// Tensor-core forward (score_attention_tcgen05.cuh): 16-bit types, head dimension a multiple of 8 up to 128, operands that TMA can address.
bool sa_tc_forward_supported(const ScoreParams& p);
cudaError_t sa_tc_forward(const ScoreParams& p, int device, cudaStream_t stream);

// The batch's single-token queries against the shared prefix on the same kernel: row tiles of 128 / group entries, the key tiles cut into
// `parts` parts of `tiles_per_part`, results in part_out / part_lse (score_attention_decode.cu).
cudaError_t sa_tc_prefix(const ScoreParams& p, int parts, int tiles_per_part, float* part_out, float* part_lse, int device, cudaStream_t stream);

// Tensor-core gradients (score_attention_grad_tcgen05.cuh); the same limits.  `workspace` is what sa_tc_grad_workspace asks for behind the
// three per-row arrays.
bool sa_tc_grad_supported(const ScoreParams& p);
size_t sa_tc_grad_workspace(const ScoreParams& p, int sms);
cudaError_t sa_tc_grad(const ScoreParams& p, void* workspace, int device, int sms, cudaStream_t stream, int* launches);

// Single-token form for 16-bit types (score_attention_decode.cu): the same limits.
bool sa_tma_ok(const void* ptr, const int64_t* strides, const int64_t* extents, int count);
bool sa_tc_types_ok(const ScoreParams& p);
bool sa_tc_decode_supported(const ScoreParams& p);
size_t sa_tc_decode_workspace(const ScoreParams& p, int sms);
cudaError_t sa_tc_decode(const ScoreParams& p, void* workspace, int device, int sms, cudaStream_t stream, int* launches);

// Launcher state shared with launcher.cu: the current device (compute capability 10.x), the wait limit, and the
// bookkeeping behind sm120_get_launch_count / sm120_get_last_kernel_name.
cudaError_t current_device(int* device, int* sm_count);
uint64_t launch_wait_limit_ns();
void note_launches(const char* name, int count);

}  // namespace sm120
