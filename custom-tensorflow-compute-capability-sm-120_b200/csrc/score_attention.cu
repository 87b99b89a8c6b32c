// C entry points of the score-modified attention: argument checks, workspaces and the choice of the
// kernel family.  The mathematics is stated with SM120ScoreAttentionDesc in the public header.

#include <string.h>

#include "score_attention.h"

namespace sm120 {
namespace {

constexpr int64_t INT31 = (1ll << 31) - 1;
constexpr int64_t MAX_ROWS = 1ll << 32;       // rows of one launch (four to a block of the plain kernels)

// written tensors: no two elements may share an address through a stride of 0
bool distinct(const int64_t (&st)[3], int64_t a, int64_t b, int64_t c) { return (a <= 1 || st[0] > 0) && (b <= 1 || st[1] > 0) && (c <= 1 || st[2] > 0); }

enum class Form { FORWARD, GRADIENT, TOKEN };

// Checks what can be checked without a device and fills `p`.  *empty: nothing to compute.
cudaError_t resolve(const SM120ScoreAttentionDesc* d, Form form, ScoreParams* p, bool* empty) {
    *empty = false;
    if (d == nullptr || d->struct_size != sizeof(SM120ScoreAttentionDesc)) return cudaErrorInvalidValue;
    if (d->dtype != SM120_DTYPE_FLOAT32 && d->dtype != SM120_DTYPE_FLOAT16 && d->dtype != SM120_DTYPE_BFLOAT16) return cudaErrorInvalidValue;
    if (d->batch < 0 || d->seq_q < 0 || d->seq_k < 0 || d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads != 0) return cudaErrorInvalidValue;
    if (d->head_dim < 1 || d->head_dim > 256) return cudaErrorInvalidValue;
    if (d->batch > 65535 || d->heads > 65535 || d->prefix_len < 0) return cudaErrorInvalidValue;
    // positions and their differences are 32-bit: a quarter of the range leaves room for tiles behind the end
    if (d->seq_q > INT31 / 4 || d->seq_k > INT31 / 4 || d->prefix_len > INT31 / 4) return cudaErrorInvalidValue;
    if (!(d->softcap >= 0.0f) || d->softcap > 1e30f || !(d->scale == d->scale)) return cudaErrorInvalidValue;
    if (d->num_documents < 0 || d->num_documents > INT31 / 2 || (d->batch > 0 && (d->num_documents > 0) != (d->document_offsets != nullptr))) return cudaErrorInvalidValue;
    if (d->prefix_lengths != nullptr && (!d->causal || d->num_documents > 0)) return cudaErrorInvalidValue;
    const bool token = form == Form::TOKEN;
    if (token && (d->seq_q != 1 || d->causal || d->num_documents > 0 || d->prefix_lengths != nullptr)) return cudaErrorInvalidValue;
    if (!token && (d->key_lengths != nullptr || d->prefix_len != 0)) return cudaErrorInvalidValue;
    if (d->batch * d->heads * (d->seq_q + SA_GRAD_TILE + SA_ROW_PAD) > MAX_ROWS || d->batch * d->kv_heads * d->seq_k > MAX_ROWS) return cudaErrorInvalidValue;
    for (int a = 0; a < 3; ++a) {
        if (d->q_stride[a] < 0 || d->k_stride[a] < 0 || d->v_stride[a] < 0 || d->out_stride[a] < 0) return cudaErrorInvalidValue;
        if (form == Form::GRADIENT && (d->grad_out_stride[a] < 0 || d->grad_q_stride[a] < 0 || d->grad_k_stride[a] < 0 || d->grad_v_stride[a] < 0))
            return cudaErrorInvalidValue;
    }
    if (d->prefix_k_stride[0] < 0 || d->prefix_k_stride[1] < 0 || d->prefix_v_stride[0] < 0 || d->prefix_v_stride[1] < 0) return cudaErrorInvalidValue;
    if (form == Form::GRADIENT) *empty = d->batch == 0 || (d->seq_q == 0 && d->seq_k == 0);
    else *empty = d->batch == 0 || d->seq_q == 0;
    if (*empty) return cudaSuccess;
    if (d->seq_q > 0 && (d->q == nullptr || d->out == nullptr)) return cudaErrorInvalidValue;
    if (d->seq_k > 0 && (d->k == nullptr || d->v == nullptr)) return cudaErrorInvalidValue;
    if (token && (d->key_lengths == nullptr || (d->prefix_len > 0 && (d->prefix_k == nullptr || d->prefix_v == nullptr)))) return cudaErrorInvalidValue;
    if (form == Form::GRADIENT) {
        if (d->seq_q > 0 && (d->lse == nullptr || d->grad_out == nullptr || d->grad_q == nullptr)) return cudaErrorInvalidValue;
        if (d->seq_k > 0 && (d->grad_k == nullptr || d->grad_v == nullptr)) return cudaErrorInvalidValue;
    }
    if (form == Form::GRADIENT) {
        if (!distinct(d->grad_q_stride, d->batch, d->heads, d->seq_q) || !distinct(d->grad_k_stride, d->batch, d->kv_heads, d->seq_k) ||
            !distinct(d->grad_v_stride, d->batch, d->kv_heads, d->seq_k))
            return cudaErrorInvalidValue;
    } else if (!distinct(d->out_stride, d->batch, d->heads, d->seq_q)) {
        return cudaErrorInvalidValue;
    }
    p->batch = static_cast<int>(d->batch); p->heads = static_cast<int>(d->heads); p->kv_heads = static_cast<int>(d->kv_heads);
    p->group = p->heads / p->kv_heads;
    p->seq_q = static_cast<int>(d->seq_q); p->seq_k = static_cast<int>(d->seq_k); p->head_dim = static_cast<int>(d->head_dim);
    p->seq_q_pad = (p->seq_q + SA_GRAD_TILE + SA_ROW_PAD - 1) / SA_ROW_PAD * SA_ROW_PAD;
    p->dtype = d->dtype; p->causal = d->causal != 0; p->num_documents = d->num_documents;
    p->scale = d->scale; p->softcap = d->softcap;
    p->slopes = d->alibi_slopes; p->document_offsets = d->document_offsets; p->prefix_lengths = d->prefix_lengths;
    p->q = d->q; p->k = d->k; p->v = d->v; p->out = d->out; p->lse = d->lse;
    p->grad_out = d->grad_out; p->grad_q = d->grad_q; p->grad_k = d->grad_k; p->grad_v = d->grad_v;
    for (int a = 0; a < 3; ++a) {
        p->q_st[a] = d->q_stride[a]; p->k_st[a] = d->k_stride[a]; p->v_st[a] = d->v_stride[a]; p->o_st[a] = d->out_stride[a];
        p->go_st[a] = d->grad_out_stride[a]; p->gq_st[a] = d->grad_q_stride[a]; p->gk_st[a] = d->grad_k_stride[a]; p->gv_st[a] = d->grad_v_stride[a];
    }
    p->key_lengths = d->key_lengths; p->prefix_k = d->prefix_k; p->prefix_v = d->prefix_v; p->prefix_len = static_cast<int>(d->prefix_len);
    for (int a = 0; a < 2; ++a) {
        p->pk_st[a] = d->prefix_k_stride[a];
        p->pv_st[a] = d->prefix_v_stride[a];
    }
    return cudaSuccess;
}

// the three arrays of the gradient workspace; seq_q_pad keeps each a multiple of 16 bytes
size_t stats_bytes(const ScoreParams& p) { return static_cast<size_t>(p.batch) * p.heads * p.seq_q_pad * sizeof(float); }
size_t ranges_bytes(const ScoreParams& p) { return static_cast<size_t>(p.batch) * p.seq_q_pad * sizeof(int2); }
size_t row_bytes(const ScoreParams& p) { return 2 * stats_bytes(p) + ranges_bytes(p); }
size_t grad_workspace(const ScoreParams& p, int sms) { return row_bytes(p) + (sa_tc_grad_supported(p) ? sa_tc_grad_workspace(p, sms) : 0); }

bool workspace_ok(const SM120ScoreAttentionDesc* d, size_t need) {
    return need == 0 || (d->workspace != nullptr && (reinterpret_cast<uintptr_t>(d->workspace) & 15u) == 0 && d->workspace_bytes >= need);
}

}  // namespace
}  // namespace sm120

using namespace sm120;

extern "C" {

void sm120_score_attention_desc_init(SM120ScoreAttentionDesc* desc) {
    if (desc == nullptr) return;
    memset(desc, 0, sizeof(*desc));
    desc->struct_size = sizeof(*desc);
    desc->batch = desc->heads = desc->kv_heads = 1;
    desc->scale = 1.0f;
}

cudaError_t sm120_launch_score_attention(const SM120ScoreAttentionDesc* desc) {
    ScoreParams p{};
    bool empty = false;
    cudaError_t e = resolve(desc, Form::FORWARD, &p, &empty);
    if (e != cudaSuccess || empty) return e;
    int device = 0, sms = 0;
    e = current_device(&device, &sms);
    if (e != cudaSuccess) return e;
    const bool tc = sa_tc_forward_supported(p);
    e = tc ? sa_tc_forward(p, device, desc->stream) : sa_simt_forward(p, desc->stream);
    if (e == cudaSuccess) note_launches(tc ? (p.head_dim > 64 ? "score_attention_tcgen05_d128" : "score_attention_tcgen05_d64") : "score_attention_simt", 1);
    return e;
}

size_t sm120_score_attention_grad_workspace_bytes(const SM120ScoreAttentionDesc* desc) {
    ScoreParams p{};
    bool empty = false;
    int device = 0, sms = 0;
    if (resolve(desc, Form::GRADIENT, &p, &empty) != cudaSuccess || empty || current_device(&device, &sms) != cudaSuccess) return 0;
    return grad_workspace(p, sms);
}

cudaError_t sm120_launch_score_attention_grad(const SM120ScoreAttentionDesc* desc) {
    ScoreParams p{};
    bool empty = false;
    cudaError_t e = resolve(desc, Form::GRADIENT, &p, &empty);
    if (e != cudaSuccess || empty) return e;
    // what no device is needed for first: the per-row arrays are the least a workspace holds
    if (!workspace_ok(desc, row_bytes(p))) return cudaErrorInvalidValue;
    int device = 0, sms = 0;
    e = current_device(&device, &sms);
    if (e != cudaSuccess) return e;
    if (!workspace_ok(desc, grad_workspace(p, sms))) return cudaErrorInvalidValue;
    p.neg_lse = static_cast<float*>(desc->workspace);
    p.neg_delta = p.neg_lse + stats_bytes(p) / sizeof(float);
    p.ranges = reinterpret_cast<int2*>(p.neg_delta + stats_bytes(p) / sizeof(float));
    if (!sa_tc_grad_supported(p)) {
        e = sa_simt_grad(p, desc->stream);
        if (e == cudaSuccess) note_launches("score_attention_grad_simt", 3);
        return e;
    }
    int launches = 0;
    e = sa_tc_grad(p, static_cast<char*>(desc->workspace) + row_bytes(p), device, sms, desc->stream, &launches);
    if (e == cudaSuccess) note_launches(p.head_dim > 64 ? "score_attention_grad_tcgen05_d128" : "score_attention_grad_tcgen05_d64", launches);
    return e;
}

size_t sm120_score_attention_decode_workspace_bytes(const SM120ScoreAttentionDesc* desc) {
    ScoreParams p{};
    bool empty = false;
    int device = 0, sms = 0;
    if (resolve(desc, Form::TOKEN, &p, &empty) != cudaSuccess || empty || current_device(&device, &sms) != cudaSuccess) return 0;
    return sa_tc_decode_supported(p) ? sa_tc_decode_workspace(p, sms) : 0;
}

cudaError_t sm120_launch_score_attention_decode(const SM120ScoreAttentionDesc* desc) {
    ScoreParams p{};
    bool empty = false;
    cudaError_t e = resolve(desc, Form::TOKEN, &p, &empty);
    if (e != cudaSuccess || empty) return e;
    int device = 0, sms = 0;
    e = current_device(&device, &sms);
    if (e != cudaSuccess) return e;
    if (!sa_tc_decode_supported(p)) {
        e = sa_simt_decode(p, desc->stream);
        if (e == cudaSuccess) note_launches("score_attention_decode_simt", 1);
        return e;
    }
    if (!workspace_ok(desc, sa_tc_decode_workspace(p, sms))) return cudaErrorInvalidValue;
    int launches = 0;
    e = sa_tc_decode(p, desc->workspace, device, sms, desc->stream, &launches);
    if (e == cudaSuccess) note_launches(p.head_dim > 64 ? "score_attention_decode_d128" : "score_attention_decode_d64", launches);
    return e;
}

}  // extern "C"
