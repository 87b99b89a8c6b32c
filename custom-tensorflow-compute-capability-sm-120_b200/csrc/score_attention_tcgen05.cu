// Host side of the tensor-core kernels of the score-modified attention: what TMA can address, tensor maps, grids.
// The device code is in score_attention_tcgen05.cuh and score_attention_grad_tcgen05.cuh.

#include "score_attention_grad_tcgen05.cuh"
#include "score_attention_tcgen05.cuh"

namespace sm120 {

extern template cudaError_t sa_fwd_launch_d<64>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const SaFwdParams&, bool, dim3, int, cudaStream_t);
extern template cudaError_t sa_fwd_launch_d<128>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const SaFwdParams&, bool, dim3, int, cudaStream_t);

// 16-byte aligned base, and strides that are positive multiples of 16 bytes below TMA's 2^40 bytes wherever a second element exists
bool sa_tma_ok(const void* ptr, const int64_t* strides, const int64_t* extents, int count) {
    if ((reinterpret_cast<uintptr_t>(ptr) & 15u) != 0) return false;
    for (int a = 0; a < count; ++a)
        if (extents[a] > 1 && (strides[a] < 8 || (strides[a] & 7) != 0 || strides[a] >= (1ll << 39))) return false;
    return true;
}

bool sa_tc_types_ok(const ScoreParams& p) {
    return (p.dtype == SM120_DTYPE_FLOAT16 || p.dtype == SM120_DTYPE_BFLOAT16) && p.head_dim % 8 == 0 && p.head_dim <= 128;
}

static void sa_fwd_constants(SaFwdParams& fp, const ScoreParams& p, int device) {
    fp.s = p;
    fp.scale_log2 = p.scale * SA_LOG2E;
    fp.cap_in = p.softcap > 0.0f ? 2.0f * SA_LOG2E * p.scale / p.softcap : 0.0f;
    fp.cap_log2 = p.softcap * SA_LOG2E;
    fp.cap_u = p.softcap > 0.0f ? p.scale / p.softcap : 0.0f;
    fp.out_bf16 = p.dtype == SM120_DTYPE_BFLOAT16 ? 1 : 0;
    fp.wait_limit_ns = launch_wait_limit_ns();
    fp.status = tc_status_address(device);
}

bool sa_tc_forward_supported(const ScoreParams& p) {
    if (!sa_tc_types_ok(p) || p.seq_k < 1) return false;
    const int64_t qe[3] = {p.batch, p.heads, p.seq_q}, ke[3] = {p.batch, p.kv_heads, p.seq_k};
    if (!sa_tma_ok(p.q, p.q_st, qe, 3) || !sa_tma_ok(p.out, p.o_st, qe, 3) || !sa_tma_ok(p.k, p.k_st, ke, 3) || !sa_tma_ok(p.v, p.v_st, ke, 3)) return false;
    return p.seq_q <= 65535 * ATT_BM && static_cast<int64_t>(p.batch) * p.heads < (1ll << 31);      // grid limits
}

cudaError_t sa_tc_forward(const ScoreParams& p, int device, cudaStream_t stream) {
    SaFwdParams fp{};
    sa_fwd_constants(fp, p, device);
    if (fp.status == nullptr) return cudaErrorInvalidSymbol;
    CUtensorMap tq, tk, tv;
    const int64_t d = p.head_dim;
    if (!tc_encode_4d(&tq, p.q, p.dtype, {d, p.seq_q, p.heads, p.batch}, {p.q_st[2], p.q_st[1], p.q_st[0]}, {64, ATT_BM, 1, 1}) ||
        !tc_encode_4d(&tk, p.k, p.dtype, {d, p.seq_k, p.kv_heads, p.batch}, {p.k_st[2], p.k_st[1], p.k_st[0]}, {64, ATT_BN, 1, 1}) ||
        !tc_encode_4d(&tv, p.v, p.dtype, {d, p.seq_k, p.kv_heads, p.batch}, {p.v_st[2], p.v_st[1], p.v_st[0]}, {64, 64, 1, 1}))
        return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(p.batch) * p.heads, (p.seq_q + ATT_BM - 1) / ATT_BM, 1);
    return d > 64 ? sa_fwd_launch_d<128>(tq, tk, tv, fp, false, grid, device, stream) : sa_fwd_launch_d<64>(tq, tk, tv, fp, false, grid, device, stream);
}

cudaError_t sa_tc_prefix(const ScoreParams& p, int parts, int tiles_per_part, float* part_out, float* part_lse, int device, cudaStream_t stream) {
    SaFwdParams fp{};
    sa_fwd_constants(fp, p, device);
    if (fp.status == nullptr) return cudaErrorInvalidSymbol;
    fp.batch_per_tile = ATT_BM / p.group;
    fp.tiles_per_part = tiles_per_part;
    fp.part_out = part_out;
    fp.part_lse = part_lse;
    CUtensorMap tq, tk, tv;
    const int64_t d = p.head_dim;
    // queries as [key head][entry][head of the group]: a box of all the group's heads and batch_per_tile entries is a row tile
    if (!tc_encode_4d(&tq, p.q, p.dtype, {d, p.group, p.batch, p.kv_heads}, {p.q_st[1], p.q_st[0], p.q_st[1] * p.group}, {64, p.group, fp.batch_per_tile, 1}) ||
        !tc_encode_4d(&tk, p.prefix_k, p.dtype, {d, p.prefix_len, p.kv_heads, 1}, {p.pk_st[1], p.pk_st[0], 0}, {64, ATT_BN, 1, 1}) ||
        !tc_encode_4d(&tv, p.prefix_v, p.dtype, {d, p.prefix_len, p.kv_heads, 1}, {p.pv_st[1], p.pv_st[0], 0}, {64, 64, 1, 1}))
        return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(p.kv_heads), (p.batch + fp.batch_per_tile - 1) / fp.batch_per_tile, parts);
    return d > 64 ? sa_fwd_launch_d<128>(tq, tk, tv, fp, true, grid, device, stream) : sa_fwd_launch_d<64>(tq, tk, tv, fp, true, grid, device, stream);
}

extern template cudaError_t sa_grad_launch_d<64>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const SaGradParams&, bool, dim3, int, cudaStream_t);
extern template cudaError_t sa_grad_launch_d<128>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const SaGradParams&, bool, dim3, int, cudaStream_t);

bool sa_tc_grad_supported(const ScoreParams& p) {
    if (!sa_tc_types_ok(p) || p.seq_k < 1 || p.seq_q < 1) return false;
    const int64_t qe[3] = {p.batch, p.heads, p.seq_q}, ke[3] = {p.batch, p.kv_heads, p.seq_k};
    if (!sa_tma_ok(p.q, p.q_st, qe, 3) || !sa_tma_ok(p.grad_out, p.go_st, qe, 3) || !sa_tma_ok(p.grad_q, p.gq_st, qe, 3) ||
        !sa_tma_ok(p.k, p.k_st, ke, 3) || !sa_tma_ok(p.v, p.v_st, ke, 3) || !sa_tma_ok(p.grad_k, p.gk_st, ke, 3) || !sa_tma_ok(p.grad_v, p.gv_st, ke, 3))
        return false;
    return p.seq_q <= 65535 * ATT_BM && p.seq_k <= 65535 * ATT_BM;      // grid limits
}

cudaError_t sa_tc_grad(const ScoreParams& p, int device, cudaStream_t stream) {
    SaGradParams gp{};
    gp.s = p;
    gp.scale_log2 = p.scale * SA_LOG2E;
    gp.cap_in = p.softcap > 0.0f ? 2.0f * SA_LOG2E * p.scale / p.softcap : 0.0f;
    gp.cap_log2 = p.softcap * SA_LOG2E;
    gp.cap_u = p.softcap > 0.0f ? p.scale / p.softcap : 0.0f;
    gp.bf16 = p.dtype == SM120_DTYPE_BFLOAT16 ? 1 : 0;
    gp.wait_limit_ns = launch_wait_limit_ns();
    gp.status = tc_status_address(device);
    if (gp.status == nullptr) return cudaErrorInvalidSymbol;
    const int64_t d = p.head_dim;
    auto encode = [&](CUtensorMap* map, const void* ptr, const int64_t (&st)[3], int64_t seq, int64_t heads, int rows) {
        return tc_encode_4d(map, ptr, p.dtype, {d, seq, heads, p.batch}, {st[2], st[1], st[0]}, {64, rows, 1, 1});
    };
    CUtensorMap x, y, u, w;
    // queries as rows, then keys as rows
    if (!encode(&x, p.q, p.q_st, p.seq_q, p.heads, ATT_BM) || !encode(&y, p.grad_out, p.go_st, p.seq_q, p.heads, ATT_BM) ||
        !encode(&u, p.k, p.k_st, p.seq_k, p.kv_heads, SG_T) || !encode(&w, p.v, p.v_st, p.seq_k, p.kv_heads, SG_T))
        return cudaErrorInvalidValue;
    dim3 grid(static_cast<unsigned>(p.batch) * p.heads, (p.seq_q + ATT_BM - 1) / ATT_BM, 1);
    cudaError_t e = d > 64 ? sa_grad_launch_d<128>(x, y, u, w, gp, false, grid, device, stream) : sa_grad_launch_d<64>(x, y, u, w, gp, false, grid, device, stream);
    if (e != cudaSuccess) return e;
    if (!encode(&x, p.k, p.k_st, p.seq_k, p.kv_heads, ATT_BM) || !encode(&y, p.v, p.v_st, p.seq_k, p.kv_heads, ATT_BM) ||
        !encode(&u, p.q, p.q_st, p.seq_q, p.heads, SG_T) || !encode(&w, p.grad_out, p.go_st, p.seq_q, p.heads, SG_T))
        return cudaErrorInvalidValue;
    grid = dim3(static_cast<unsigned>(p.batch) * p.kv_heads, (p.seq_k + ATT_BM - 1) / ATT_BM, 1);
    return d > 64 ? sa_grad_launch_d<128>(x, y, u, w, gp, true, grid, device, stream) : sa_grad_launch_d<64>(x, y, u, w, gp, true, grid, device, stream);
}

}  // namespace sm120
