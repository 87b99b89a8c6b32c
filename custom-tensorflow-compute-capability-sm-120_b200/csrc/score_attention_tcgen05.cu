// Host side of the tensor-core kernels of the score-modified attention: what TMA can address, tensor maps, grids.
// The device code is in score_attention_tcgen05.cuh and score_attention_grad_tcgen05.cuh.

#include "score_attention_grad_tcgen05.cuh"
#include "score_attention_tcgen05.cuh"

namespace sm120 {

extern template cudaError_t sa_fwd_launch_d<64>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const SaFwdParams&, bool, dim3, int, cudaStream_t);
extern template cudaError_t sa_fwd_launch_d<128>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const SaFwdParams&, bool, dim3, int, cudaStream_t);

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
    CUtensorMap tq, tk, tv, to;
    const int64_t d = p.head_dim;
    if (!tc_encode_4d(&tq, p.q, p.dtype, {d, p.seq_q, p.heads, p.batch}, {p.q_st[2], p.q_st[1], p.q_st[0]}, {64, ATT_BM, 1, 1}) ||
        !tc_encode_4d(&tk, p.k, p.dtype, {d, p.seq_k, p.kv_heads, p.batch}, {p.k_st[2], p.k_st[1], p.k_st[0]}, {64, ATT_BN, 1, 1}) ||
        !tc_encode_4d(&tv, p.v, p.dtype, {d, p.seq_k, p.kv_heads, p.batch}, {p.v_st[2], p.v_st[1], p.v_st[0]}, {64, 64, 1, 1}) ||
        !tc_encode_4d(&to, p.out, p.dtype, {d, p.seq_q, p.heads, p.batch}, {p.o_st[2], p.o_st[1], p.o_st[0]}, {64, 32, 1, 1}))
        return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(p.batch) * p.heads, (p.seq_q + ATT_BM - 1) / ATT_BM, 1);
    return d > 64 ? sa_fwd_launch_d<128>(tq, tk, tv, to, fp, false, grid, device, stream) : sa_fwd_launch_d<64>(tq, tk, tv, to, fp, false, grid, device, stream);
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
    return d > 64 ? sa_fwd_launch_d<128>(tq, tk, tv, tq, fp, true, grid, device, stream) : sa_fwd_launch_d<64>(tq, tk, tv, tq, fp, true, grid, device, stream);
}

extern template cudaError_t sa_grad_launch_d<64>(const SaGradMaps&, const SaGradParams&, bool, dim3, int, cudaStream_t);
extern template cudaError_t sa_grad_launch_d<128>(const SaGradMaps&, const SaGradParams&, bool, dim3, int, cudaStream_t);

bool sa_tc_grad_supported(const ScoreParams& p) {
    if (!sa_tc_types_ok(p) || p.seq_k < 1 || p.seq_q < 1) return false;
    const int64_t qe[3] = {p.batch, p.heads, p.seq_q}, ke[3] = {p.batch, p.kv_heads, p.seq_k};
    if (!sa_tma_ok(p.q, p.q_st, qe, 3) || !sa_tma_ok(p.grad_out, p.go_st, qe, 3) || !sa_tma_ok(p.grad_q, p.gq_st, qe, 3) ||
        !sa_tma_ok(p.k, p.k_st, ke, 3) || !sa_tma_ok(p.v, p.v_st, ke, 3) || !sa_tma_ok(p.grad_k, p.gk_st, ke, 3) || !sa_tma_ok(p.grad_v, p.gv_st, ke, 3))
        return false;
    // D reads out and grad_out 16 bytes at a time
    if (!sa_tma_ok(p.out, p.o_st, qe, 3)) return false;
    return p.seq_q <= 65535 * ATT_BM && p.seq_k <= 65535 * ATT_BM;      // grid limits
}

// grad_K and grad_V from the parts, added in ascending order; four columns per thread
__global__ void __launch_bounds__(256)
sm120_score_attention_grad_join_kernel(const __grid_constant__ SaGradParams p) {
    const ScoreParams& sp = p.s;
    const int quads = sp.head_dim / 4;
    const int64_t rows = static_cast<int64_t>(sp.batch) * sp.kv_heads * sp.seq_k, all = rows * quads;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int which = blockIdx.y;                        // grad_K, grad_V
    if (idx >= all) return;
    const int64_t row = idx / quads;
    const int col = static_cast<int>(idx % quads) * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int part = 0; part < p.parts; ++part) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p.part_sums + ((static_cast<int64_t>(part) * 2 + which) * rows + row) * sp.head_dim + col));
        sum.x += x.x;
        sum.y += x.y;
        sum.z += x.z;
        sum.w += x.w;
    }
    const int key = static_cast<int>(row % sp.seq_k);
    const int64_t bh = row / sp.seq_k;
    const int h = static_cast<int>(bh % sp.kv_heads), b = static_cast<int>(bh / sp.kv_heads);
    const int64_t* st = which == 0 ? sp.gk_st : sp.gv_st;
    uint16_t* dst = static_cast<uint16_t*>(which == 0 ? sp.grad_k : sp.grad_v) + b * st[0] + h * st[1] + key * st[2] + col;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack16(sum.x, sum.y, p.bf16), pack16(sum.z, sum.w, p.bf16));
}

// Parts of the KEYS blocks' streams.  A block walks every query tile of every head that shares its key head; when the blocks are few, or a
// causal mask gives the first key tiles most of the work, one block's walk is longer than an even share of all of them.  In units of a tile
// (about 1 us): the longest walk or the even share, whichever is more, plus the join's launch and traffic.
static int grad_parts(const ScoreParams& p, int sms) {
    const double longest = static_cast<double>(p.group) * ((p.seq_q + SG_T - 1) / SG_T);
    const double blocks = static_cast<double>(p.batch) * p.kv_heads * ((p.seq_k + ATT_BM - 1) / ATT_BM);
    const double share = blocks * longest * (p.causal ? 0.5 : 1.0) / sms;
    const double part_us = static_cast<double>(p.batch) * p.kv_heads * p.seq_k * p.head_dim * 16.0 / 6.5e6;     // both sums, written and read
    int best = 1;
    double least = longest > share ? longest : share;
    for (int parts = 2; parts <= 8; ++parts) {
        const double walk = longest / parts;
        const double cost = (walk > share ? walk : share) + parts * part_us + 4.0;
        if (cost < 0.9 * least && walk >= 4.0) {
            best = parts;
            least = cost;
        }
    }
    return best;
}

size_t sa_tc_grad_workspace(const ScoreParams& p, int sms) {
    const int parts = grad_parts(p, sms);
    return parts == 1 ? 0 : static_cast<size_t>(parts) * 2 * p.batch * p.kv_heads * p.seq_k * p.head_dim * sizeof(float);
}

cudaError_t sa_tc_grad(const ScoreParams& p, void* workspace, int device, int sms, cudaStream_t stream, int* launches) {
    SaGradParams gp{};
    gp.parts = grad_parts(p, sms);
    gp.part_sums = static_cast<float*>(workspace);
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
    SaGradMaps m;
    // queries as rows, then keys as rows
    if (!encode(&m.x, p.q, p.q_st, p.seq_q, p.heads, ATT_BM) || !encode(&m.y, p.grad_out, p.go_st, p.seq_q, p.heads, ATT_BM) ||
        !encode(&m.u, p.k, p.k_st, p.seq_k, p.kv_heads, SG_T) || !encode(&m.w, p.v, p.v_st, p.seq_k, p.kv_heads, SG_T) ||
        !encode(&m.g1, p.grad_q, p.gq_st, p.seq_q, p.heads, 32))
        return cudaErrorInvalidValue;
    m.g2 = m.g1;
    dim3 grid(static_cast<unsigned>(p.batch) * p.heads, (p.seq_q + ATT_BM - 1) / ATT_BM, 1);
    cudaError_t e = d > 64 ? sa_grad_launch_d<128>(m, gp, false, grid, device, stream) : sa_grad_launch_d<64>(m, gp, false, grid, device, stream);
    if (e != cudaSuccess) return e;
    if (!encode(&m.x, p.k, p.k_st, p.seq_k, p.kv_heads, ATT_BM) || !encode(&m.y, p.v, p.v_st, p.seq_k, p.kv_heads, ATT_BM) ||
        !encode(&m.u, p.q, p.q_st, p.seq_q, p.heads, SG_T) || !encode(&m.w, p.grad_out, p.go_st, p.seq_q, p.heads, SG_T) ||
        !encode(&m.g1, p.grad_k, p.gk_st, p.seq_k, p.kv_heads, 32) || !encode(&m.g2, p.grad_v, p.gv_st, p.seq_k, p.kv_heads, 32))
        return cudaErrorInvalidValue;
    grid = dim3(static_cast<unsigned>(p.batch) * p.kv_heads, (p.seq_k + ATT_BM - 1) / ATT_BM, gp.parts);
    e = d > 64 ? sa_grad_launch_d<128>(m, gp, true, grid, device, stream) : sa_grad_launch_d<64>(m, gp, true, grid, device, stream);
    *launches = 2;
    if (e != cudaSuccess || gp.parts == 1) return e;
    const int64_t quads = static_cast<int64_t>(p.batch) * p.kv_heads * p.seq_k * (p.head_dim / 4);
    sm120_score_attention_grad_join_kernel<<<dim3(static_cast<unsigned>((quads + 255) / 256), 2, 1), 256, 0, stream>>>(gp);
    *launches = 3;
    return cudaGetLastError();
}

}  // namespace sm120
