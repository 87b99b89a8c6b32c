#pragma once
// Gradients of the score-modified attention for B200 (sm_100a), 16-bit types, head dimension up to 128.
// With P = exp2(z + neg_lse) and dx = P (dP + neg_delta) (1 - tanh^2):
//     KEYS kernel     grad_K = scale dx^T Q,  grad_V = P^T grad_O      one CTA per 128 keys of a key head
//     QUERIES kernel  grad_Q = scale dx K                              one CTA per 128 queries of a head
// Both form every score again from Q and K (seven products in all instead of five): each output row then has one owner that
// walks its partners in a fixed order, so nothing is added atomically, results are reproducible, the heads that share
// a key head are summed where they are used, and no fp32 copy of grad_Q goes through memory.
//
// The two are one kernel, because they are the same with the roles of queries and keys exchanged:
//                 rows (fixed, 128)      streamed (tiles of 64)     S = X U^T     dP = Y W^T     sums in TMEM
//     KEYS        X = K,  Y = V          U = Q, W = grad_O          S^T           dP^T           A1 += dx^T U,  A2 += P^T W
//     QUERIES     X = Q,  Y = grad_O     U = K, W = V               S             dP             A1 += dx U,  A2 += P (1 - tanh^2) U
// QUERIES runs first, and each of its blocks prepares its rows: neg_lse, D = <grad_O, O> and the key range, which it writes out for the
// KEYS launch.  (A pass of its own for them costs the same time on long rows, 18 us of 1420 at 16 heads x 8192 x 128, and one launch more on
// short ones: a step of 2 x 8 x 257 x 64 took 82 us by itself instead of 78.)
// It also makes D exact.  <grad_O, O> carries the rounding of O to 16 bits, which where few keys
// dominate a row is as large as the rest of the error together.  The row's sum of P (dP - D) is what D lacks; it corrects grad_Q through A2
// (grad_Q = scale (A1 - lack A2), one product more) and goes into neg_delta for the KEYS kernel.  Measured on peaked capped
// scores (relative error of grad_Q, bf16, against 64 bits, 2 x 16 heads x 2048 causal, cap 30): 2.9e-3 before, 2.4e-3 with it, for 4 % of a training step's time.
// Warp 0 feeds shared memory by TMA (X and Y once, U and W through a four-stage ring), warp 1 issues tcgen05.mma,
// and two groups of eight warps take alternate tiles: a thread owns half a row (TMEM lane, 32 of the 64 columns), reads its scores and dP,
// and writes P and dx as packed 16-bit pairs over the first half of the columns it has just read, where they
// are the A operands of the sums.  (Four warps per group, a whole row per thread: 2136 instead of 2094 us at 16 heads x 8192 x 128.)  U and W serve both products of their kernel from one copy: rows of 128 swizzled bytes are K-major
// for S and dP and N-major for the sums.  Issue order ... A_j, S_{j+2}, dP_{j+2}, A_{j+1} ...: one thread's MMAs run in order, so the
// buffers are free when the next scores overwrite them.  A tile's sums and the scores two tiles on are issued in one go: the
// issuing warp's wait and election cost 150 to 230 cycles of each tile's ~1800, so there is one of them (P and dx handed over in two halves, the
// first half's sums under the second's arithmetic: 1554 instead of 1402 us at 16 heads x 8192 x 64, the same at head size 128).
// What bounds it at D = 128 (cycle stamps): the tensor pipe.  A tile's sums take 8 x 64 cycles, its scores 16 x 80: an MMA whose A operand comes
// from shared memory pays 64 cycles for its 4 KB whatever N is, and TMEM has no room for X and Y beside double-buffered scores.  At D = 64 there is: the rows go
// there once and the scores read them as the sums read P (16 heads x 8192 x 64: 1390 to 1430 -> 1275 us).
// TMEM at D = 128: 2 x (64 + 64) scores and dP, 128 + 128 sums = 512 columns: no room for 128-row stream tiles.
// What a row of the stream needs (neg_lse, neg_delta, its key range) comes with the tile in the KEYS kernel and sits in
// registers in the other.

#include <type_traits>

#include "attention_common.cuh"
#include "score_attention.h"

namespace sm120 {

constexpr int SG_T = SA_GRAD_TILE;       // streamed rows per tile
constexpr int SG_STAGES = 4;
constexpr int SG_THREADS = 640;          // warp group 0: TMA, MMA and two idle warps; sixteen warps form P and dx
constexpr int SG_REGS_LOW = 40, SG_REGS_HIGH = 104, SG_REGS_LAUNCH = 96;
// as in attention_common.cuh: the sixteen warps may only ask for what warp group 0 gives back
static_assert(16 * (SG_REGS_HIGH - SG_REGS_LAUNCH) <= 4 * (SG_REGS_LAUNCH - SG_REGS_LOW), "register hand-over does not balance");
static_assert(SG_REGS_LAUNCH * SG_THREADS <= 65536, "register file");

struct SaGradParams {
    ScoreParams s;
    float scale_log2, cap_in, cap_log2, cap_u;           // as in SaFwdParams
    int bf16;
    int parts;                           // KEYS: the streamed tiles of a block are cut into this many parts, one block each
    float* part_sums;                    // [part][grad_K, grad_V][batch][kv_heads][seq_k][head_dim], read when parts > 1
    unsigned long long wait_limit_ns;
    unsigned int* status;
};

template <int D>
struct SgCfg {
    static_assert(D == 64 || D == 128, "head dimension");
    static constexpr uint32_t X_BYTES = ATT_BM * D * 2;              // [D / 64][128 rows x 128 bytes]
    static constexpr uint32_t U_BYTES = SG_T * D * 2;                // [D / 64][64 rows x 128 bytes]
    static constexpr uint32_t STAT_BYTES = SG_T * 16;                // neg_lse, neg_delta, ranges of a stream tile
    static constexpr uint32_t STAGE_BYTES = 2 * U_BYTES;
    static constexpr uint32_t STAT_OFF = 2 * X_BYTES + SG_STAGES * STAGE_BYTES;
    static constexpr uint32_t BAR_OFF = STAT_OFF + SG_STAGES * STAT_BYTES;
    // barriers, what the four threads of a row tell each other and the rows' <grad_O, O> (QUERIES)
    static constexpr size_t SMEM_USED = BAR_OFF + 256 + (4 + 1) * ATT_BM * 4 + 1024;
    // every CTA allocates all 512 TMEM columns, so two CTAs must never share an SM: request more than half of its shared memory
    static constexpr size_t SMEM = SMEM_USED > 118784 ? SMEM_USED : 118784;
    static constexpr uint32_t TMEM_COLS = 512;
    // S_0, dP_0, S_1, dP_1, each SG_T columns; A1; A2
    static constexpr uint32_t TMEM_A = 4 * SG_T;
    // at D = 64 there is room for X and Y behind the sums, two 16-bit elements per column
    static constexpr bool ROWS_IN_TMEM = D == 64;
    static constexpr uint32_t TMEM_X = TMEM_A + 2 * D, TMEM_Y = TMEM_X + D / 2;
    static_assert(SMEM <= 232448, "shared memory budget exceeded");
    static_assert(TMEM_A + 2 * D + (ROWS_IN_TMEM ? D : 0) <= TMEM_COLS, "TMEM budget exceeded");
};

// 16-byte aligned untiled copy global -> shared, counted on `bar`
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// The bias is linear in the column where all keys of a tile lie on one side of all its queries; tiles across the diagonal take the EDGE form,
// which forms the distance column by column.
// P and dx of 32 of a row's columns, packed.  Column c of the tile stands at distance rel + DIR * c (key position minus query
// position; DIR = -1 where the columns are queries).  EDGE: columns outside the range count as 0 whatever they hold.
// KEYS reads neg_lse, neg_delta and the ranges of the columns from shared memory; otherwise they belong to the row, P comes out times
// (1 - tanh^2), and the row's P (dP + neg_delta) is added to `lack`.
// SMALL: every |score| is inside the range of the tanh polynomial.
template <bool KEYS, bool CAP, bool BIAS, bool EDGE, bool SMALL>
__device__ __forceinline__ void sg_chunk(const uint32_t (&s)[32], const uint32_t (&dp)[32], uint32_t (&pp)[16], uint32_t (&pd)[16], int c0,
                                         const SaGradParams& p, float slope_log2, float rel, bool before, const float* col_lse, const float* col_delta,
                                         const int2* col_range, float row_lse, float row_delta, uint32_t off0, uint32_t width, float& lack) {
    const uint64_t scale2 = f32x2(p.scale_log2, p.scale_log2), in2 = f32x2(p.cap_in, p.cap_in), small2 = f32x2(p.cap_u, p.cap_u), one2 = f32x2(1.0f, 1.0f),
                   cap2 = f32x2(p.cap_log2, p.cap_log2), minus2 = f32x2(-1.0f, -1.0f);
    const float dir = KEYS ? -1.0f : 1.0f;
    const float sl = before ? slope_log2 : -slope_log2;
    const float step = sl * dir, base = sl * rel;
    uint64_t lack2 = f32x2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const int c = c0 + i;
        uint64_t add = KEYS ? *reinterpret_cast<const uint64_t*>(col_lse + c) : f32x2(row_lse, row_lse);
        if constexpr (BIAS) {
            // scalar: the column is an immediate of the multiply-add
            if constexpr (EDGE) add = add2(add, f32x2(-slope_log2 * fabsf(rel + dir * static_cast<float>(c)), -slope_log2 * fabsf(rel + dir * static_cast<float>(c + 1))));
            else add = add2(add, f32x2(fmaf(step, static_cast<float>(c), base), fmaf(step, static_cast<float>(c + 1), base)));
        }
        const uint64_t x2 = f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        uint64_t z2, curve2 = 0;
        if constexpr (CAP) {
            uint64_t tanh2;
            if constexpr (SMALL) {
                const uint64_t u2 = mul2(x2, small2);
                tanh2 = mul2(u2, sa_tanh_ratio2(mul2(u2, u2)));
            } else {
                float a, b;
                f32x2_split(mul2(x2, in2), a, b);
                f32x2_split(add2(f32x2(att_exp2(a), att_exp2(b)), one2), a, b);
                tanh2 = fma2(f32x2(att_rcp(a), att_rcp(b)), f32x2(-2.0f, -2.0f), one2);
            }
            z2 = fma2(tanh2, cap2, add);
            curve2 = fma2(mul2(tanh2, minus2), tanh2, one2);
        } else {
            z2 = fma2(x2, scale2, add);
        }
        float p0, p1, d0, d1;
        f32x2_split(z2, p0, p1);
        p0 = att_exp2(p0);
        p1 = att_exp2(p1);
        uint64_t d2 = add2(f32x2(__uint_as_float(dp[i]), __uint_as_float(dp[i + 1])),
                           KEYS ? *reinterpret_cast<const uint64_t*>(col_delta + c) : f32x2(row_delta, row_delta));
        if constexpr (KEYS) {
            if constexpr (CAP) d2 = mul2(d2, curve2);
            f32x2_split(mul2(d2, f32x2(p0, p1)), d0, d1);
        }
        if constexpr (EDGE) {
            bool in0, in1;
            if constexpr (KEYS) {
                // `off0` is the row's key position
                const int4 r = *reinterpret_cast<const int4*>(col_range + c);
                in0 = off0 - static_cast<uint32_t>(r.x) < static_cast<uint32_t>(r.y - r.x);
                in1 = off0 - static_cast<uint32_t>(r.z) < static_cast<uint32_t>(r.w - r.z);
            } else {
                in0 = off0 + c < width;
                in1 = off0 + c + 1 < width;
            }
            if constexpr (KEYS) {
                if (!in0) p0 = d0 = 0.0f;
                if (!in1) p1 = d1 = 0.0f;
            } else {
                // dP of a key outside the range may be anything as well
                float e0, e1;
                f32x2_split(d2, e0, e1);
                if (!in0) p0 = e0 = 0.0f;
                if (!in1) p1 = e1 = 0.0f;
                d2 = f32x2(e0, e1);
            }
        }
        if constexpr (!KEYS) {
            uint64_t p2 = f32x2(p0, p1);
            if constexpr (CAP) {
                lack2 = fma2(d2, p2, lack2);
                p2 = mul2(p2, curve2);
                d2 = mul2(d2, p2);
                f32x2_split(p2, p0, p1);
            } else {
                d2 = mul2(d2, p2);
                lack2 = add2(lack2, d2);
            }
            f32x2_split(d2, d0, d1);
        }
        pp[i >> 1] = pack16(p0, p1, p.bf16);
        pd[i >> 1] = pack16(d0, d1, p.bf16);
    }
    float la, lb;
    f32x2_split(lack2, la, lb);
    lack += la + lb;
}

// sum + the products of two rows' eight 16-bit elements
__device__ __forceinline__ float sg_dot8(const uint4& x, const uint4& y, bool bf16, float sum) {
    const uint32_t a[4] = {x.x, x.y, x.z, x.w}, c[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float2 u, v;
        if (bf16) {
            u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&a[k]));
            v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&c[k]));
        } else {
            u = __half22float2(*reinterpret_cast<const __half2*>(&a[k]));
            v = __half22float2(*reinterpret_cast<const __half2*>(&c[k]));
        }
        sum = fmaf(u.x, v.x, sum);
        sum = fmaf(u.y, v.y, sum);
    }
    return sum;
}

// Zeroes rows [r0, r1) of a stream tile's U and W and hands the writes to the async proxy.  One warp; it issues the products that read them.
template <int D>
__device__ __forceinline__ void sg_zero_rows(uint8_t* stage, int r0, int r1, int lane) {
    constexpr int CHUNKS = 2 * D / 64 * 8;                   // 16-byte pieces of a row of U and W
    for (int c = lane; c < (r1 - r0) * CHUNKS; c += 32) {
        const int row = r0 + c / CHUNKS, piece = c % CHUNKS;
        *reinterpret_cast<uint4*>(stage + (piece >> 3) * (SG_T * 128) + row * 128 + (piece & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    __syncwarp();
}

template <int D, bool KEYS, bool CAP, bool BIAS>
__global__ void __launch_bounds__(SG_THREADS, 1)
sm120_score_attention_grad_kernel(const __grid_constant__ CUtensorMap tmap_x,
                                  const __grid_constant__ CUtensorMap tmap_y,
                                  const __grid_constant__ CUtensorMap tmap_u,
                                  const __grid_constant__ CUtensorMap tmap_w,
                                  const __grid_constant__ CUtensorMap tmap_g1,
                                  const __grid_constant__ CUtensorMap tmap_g2,
                                  const __grid_constant__ SaGradParams p) {
    using Cfg = SgCfg<D>;
    constexpr int DB = D / 64;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    const uint32_t x_smem = smem_u32(smem), y_smem = x_smem + Cfg::X_BYTES, ring = x_smem + 2 * Cfg::X_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFF);
    const uint32_t xy_full = smem_u32(bars + 0);
    const uint32_t full = smem_u32(bars + 1);        // [4]
    const uint32_t empty = smem_u32(bars + 5);       // [4]
    const uint32_t s_full = smem_u32(bars + 9);      // [2]  S_j and dP_j are complete in TMEM (and with them every product issued before)
    const uint32_t a_ready = smem_u32(bars + 11);    // [2]  S_j and dP_j have been read, P_j and dx_j are in TMEM
    const uint32_t xy_tmem = smem_u32(bars + 13);    // X and Y are in TMEM (D = 64)
    const uint32_t sums_done = smem_u32(bars + 15);
    const uint32_t drain_bar = smem_u32(bars + 16);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 18);
    volatile uint32_t* abort_flag = tmem_holder + 1;
    volatile int* stream_range = reinterpret_cast<volatile int*>(tmem_holder + 2);      // first streamed row, end
    float* lacks = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 256);     // [group, half][ATT_BM]
    float* dots = lacks + 4 * ATT_BM;                                                    // [ATT_BM]

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const ScoreParams& sp = p.s;
    // Grid: (batch x row heads, row tiles, parts).  A causal launch starts the long tiles first: the first keys, the last queries.
    const int row_heads = KEYS ? sp.kv_heads : sp.heads;
    const int b = static_cast<int>(blockIdx.x) / row_heads, rh = static_cast<int>(blockIdx.x) % row_heads;
    const int r0 = static_cast<int>(!KEYS && sp.causal ? gridDim.y - 1 - blockIdx.y : blockIdx.y) * ATT_BM;
    const int rows = KEYS ? sp.seq_k : sp.seq_q, stream_rows = KEYS ? sp.seq_q : sp.seq_k;
    const int kvh = KEYS ? rh : rh / sp.group;
    const int first_pos = sp.seq_k - sp.seq_q;
    WaitCtx wctx{p.status, abort_flag, 0u, p.wait_limit_ns};

    // Streamed tiles: KEYS walks [u_lo, u_hi) of every head of the group; tiles start at a multiple of four rows (the alignment of their
    // statistics' copies).  Rows outside [u_lo, u_hi) may hold anything: the issuing warp zeroes them in shared memory.
    auto tile_start = [&](int u_lo, int t) { return (u_lo & ~3) + t * SG_T; };
    auto load_tile = [&](int j, int head, int u0) {
        const uint32_t st = j % SG_STAGES, bar = full + 8 * st, dst = ring + st * Cfg::STAGE_BYTES;
        mbar_expect_tx(bar, Cfg::STAGE_BYTES + (KEYS ? Cfg::STAT_BYTES : 0u));
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            tma_load_4d(dst + d * (SG_T * 128), &tmap_u, bar, d * 64, u0, head, b);
            tma_load_4d(dst + Cfg::U_BYTES + d * (SG_T * 128), &tmap_w, bar, d * 64, u0, head, b);
        }
        if (KEYS) {
            const uint32_t stat = x_smem + Cfg::STAT_OFF + st * Cfg::STAT_BYTES;
            const int64_t at = (static_cast<int64_t>(b) * sp.heads + head) * sp.seq_q_pad + u0;
            bulk_load(stat, sp.neg_lse + at, SG_T * 4, bar);
            bulk_load(stat + SG_T * 4, sp.neg_delta + at, SG_T * 4, bar);
            bulk_load(stat + SG_T * 8, sp.ranges + static_cast<int64_t>(b) * sp.seq_q_pad + u0, SG_T * 8, bar);
        }
    };

    if (threadIdx.x == 0) {
        mbar_init(xy_full, 1);
        for (int st = 0; st < SG_STAGES; ++st) {
            mbar_init(full + 8 * st, 1);
            mbar_init(empty + 8 * st, 1);
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(s_full + 8 * g, 1);
            mbar_init(a_ready + 8 * g, 8);           // one arrival per warp of the group
        }
        mbar_init(xy_tmem, 16);                      // one arrival per warp
        mbar_init(sums_done, 1);
        mbar_init(drain_bar, 1);
        *abort_flag = 0u;
        fence_barrier_init();
        fence_proxy_async_smem();
        prefetch_tmap(&tmap_x);
        prefetch_tmap(&tmap_y);
        prefetch_tmap(&tmap_u);
        prefetch_tmap(&tmap_w);
        int lo, hi, other;
        if (KEYS) {
            sa_query_range(sp, b, r0, min(r0 + ATT_BM, sp.seq_k), lo, hi);
        } else {
            sa_row_range(sp, b, r0, lo, other);
            sa_row_range(sp, b, min(r0 + ATT_BM, sp.seq_q) - 1, other, hi);
        }
        stream_range[0] = lo;
        stream_range[1] = hi;
        if (lo < hi) {
            mbar_expect_tx(xy_full, 2 * Cfg::X_BYTES);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                tma_load_4d(x_smem + d * (ATT_BM * 128), &tmap_x, xy_full, d * 64, r0, rh, b);
                tma_load_4d(y_smem + d * (ATT_BM * 128), &tmap_y, xy_full, d * 64, r0, rh, b);
            }
        }
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(tmem_holder), Cfg::TMEM_COLS);
        tmem_relinquish<1>();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    const int u_lo = stream_range[0], u_hi = stream_range[1];
    const int per_head = u_hi > u_lo ? (u_hi - (u_lo & ~3) + SG_T - 1) / SG_T : 0;       // tiles of one head
    // this block's tiles: all of them, or one of `parts` even shares (blockIdx.z) of the group's heads x tiles
    const int64_t all_tiles = KEYS ? static_cast<int64_t>(per_head) * sp.group : per_head;
    const int first_tile = KEYS ? static_cast<int>(all_tiles * blockIdx.z / p.parts) : 0;
    const int n_tiles = KEYS ? static_cast<int>(all_tiles * (blockIdx.z + 1) / p.parts) - first_tile : per_head;
    const int t_first = first_tile > 0 ? first_tile % per_head : 0;                      // tile index inside its head, and head, of the first one
    const int head0 = KEYS ? rh * sp.group + (first_tile > 0 ? first_tile / per_head : 0) : kvh;

    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SG_REGS_LOW));

    if (warp == 0) {
        // ------------------------------ TMA producer ------------------------------
        int issued = 0;
        int t = t_first, head = head0;
        for (int j = 0; j < n_tiles; ++j) {
            bool w = att_wait(empty + 8 * (j % SG_STAGES), ((j / SG_STAGES) & 1) ^ 1u, wctx, 0x42000000u);
            w = __all_sync(0xFFFFFFFFu, w);
            if (!w) break;
            if (elect_one_sync()) load_tile(j, head, tile_start(u_lo, t));
            __syncwarp();
            ++issued;
            if (++t == per_head) {
                t = 0;
                ++head;
            }
        }
        // before leaving: every copy issued must have landed (immediate unless the CTA is aborting)
        if (n_tiles > 0) att_wait(xy_full, 0u, wctx, 0x43000000u, false);
        for (int i = max(0, issued - SG_STAGES); i < issued; ++i)
            att_wait(full + 8 * (i % SG_STAGES), (i / SG_STAGES) & 1, wctx, 0x43000000u, false);
    } else if (warp == 1) {
        // ------------------------------ MMA issuer ------------------------------
        const uint32_t fmt = p.bf16 ? 1u : 0u;
        // M = 128.  Scores: N = 64, both operands K-major; sums: N = D, A from TMEM, B N-major (bit 16)
        const uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(SG_T >> 3) << 17) | (static_cast<uint32_t>(ATT_BM >> 4) << 24);
        const uint32_t idesc_a = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(ATT_BM >> 4) << 24);
        const uint64_t desc_hi = (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
        const uint32_t lbo_k = (16u >> 4) << 16;                       // K-major operands
        const uint32_t lbo_n = (static_cast<uint32_t>(SG_T * 128) >> 4) << 16;      // N-major: distance of the 64-column boxes
        bool ok = n_tiles > 0;
        bool issued_any = false;
        if (ok) {
            bool w = att_wait(xy_full, 0u, wctx, 0x51000000u);
            if (w && Cfg::ROWS_IN_TMEM) w = att_wait(xy_tmem, 0u, wctx, 0x53000000u);
            ok = __all_sync(0xFFFFFFFFu, w);
        }
        auto score_mmas = [&](int j) {
            const uint32_t st = j % SG_STAGES, g = j & 1;
            const uint32_t u_smem = ring + st * Cfg::STAGE_BYTES, w_smem = u_smem + Cfg::U_BYTES;
            const uint32_t s_tmem = tmem_base + g * (2 * SG_T);
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
                const uint32_t a_off = (t >> 2) * (ATT_BM * 128) + (t & 3) * 32, b_off = (t >> 2) * (SG_T * 128) + (t & 3) * 32;
                const uint64_t a_desc = desc_hi | ((((x_smem + a_off) >> 4) & 0x3FFFu) | lbo_k);
                const uint64_t b_desc = desc_hi | ((((u_smem + b_off) >> 4) & 0x3FFFu) | lbo_k);
                if constexpr (Cfg::ROWS_IN_TMEM) umma_ts_f16(s_tmem, tmem_base + Cfg::TMEM_X + t * 8, b_desc, idesc_s, t != 0 ? 1u : 0u);
                else umma_ss<KIND_F16, 1>(s_tmem, a_desc, b_desc, idesc_s, t != 0 ? 1u : 0u);
            }
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
                const uint32_t a_off = (t >> 2) * (ATT_BM * 128) + (t & 3) * 32, b_off = (t >> 2) * (SG_T * 128) + (t & 3) * 32;
                const uint64_t a_desc = desc_hi | ((((y_smem + a_off) >> 4) & 0x3FFFu) | lbo_k);
                const uint64_t b_desc = desc_hi | ((((w_smem + b_off) >> 4) & 0x3FFFu) | lbo_k);
                if constexpr (Cfg::ROWS_IN_TMEM) umma_ts_f16(s_tmem + SG_T, tmem_base + Cfg::TMEM_Y + t * 8, b_desc, idesc_s, t != 0 ? 1u : 0u);
                else umma_ss<KIND_F16, 1>(s_tmem + SG_T, a_desc, b_desc, idesc_s, t != 0 ? 1u : 0u);
            }
            umma_commit<1>(s_full + 8 * g);
        };
        // the tile's rows into the sums (one elected thread)
        auto sum_mmas = [&](int j) {
            const uint32_t st = j % SG_STAGES, g = j & 1;
            const uint32_t u_smem = ring + st * Cfg::STAGE_BYTES, w_smem = u_smem + Cfg::U_BYTES;
            const uint32_t p_tmem = tmem_base + g * (2 * SG_T), d_tmem = p_tmem + SG_T;
            const uint32_t a1 = tmem_base + Cfg::TMEM_A, a2 = a1 + D;
#pragma unroll
            for (int t = 0; t < SG_T / 16; ++t) {
                const uint32_t acc = (t != 0 || j != 0) ? 1u : 0u;
                const uint64_t u_desc = desc_hi | ((((u_smem + t * 2048) >> 4) & 0x3FFFu) | lbo_n);      // 16 rows of 128 bytes per K step
                const uint32_t cell = (t >> 1) * 32 + (t & 1) * 8;                                        // 16 rows = 8 cells of a half's 16
                umma_ts_f16(a1, d_tmem + cell, u_desc, idesc_a, acc);
                const uint64_t w_desc = desc_hi | ((((w_smem + t * 2048) >> 4) & 0x3FFFu) | lbo_n);
                umma_ts_f16(a2, p_tmem + cell, KEYS ? w_desc : u_desc, idesc_a, acc);
            }
            umma_commit<1>(empty + 8 * st);
            if (j == n_tiles - 1) umma_commit<1>(sums_done);
        };
        // rows of tile j that lie inside the tensor but outside [u_lo, u_hi) become zeros (behind the tensor TMA has filled in zeros)
        int clean_t = t_first;                                 // tile index inside its head
        auto clean = [&](int j) {
            const int u0 = tile_start(u_lo, clean_t);
            uint8_t* stage = smem + 2 * Cfg::X_BYTES + (j % SG_STAGES) * Cfg::STAGE_BYTES;
            if (u0 < u_lo) sg_zero_rows<D>(stage, 0, u_lo - u0, lane);
            if (u0 + SG_T > u_hi && u_hi < stream_rows) sg_zero_rows<D>(stage, u_hi - u0, SG_T, lane);
            if (++clean_t == per_head) clean_t = 0;
        };
        for (int j0 = 0; ok && j0 < 2 && j0 < n_tiles; ++j0) {
            bool w = att_wait(full + 8 * j0, 0u, wctx, 0x52000000u);
            ok = __all_sync(0xFFFFFFFFu, w);
            if (!ok) break;
            clean(j0);
            tcgen05_fence_after();
            if (elect_one_sync()) score_mmas(j0);
            __syncwarp();
            issued_any = true;
        }
        for (int j = 0; ok && j < n_tiles; ++j) {
            const uint32_t g = j & 1, ph = (j >> 1) & 1;
            const bool more = j + 2 < n_tiles;
            bool w;
            if (more) w = att_wait2(a_ready + 8 * g, ph, full + 8 * ((j + 2) % SG_STAGES), ((j + 2) / SG_STAGES) & 1, wctx, 0x54000000u, 0x52000000u);
            else w = att_wait(a_ready + 8 * g, ph, wctx, 0x54000000u);
            ok = __all_sync(0xFFFFFFFFu, w);
            if (!ok) break;
            if (more) clean(j + 2);
            tcgen05_fence_after();
            if (elect_one_sync()) {
                sum_mmas(j);
                if (more) score_mmas(j + 2);
            }
            __syncwarp();
        }
        if (*abort_flag != 0u && issued_any) {
            if (elect_one_sync()) umma_commit<1>(drain_bar);
            __syncwarp();
            att_wait(drain_bar, 0u, wctx, 0x57000000u, false);
        }
    } else if (warp >= 4) {
        // ------------------------------ P, dx and output ------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SG_REGS_HIGH));
        const int lane_group = warp & 3;
        const int g = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1;      // group (tiles j % 2 == g), columns [32 * half, +32)
        const int row = lane_group * 32 + lane;
        const int r = r0 + row;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(lane_group * 32) << 16);
        const uint32_t t_s = t_lane + g * (2 * SG_T) + half * 32, t_d = t_s + SG_T;
        // QUERIES: what belongs to the row
        int lo = 0, hi = 0;
        float row_lse = 0.0f, row_delta = 0.0f, slope_log2 = 0.0f, lack = 0.0f;
        if (!KEYS) {
            // D of the block's rows: eight rows per warp, sixteen lanes and 16-byte loads per row.  (Each row by the threads that own it: every load
            // then touches 32 rows, and the 4000 cycles that takes came before a block's first tile.)
            const uint16_t* o = static_cast<const uint16_t*>(sp.out) + b * sp.o_st[0] + rh * sp.o_st[1];
            const uint16_t* go = static_cast<const uint16_t*>(sp.grad_out) + b * sp.go_st[0] + rh * sp.go_st[1];
            const int col0 = (lane & 15) * 8, sub0 = (warp - 4) * 8 + (lane >> 4);
            uint4 x[4], y[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int i = r0 + sub0 + 2 * n;
                const bool there = i < sp.seq_q && col0 < sp.head_dim;
                x[n] = there ? __ldg(reinterpret_cast<const uint4*>(o + i * sp.o_st[2] + col0)) : make_uint4(0u, 0u, 0u, 0u);
                y[n] = there ? __ldg(reinterpret_cast<const uint4*>(go + i * sp.go_st[2] + col0)) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float d = sg_dot8(x[n], y[n], p.bf16, 0.0f);
#pragma unroll
                for (int sh = 8; sh > 0; sh >>= 1) d += __shfl_xor_sync(0xFFFFFFFFu, d, sh);
                if ((lane & 15) == 0) dots[sub0 + 2 * n] = d;
            }
            asm volatile("bar.sync 1, 512;" ::: "memory");
            const float dot = dots[row];
            const int rr = min(r, sp.seq_q - 1);
            const float lse = r < sp.seq_q ? __ldg(sp.lse + (static_cast<int64_t>(b) * sp.heads + rh) * sp.seq_q + r) : -CUDART_INF_F;
            const bool none = lse == -CUDART_INF_F;            // behind the last row, or a row that saw no key: P = 0
            row_lse = none ? -CUDART_INF_F : -lse * SA_LOG2E;
            row_delta = none ? 0.0f : -dot;
            sa_row_range(sp, b, rr, lo, hi);
            if (g == 0 && half == 0) {
                // rows up to the padded end: the last block writes those behind it as well
                for (int i = r; i < (r0 + ATT_BM >= sp.seq_q ? sp.seq_q_pad : r + 1); i += ATT_BM) {
                    const int64_t at = (static_cast<int64_t>(b) * sp.heads + rh) * sp.seq_q_pad + i;
                    sp.neg_lse[at] = i == r ? row_lse : -CUDART_INF_F;
                    if (i >= sp.seq_q) sp.neg_delta[at] = 0.0f;                  // the others once they are exact, below
                    if (rh == 0) sp.ranges[static_cast<int64_t>(b) * sp.seq_q_pad + i] = i < sp.seq_q ? make_int2(lo, hi) : make_int2(0, 0);
                }
            }
            if (BIAS) slope_log2 = __ldg(sp.slopes + rh) * SA_LOG2E;
        }
        int t = t_first, head = head0;
        bool ok = true;
        if constexpr (Cfg::ROWS_IN_TMEM) {
            // X (group 0) and Y (group 1) go from shared memory to TMEM, half a row per thread, and are the scores' A operands there
            if (n_tiles > 0) {
                ok = att_wait(xy_full, 0u, wctx, 0x63000000u);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (ok) {
                    uint32_t v[16];
                    const uint8_t* src = smem + g * Cfg::X_BYTES + row * 128;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint4 x = *reinterpret_cast<const uint4*>(src + (((half * 4 + c) ^ (row & 7)) << 4));
                        v[4 * c] = x.x;
                        v[4 * c + 1] = x.y;
                        v[4 * c + 2] = x.z;
                        v[4 * c + 3] = x.w;
                    }
                    tmem_st_32x32(t_lane + (g == 0 ? Cfg::TMEM_X : Cfg::TMEM_Y) + half * 16, v);
                    tmem_st_wait();
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(xy_tmem);
                }
            }
        }
        auto next_tile = [&]() {
            if (++t == per_head) {
                t = 0;
                ++head;
            }
        };
        if (g == 1 && n_tiles > 0) next_tile();
        for (int j = g; ok && j < n_tiles; j += 2) {
            const uint32_t st = j % SG_STAGES;
            const int u0 = tile_start(u_lo, t);
            const uint8_t* stat = smem + Cfg::STAT_OFF + st * Cfg::STAT_BYTES;
            const float* col_lse = reinterpret_cast<const float*>(stat);
            const float* col_delta = col_lse + SG_T;
            const int2* col_range = reinterpret_cast<const int2*>(col_delta + SG_T);
            if (KEYS && BIAS) slope_log2 = __ldg(sp.slopes + head) * SA_LOG2E;
            ok = att_wait(s_full + 8 * g, (j >> 1) & 1, wctx, 0x61000000u);
            // the statistics came with the tile: its barrier orders them (complete since the scores needed the tile)
            if (ok && KEYS) ok = att_wait(full + 8 * st, (j / SG_STAGES) & 1, wctx, 0x62000000u);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tcgen05_fence_after();
            uint32_t s[32], dp[32];
            __syncwarp();
            tmem_ld_32x32(t_s, s);
            tmem_ld_32x32(t_d, dp);
            tmem_ld_wait_regs(s);
            tmem_ld_wait_regs(dp);
            bool small = false;
            if constexpr (CAP) {
                float top = __uint_as_float(s[0]), low = top;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    top = att_max3(top, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                    low = att_min3(low, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                }
                small = __all_sync(0xFFFFFFFFu, fmaxf(top, -low) * fabsf(p.cap_u) <= SA_TANH_RANGE);
            }
            bool edge;
            uint32_t off0, width = 0;
            float rel;
            bool before = true;
            if (KEYS) {
                // the tile's first and last row bound every row's range
                const int2 first = col_range[0], last = col_range[min(SG_T, sp.seq_q - u0) - 1];
                const int w0 = r0 + lane_group * 32;
                edge = last.x > w0 || first.y < w0 + 32;
                off0 = static_cast<uint32_t>(r);
                rel = static_cast<float>(r - (u0 + first_pos));
                if (BIAS) {
                    before = r0 + ATT_BM - 1 <= u0 + first_pos;
                    edge = edge || (!before && r0 < u0 + first_pos + SG_T - 1);
                }
            } else {
                edge = __any_sync(0xFFFFFFFFu, u0 < lo || u0 + SG_T > hi);
                off0 = static_cast<uint32_t>(u0 - lo);
                width = static_cast<uint32_t>(hi - lo);
                rel = static_cast<float>(u0 - (r + first_pos));
                if (BIAS) {
                    before = u0 + SG_T - 1 <= r0 + first_pos;
                    edge = edge || (!before && u0 < r0 + first_pos + ATT_BM - 1);
                }
            }
            uint32_t pp[16], pd[16];
            auto chunk = [&](auto on_edge, auto in_range) {
                sg_chunk<KEYS, CAP, BIAS, decltype(on_edge)::value, decltype(in_range)::value>(s, dp, pp, pd, half * 32, p, slope_log2, rel, before, col_lse,
                                                                                              col_delta, col_range, row_lse, row_delta, off0, width, lack);
            };
            if (CAP && small) {
                if (edge) chunk(std::true_type{}, std::true_type{});
                else chunk(std::false_type{}, std::true_type{});
            } else {
                if (edge) chunk(std::true_type{}, std::false_type{});
                else chunk(std::false_type{}, std::false_type{});
            }
            tmem_st_32x32(t_s, pp);
            tmem_st_32x32(t_d, pd);
            tmem_st_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(a_ready + 8 * g);
            next_tile();
            if (j + 2 < n_tiles) next_tile();
        }
        if (ok && n_tiles > 0) {
            ok = att_wait(sums_done, 0u, wctx, 0x64000000u);
            ok = __all_sync(0xFFFFFFFFu, ok);
        }
        if (!KEYS) {
            // what D lacks, from the row's four threads in one order.  Every one of the sixteen warps comes here, aborted or not.
            lacks[(g * 2 + half) * ATT_BM + row] = lack;
            asm volatile("bar.sync 1, 512;" ::: "memory");
            lack = (lacks[row] + lacks[ATT_BM + row]) + (lacks[2 * ATT_BM + row] + lacks[3 * ATT_BM + row]);
            if (ok && g == 0 && half == 0 && r < rows)
                sp.neg_delta[(static_cast<int64_t>(b) * sp.heads + rh) * sp.seq_q_pad + r] = row_delta - lack;
        }
        if (ok) {
            constexpr int CW = D / 4;                           // this thread writes columns [col, +CW) of its row
            const int col = (g * 2 + half) * CW;
            tcgen05_fence_after();
#pragma unroll
            for (int which = 0; which < (KEYS ? 2 : 1); ++which) {
                const float factor = which == 0 ? sp.scale : 1.0f;
                uint32_t o[CW];
                auto load_sums = [&](uint32_t taddr, uint32_t (&v)[CW]) {
                    if constexpr (CW == 32) tmem_ld_32x32_sync(taddr, v);
                    else tmem_ld_32x16_sync(taddr, v);
                };
                if (n_tiles > 0) {
                    __syncwarp();
                    load_sums(t_lane + Cfg::TMEM_A + which * D + col, o);
                    if (!KEYS) {
                        uint32_t o2[CW];
                        load_sums(t_lane + Cfg::TMEM_A + D + col, o2);
#pragma unroll
                        for (int i = 0; i < CW; ++i) o[i] = __float_as_uint(fmaf(-lack, __uint_as_float(o2[i]), __uint_as_float(o[i])));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < CW; ++i) o[i] = 0u;
                }
                if (KEYS && p.parts > 1) {
                    if (r < rows) {
                        float* part = p.part_sums + (((static_cast<int64_t>(blockIdx.z) * 2 + which) * sp.batch + b) * sp.kv_heads + rh) * static_cast<int64_t>(sp.seq_k) * sp.head_dim +
                                      static_cast<int64_t>(r) * sp.head_dim;
#pragma unroll
                        for (int v = 0; v < CW / 4; ++v)
                            if (col + v * 4 < sp.head_dim)
                                *reinterpret_cast<float4*>(part + col + v * 4) =
                                    make_float4(__uint_as_float(o[v * 4]) * factor, __uint_as_float(o[v * 4 + 1]) * factor, __uint_as_float(o[v * 4 + 2]) * factor,
                                                __uint_as_float(o[v * 4 + 3]) * factor);
                    }
                } else {
                    // every product is complete: X's and Y's places take the block's rows, in the swizzle of a TMA box
                    const uint32_t dst = (which == 0 ? x_smem : y_smem) + (col >> 6) * (ATT_BM * 128) + row * 128;
#pragma unroll
                    for (int v = 0; v < CW / 8; ++v) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            w[k] = pack16(__uint_as_float(o[v * 8 + 2 * k]) * factor, __uint_as_float(o[v * 8 + 2 * k + 1]) * factor, p.bf16);
                        st_shared_v4(dst + (((((col & 63) >> 3) + v) ^ (row & 7)) << 4), w[0], w[1], w[2], w[3]);
                    }
                }
            }
            tcgen05_fence_before();
        }
        if (!KEYS || p.parts == 1) {
            // the four warps of a lane group hold the columns of the same 32 rows; every warp comes here, aborted or not
            fence_proxy_async_smem();
            asm volatile("bar.sync %0, 128;" ::"r"(2 + lane_group) : "memory");
            const int first = r0 + lane_group * 32;
            if (ok && first < rows && g == 0 && half == 0 && elect_one_sync()) {
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    if (d * 64 >= sp.head_dim) continue;
                    tma_store_4d(&tmap_g1, x_smem + d * (ATT_BM * 128) + lane_group * (32 * 128), d * 64, first, rh, b);
                    if (KEYS) tma_store_4d(&tmap_g2, y_smem + d * (ATT_BM * 128) + lane_group * (32 * 128), d * 64, first, rh, b);
                }
                bulk_commit_group();
                bulk_wait_group_read<0>();
            }
            __syncwarp();
        }
    }

    // ------------------------------ teardown ------------------------------
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tcgen05_fence_after();
        tmem_dealloc<1>(tmem_base, Cfg::TMEM_COLS);
    }
}

struct SaGradMaps {
    CUtensorMap x, y, u, w, g1, g2;      // rows, stream, and the outputs of A1 and (KEYS) A2
};

template <int D, bool KEYS, bool CAP, bool BIAS>
cudaError_t sa_grad_variant(const SaGradMaps& m, const SaGradParams& p, dim3 grid, int device, cudaStream_t stream) {
    static std::atomic<uint64_t> attr_done{0};
    auto kern = sm120_score_attention_grad_kernel<D, KEYS, CAP, BIAS>;
    const uint64_t bit = 1ull << (device & 63);
    if ((attr_done.load(std::memory_order_acquire) & bit) == 0) {
        // the register hand-over inside the kernel balances only if the kernel starts with SG_REGS_LAUNCH registers
        cudaFuncAttributes fa{};
        cudaError_t e = cudaFuncGetAttributes(&fa, kern);
        if (e != cudaSuccess) return e;
        if (fa.numRegs != SG_REGS_LAUNCH) return cudaErrorLaunchOutOfResources;
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SgCfg<D>::SMEM));
        if (e != cudaSuccess) return e;
        attr_done.fetch_or(bit, std::memory_order_release);
    }
    kern<<<grid, SG_THREADS, SgCfg<D>::SMEM, stream>>>(m.x, m.y, m.u, m.w, m.g1, m.g2, p);
    return cudaGetLastError();
}

// the variants are compiled in score_attention_grad_tcgen05_d64.cu and _d128.cu
template <int D>
cudaError_t sa_grad_launch_d(const SaGradMaps& m, const SaGradParams& p, bool keys, dim3 grid, int device, cudaStream_t stream);

#define SA_GRAD_INSTANTIATE(D)                                                                                                        \
    template <>                                                                                                                       \
    cudaError_t sa_grad_launch_d<D>(const SaGradMaps& m, const SaGradParams& p, bool keys, dim3 grid, int device, cudaStream_t stream) { \
        const bool cap = p.s.softcap > 0.0f, bias = p.s.slopes != nullptr;                                                            \
        auto pick = [&](auto k) {                                                                                                     \
            constexpr bool K = decltype(k)::value;                                                                                    \
            if (cap) return bias ? sa_grad_variant<D, K, true, true>(m, p, grid, device, stream)                                      \
                                 : sa_grad_variant<D, K, true, false>(m, p, grid, device, stream);                                    \
            return bias ? sa_grad_variant<D, K, false, true>(m, p, grid, device, stream)                                              \
                        : sa_grad_variant<D, K, false, false>(m, p, grid, device, stream);                                            \
        };                                                                                                                            \
        return keys ? pick(std::true_type{}) : pick(std::false_type{});                                                               \
    }

}  // namespace sm120
