#pragma once
// Score-modified attention forward for B200 (sm_100a), 16-bit types, head dimension up to 128:
//     O = softmax(modified(scale * Q K^T)) V    with the modifications and masks of SM120ScoreAttentionDesc.
//
// The structure is that of the plain fused kernel (attention_tcgen05.cu): one CTA owns 128 query rows and
// walks tiles of 128 keys; warp 0 feeds shared memory by TMA, warp 1 issues tcgen05.mma, two softmax groups of
// four warps take alternate tiles, P goes back to tensor memory as the A operand of P V, and O stays there
// under a reference maximum that moves only when a tile exceeds it by 2^8.  What differs:
//   * Keys.  A CTA's rows see one contiguous key range [kv_lo, kv_hi) (causal, prefix and document masks are all
//     per-row ranges whose ends never decrease), so its tiles start exactly at kv_lo and no tile outside is touched;
//     a tile tests single keys only when some row's range ends inside it (one vote per warp).
//   * Scores.  The cap and the distance bias are applied to the 128 scores in registers before the maximum:
//     tanh(u) as a polynomial on packed FMAs while a row's scores of the tile are within 0.8 caps, else 1 - 2 / (1 + e^2u), two more
//     MUFU operations a score (ex2, rcp) next to the softmax's one, which then bound the tile (16 heads x 8192 x 128: 974 instead
//     of 727 us; 495 without a cap); the bias
//     is one packed multiply-add, because on one side of the query it is linear in the key index (the tile across
//     the diagonal of a bidirectional mask takes the absolute value key by key).  Everything is in log2 units.
//   * Tensors.  4-D tensor maps take any strides; query head h reads key head h / group.  Columns behind head_dim
//     are the map's zero fill.
//   * Keys behind kv_hi in the last tile may hold anything, and P = 0 does not silence a NaN in V: the issuing warp zeroes those
//     rows of V in shared memory before it uses the tile.
//   * Output.  Rows go through shared memory (Q's, which is done with) and leave as TMA stores of 32 rows x 64 columns per warp: written by their
//     threads, 16 bytes a row at a time, they took 3000 to 4000 of a 16-tile block's 38000 cycles: 4 x 16 heads x 2048 x 128 158 -> 149 us.
// TOKEN: the rows are the batch's single-token queries against the prefix that they share, [entry x group head]
// of one key head as 128-row tiles, so the prefix is read once per 128 rows; the key tiles are cut into
// parts, and each part writes its normalised fp32 rows and their lse for the join (score_attention_decode.cu).

#include "attention_common.cuh"
#include "score_attention.h"

namespace sm120 {

struct SaFwdParams {
    ScoreParams s;
    float scale_log2;                // scale * log2(e)
    float cap_in;                    // 2 * log2(e) * scale / softcap: e^2u = 2^(dot * cap_in)
    float cap_log2;                  // softcap * log2(e)
    float cap_u;                     // scale / softcap: u = dot * cap_u
    int out_bf16;
    // TOKEN
    int batch_per_tile;              // entries per 128-row tile: 128 / group
    int tiles_per_part;              // key tiles per part
    float* part_out;                 // [part][batch][heads][head_dim]
    float* part_lse;                 // [part][batch][heads], log2 units
    unsigned long long wait_limit_ns;
    unsigned int* status;
};

template <int D>
struct SaCfg {
    static_assert(D == 64 || D == 128, "head dimension");
    static constexpr uint32_t Q_BYTES = ATT_BM * D * 2;
    static constexpr uint32_t K_BYTES = ATT_BN * D * 2;
    static constexpr uint32_t V_BYTES = ATT_BN * D * 2;
    static constexpr uint32_t TILE_BYTES = Q_BYTES + ATT_K_STAGES * K_BYTES + ATT_V_STAGES * V_BYTES;
    // barriers, the groups' row exchange: values [parity][group][row] and sequence words [group][row]
    static constexpr uint32_t BAR_BYTES = 256 + 2 * 2 * ATT_BM * 4 + 2 * ATT_BM * 4;
    static constexpr size_t SMEM_USED = TILE_BYTES + BAR_BYTES + 1024;
    // every CTA allocates all 512 TMEM columns, so two CTAs must never share an SM: request more than half of its shared memory
    static constexpr size_t SMEM = SMEM_USED > 118784 ? SMEM_USED : 118784;
    static constexpr uint32_t TMEM_COLS = 512;
    static constexpr uint32_t TMEM_O = 2 * ATT_BN;
    static_assert(SMEM <= 232448, "shared memory budget exceeded");
};

// The scores of one row against ATT_BN keys: raw products in, log2-unit modified scores out.  `rel` is the first key's
// position minus the query's.  With BIAS the tile's keys lie on one side of the query and `slope_log2` has that side's sign, or
// (MIXED) it is negative and the distance is taken key by key.
// The bias is scalar arithmetic: the key's index is then an immediate of the multiply-add, a packed one would first have to be moved to registers.
template <bool BIAS, bool MIXED>
__device__ __forceinline__ uint64_t sa_bias2(int i, float sl, float base, float rel) {
    if constexpr (!BIAS) return 0;
    else if constexpr (MIXED) return f32x2(sl * fabsf(rel + static_cast<float>(i)), sl * fabsf(rel + static_cast<float>(i + 1)));
    else return f32x2(fmaf(sl, static_cast<float>(i), base), fmaf(sl, static_cast<float>(i + 1), base));
}
template <bool CAP, bool BIAS, bool MIXED>
__device__ __forceinline__ void sa_modify(uint32_t (&s)[ATT_BN], float scale_log2, float cap_in, float cap_log2, float sl, float rel) {
    const uint64_t one2 = f32x2(1.0f, 1.0f), in2 = f32x2(cap_in, cap_in), cap2 = f32x2(cap_log2, cap_log2),
                   ncap2 = f32x2(-2.0f * cap_log2, -2.0f * cap_log2), scale2 = f32x2(scale_log2, scale_log2);
    const float base = sl * rel;
#pragma unroll
    for (int i = 0; i < ATT_BN; i += 2) {
        uint64_t x2 = f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        const uint64_t b2 = sa_bias2<BIAS, MIXED>(i, sl, base, rel);
        float a, b;
        if constexpr (CAP) {
            f32x2_split(mul2(x2, in2), a, b);
            f32x2_split(add2(f32x2(att_exp2(a), att_exp2(b)), one2), a, b);
            x2 = fma2(f32x2(att_rcp(a), att_rcp(b)), ncap2, cap2);
            if constexpr (BIAS) x2 = add2(x2, b2);
        } else {
            x2 = fma2(x2, scale2, b2);
        }
        f32x2_split(x2, a, b);
        s[i] = __float_as_uint(a);
        s[i + 1] = __float_as_uint(b);
    }
}

// The capped form for scores within the range of the tanh polynomial.  Returns the largest u^2: above SA_TANH_RANGE^2 the result is not used.
template <bool BIAS, bool MIXED>
__device__ __forceinline__ float sa_modify_small(uint32_t (&s)[ATT_BN], float cap_u, float cap_log2, float sl, float rel) {
    const uint64_t in2 = f32x2(cap_u, cap_u), cap2 = f32x2(cap_log2, cap_log2);
    const float base = sl * rel;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < ATT_BN; i += 2) {
        const uint64_t u2 = mul2(f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), in2), v2 = mul2(u2, u2);
        float a, b;
        f32x2_split(v2, a, b);
        top = att_max3(top, a, b);
        f32x2_split(fma2(mul2(u2, cap2), sa_tanh_ratio2(v2), sa_bias2<BIAS, MIXED>(i, sl, base, rel)), a, b);
        s[i] = __float_as_uint(a);
        s[i + 1] = __float_as_uint(b);
    }
    return top;
}

// Keys outside [start, limit) of the tile become -inf in log2 units, whatever they were.  FACTOR multiplies the others into log2 units (raw
// products: the caller then goes on with factor 1).  The lower bound is looked at only where a document begins inside the tile.
template <bool FACTOR>
__device__ __forceinline__ void sa_mask(uint32_t (&s)[ATT_BN], float factor, int start, int limit) {
#pragma unroll
    for (int i = 0; i < ATT_BN; ++i) {
        const float x = FACTOR ? __uint_as_float(s[i]) * factor : __uint_as_float(s[i]);
        s[i] = __float_as_uint(i < limit ? x : -CUDART_INF_F);
    }
    if (__any_sync(0xFFFFFFFFu, start > 0)) {
#pragma unroll
        for (int i = 0; i < ATT_BN; ++i)
            if (i < start) s[i] = __float_as_uint(-CUDART_INF_F);
    }
}

// p = exp2(s * scale2 + neg_m2) (MODIFIED scores already carry the scale) for KEYS keys, packed as 16-bit pairs, added to the
// partial row sums.  The sum adds the unrounded exponentials: rounding each first changes it by a relative 2^-9 / sqrt(keys), far
// inside the output's rounding.
template <int KEYS, bool MODIFIED>
__device__ __forceinline__ void sa_exp_pack(const uint32_t (&s)[KEYS], uint32_t (&packed)[KEYS / 2], uint64_t scale2, uint64_t neg_m2, uint64_t& l2, bool bf16) {
#pragma unroll
    for (int i = 0; i < KEYS; i += 2) {
        const uint64_t x = f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        float x0, x1;
        f32x2_split(MODIFIED ? add2(x, neg_m2) : fma2(x, scale2, neg_m2), x0, x1);
        const float p0 = att_exp2(x0), p1 = att_exp2(x1);
        l2 = add2(l2, f32x2(p0, p1));
        packed[i >> 1] = pack16(p0, p1, bf16);
    }
}

// Largest of a row's ATT_BN values (smallest with MIN): four chains of three-input maxima
template <bool MIN>
__device__ __forceinline__ float sa_extreme(const uint32_t (&s)[ATT_BN]) {
    float e[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) e[c] = __uint_as_float(s[c]);
#pragma unroll
    for (int i = 4; i + 8 <= ATT_BN; i += 8)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float a = __uint_as_float(s[i + 2 * c]), b = __uint_as_float(s[i + 2 * c + 1]);
            e[c] = MIN ? att_min3(e[c], a, b) : att_max3(e[c], a, b);
        }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const float a = __uint_as_float(s[ATT_BN - 4 + 2 * c]), b = __uint_as_float(s[ATT_BN - 3 + 2 * c]);
        e[c] = MIN ? att_min3(e[c], a, b) : att_max3(e[c], a, b);
    }
    return MIN ? fminf(fminf(e[0], e[1]), fminf(e[2], e[3])) : fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3]));
}

// Zeroes rows [first, 128) of a V tile in shared memory ([2 key blocks][D / 64 boxes][64 keys x 128 bytes]; the swizzle stays
// inside a row) and hands the writes to the async proxy.  One warp; it issues the products that read the tile.
template <int D>
__device__ __forceinline__ void sa_zero_rows(uint8_t* tile, int first, int lane) {
    constexpr int CHUNKS = D / 64 * 8;                       // 16-byte pieces of one row
    for (int c = lane; c < (ATT_BN - first) * CHUNKS; c += 32) {
        const int row = first + c / CHUNKS, piece = c % CHUNKS;
        *reinterpret_cast<uint4*>(tile + ((row >> 6) * (D / 64) + (piece >> 3)) * 8192 + (row & 63) * 128 + (piece & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    __syncwarp();
}

template <int D, bool CAP, bool BIAS, bool TOKEN>
__global__ void __launch_bounds__(ATT_THREADS, 1)
sm120_score_attention_kernel(const __grid_constant__ CUtensorMap tmap_q,
                             const __grid_constant__ CUtensorMap tmap_k,
                             const __grid_constant__ CUtensorMap tmap_v,
                             const __grid_constant__ CUtensorMap tmap_o,
                             const __grid_constant__ SaFwdParams p) {
    using Cfg = SaCfg<D>;
    constexpr bool MODIFIED = CAP || BIAS;
    constexpr int DB = D / 64;                       // 64-element (128-byte) blocks along the head dimension
    constexpr int KB = ATT_BN / 64;                  // 64-key blocks per key tile
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    const uint32_t q_smem = smem_u32(smem);
    const uint32_t k_smem = q_smem + Cfg::Q_BYTES;
    const uint32_t v_smem = k_smem + ATT_K_STAGES * Cfg::K_BYTES;
    uint8_t* v_tiles = smem + Cfg::Q_BYTES + ATT_K_STAGES * Cfg::K_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::TILE_BYTES);
    const uint32_t q_full = smem_u32(bars + 0);
    const uint32_t k_full = smem_u32(bars + 1);      // [3]
    const uint32_t k_empty = smem_u32(bars + 4);     // [3]
    const uint32_t v_full = smem_u32(bars + 7);      // [2]
    const uint32_t v_empty = smem_u32(bars + 9);     // [2]
    const uint32_t s_full = smem_u32(bars + 11);     // [2]  S_j is complete in TMEM (and with it every product issued before)
    const uint32_t p_lo = smem_u32(bars + 13);       // [2]  S_j has been read, keys 0-63 of P_j (and a rescaled O_g) are in TMEM
    const uint32_t o_done = smem_u32(bars + 15);     // [2]  the group's last product is complete
    const uint32_t drain_bar = smem_u32(bars + 17);
    const uint32_t p_hi = smem_u32(bars + 19);       // [2]  keys 64-127 of P_j are in TMEM
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 22);
    volatile uint32_t* abort_flag = tmem_holder + 1;
    volatile int* key_range = reinterpret_cast<volatile int*>(tmem_holder + 2);         // kv_lo, kv_hi
    volatile float* xchg = reinterpret_cast<volatile float*>(reinterpret_cast<uint8_t*>(bars) + 256);      // [2][2][ATT_BM]
    volatile int* xseq = reinterpret_cast<volatile int*>(reinterpret_cast<uint8_t*>(bars) + 256 + 2 * 2 * ATT_BM * 4);   // [2][ATT_BM]
    if (threadIdx.x < 2 * ATT_BM) xseq[threadIdx.x] = 0;

    // the caches' launch behind this one reads nothing that this one writes: it may begin as soon as all blocks here have
    if (TOKEN) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const ScoreParams& sp = p.s;
    // Grid.  Sequences: (batch x heads, query tiles): the heads that share keys run side by side, and a causal launch walks
    // the query tiles from the last one down, long tiles first.  TOKEN: (kv_heads, row tiles, key parts).
    const int tile_q = TOKEN ? static_cast<int>(blockIdx.y) : static_cast<int>(sp.causal ? gridDim.y - 1 - blockIdx.y : blockIdx.y);
    const int b = TOKEN ? 0 : static_cast<int>(blockIdx.x) / sp.heads;
    const int h = TOKEN ? 0 : static_cast<int>(blockIdx.x) % sp.heads;
    const int kvh = TOKEN ? static_cast<int>(blockIdx.x) : h / sp.group;
    const int q0 = tile_q * ATT_BM;                          // sequences: first row
    const int b0 = tile_q * p.batch_per_tile;                // TOKEN: first entry
    const int first_pos = sp.seq_k - sp.seq_q;               // sequences: position of row 0
    WaitCtx wctx{p.status, abort_flag, 0u, p.wait_limit_ns};

    auto load_q = [&]() {
        mbar_expect_tx(q_full, TOKEN ? static_cast<uint32_t>(p.batch_per_tile * sp.group) * (D * 2) : Cfg::Q_BYTES);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            // TOKEN rows fill batch_per_tile * group of the block's 128 (rows are independent: the rest is never stored)
            if (TOKEN) tma_load_4d(q_smem + d * (ATT_BM * 128), &tmap_q, q_full, d * 64, 0, b0, kvh);
            else tma_load_4d(q_smem + d * (ATT_BM * 128), &tmap_q, q_full, d * 64, q0, h, b);
        }
    };
    auto load_keys = [&](int j, int key) {
        const uint32_t st = j % ATT_K_STAGES;
        mbar_expect_tx(k_full + 8 * st, Cfg::K_BYTES);
#pragma unroll
        for (int d = 0; d < DB; ++d)
            tma_load_4d(k_smem + st * Cfg::K_BYTES + d * (ATT_BN * 128), &tmap_k, k_full + 8 * st, d * 64, key, kvh, b);
    };

    // the keys this CTA visits: one thread finds the range, requests Q and the first two K tiles (their trip from HBM is the
    // longest part of a block's start) and tells the others behind the barrier
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int st = 0; st < ATT_K_STAGES; ++st) {
            mbar_init(k_full + 8 * st, 1);
            mbar_init(k_empty + 8 * st, 1);
        }
        for (int st = 0; st < ATT_V_STAGES; ++st) {
            mbar_init(v_full + 8 * st, 1);
            mbar_init(v_empty + 8 * st, 1);
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(s_full + 8 * g, 1);
            mbar_init(p_lo + 8 * g, 4);              // one arrival per warp of the group
            mbar_init(p_hi + 8 * g, 4);
            mbar_init(o_done + 8 * g, 1);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0u;
        fence_barrier_init();
        fence_proxy_async_smem();
        prefetch_tmap(&tmap_q);
        prefetch_tmap(&tmap_k);
        prefetch_tmap(&tmap_v);
        if (!TOKEN) prefetch_tmap(&tmap_o);
        int lo, hi, other;
        if (TOKEN) {
            lo = static_cast<int>(blockIdx.z) * p.tiles_per_part * ATT_BN;
            hi = min(sp.prefix_len, lo + p.tiles_per_part * ATT_BN);
        } else {
            sa_row_range(sp, b, q0, lo, other);
            sa_row_range(sp, b, min(q0 + ATT_BM, sp.seq_q) - 1, other, hi);
        }
        key_range[0] = lo;
        key_range[1] = hi;
        if (lo < hi) {
            load_q();
            load_keys(0, lo);
            if (lo + ATT_BN < hi) load_keys(1, lo + ATT_BN);
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
    const int kv_lo = key_range[0], kv_hi = key_range[1];
    const int n_kv = kv_hi > kv_lo ? (kv_hi - kv_lo + ATT_BN - 1) / ATT_BN : 0;

    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(ATT_REGS_LOW));

    if (warp == 0) {
        // ------------------------------ TMA producer ------------------------------
        bool ok = n_kv > 0;
        int issued_k = min(n_kv, 2), issued_v = 0;             // Q, K_0 and K_1 were requested during set-up
        // the scores run two tiles ahead of the P V products: V_j, then K_{j+2}
        for (int j = 0; ok && j < n_kv; ++j) {
            const uint32_t st = j % ATT_V_STAGES, ph = (j / ATT_V_STAGES) & 1;
            bool w = att_wait(v_empty + 8 * st, ph ^ 1u, wctx, 0x42000000u);
            w = __all_sync(0xFFFFFFFFu, w);
            if (!w) { ok = false; break; }
            if (elect_one_sync()) {
                mbar_expect_tx(v_full + 8 * st, Cfg::V_BYTES);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int d = 0; d < DB; ++d)
                        tma_load_4d(v_smem + st * Cfg::V_BYTES + (kb * DB + d) * 8192, &tmap_v, v_full + 8 * st, d * 64,
                                    kv_lo + j * ATT_BN + kb * 64, kvh, b);
            }
            __syncwarp();
            ++issued_v;
            if (j + 2 < n_kv) {
                const uint32_t kst = (j + 2) % ATT_K_STAGES, kph = ((j + 2) / ATT_K_STAGES) & 1;
                w = att_wait(k_empty + 8 * kst, kph ^ 1u, wctx, 0x41000000u);
                ok = __all_sync(0xFFFFFFFFu, w);
                if (!ok) break;
                if (elect_one_sync()) load_keys(j + 2, kv_lo + (j + 2) * ATT_BN);
                __syncwarp();
                ++issued_k;
            }
        }
        // before leaving: every copy issued must have landed (immediate unless the CTA is aborting)
        if (n_kv > 0) att_wait(q_full, 0u, wctx, 0x43000000u, false);
        for (int i = max(0, issued_k - ATT_K_STAGES); i < issued_k; ++i)
            att_wait(k_full + 8 * (i % ATT_K_STAGES), (i / ATT_K_STAGES) & 1, wctx, 0x43000000u, false);
        for (int i = max(0, issued_v - ATT_V_STAGES); i < issued_v; ++i)
            att_wait(v_full + 8 * (i % ATT_V_STAGES), (i / ATT_V_STAGES) & 1, wctx, 0x43000000u, false);
    } else if (warp == 1) {
        // ------------------------------ MMA issuer ------------------------------
        const uint32_t fmt = p.out_bf16 ? 1u : 0u;
        // M = 128; S: N = ATT_BN, both operands K-major; P V: N = D, A from TMEM, B (= V as stored) is N-major (bit 16)
        const uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(ATT_BN >> 3) << 17) | (static_cast<uint32_t>(ATT_BM >> 4) << 24);
        const uint32_t idesc_pv = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(ATT_BM >> 4) << 24);
        const uint64_t desc_hi = (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
        const uint32_t lbo_k = (16u >> 4) << 16;                   // K-major operands
        const uint32_t lbo_v = (8192u >> 4) << 16;                 // N-major V: 8 KB between its 64-column boxes
        bool ok = n_kv > 0;
        bool issued_any = false;
        if (ok) {
            bool w = att_wait(q_full, 0u, wctx, 0x51000000u);
            ok = __all_sync(0xFFFFFFFFu, w);
        }
        // S_j = Q K_j^T into S buffer j % 2, whose last reader was P_{j-2} V_{j-2}, issued before by this thread
        auto qk_mmas = [&](int j) {
            const uint32_t st = j % ATT_K_STAGES, g = j & 1;
            const uint32_t s_tmem = tmem_base + g * ATT_BN;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
                const uint32_t off = (t >> 2) * (128 * 128) + (t & 3) * 32;       // 64-element block, then 32 bytes per K step
                const uint64_t a_desc = desc_hi | ((((q_smem + off) >> 4) & 0x3FFFu) | lbo_k);
                const uint64_t b_desc = desc_hi | ((((k_smem + st * Cfg::K_BYTES + off) >> 4) & 0x3FFFu) | lbo_k);
                umma_ss<KIND_F16, 1>(s_tmem, a_desc, b_desc, idesc_s, t != 0 ? 1u : 0u);
            }
            umma_commit<1>(s_full + 8 * g);
            umma_commit<1>(k_empty + 8 * st);
        };
        // O_g += P_j[:, 16 t0 .. 16 t1) V_j[16 t0 .. 16 t1, :]   (one elected thread)
        auto pv_mmas = [&](int j, int t0, int t1) {
            const uint32_t g = j & 1, st = j % ATT_V_STAGES;
            const uint32_t p_tmem = tmem_base + g * ATT_BN + ATT_BN / 2;      // P_j: the upper 64 cells of S buffer g
            const uint32_t o_tmem = tmem_base + Cfg::TMEM_O + g * D;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                if (t < t0 || t >= t1) continue;
                const uint32_t b_off = (t >> 2) * (DB * 8192) + (t & 3) * 2048;   // 16 key rows of 128 bytes per K step
                const uint64_t b_desc = desc_hi | ((((v_smem + st * Cfg::V_BYTES + b_off) >> 4) & 0x3FFFu) | lbo_v);
                umma_ts_f16(o_tmem, p_tmem + t * 8, b_desc, idesc_pv, (t != 0 || j >= 2) ? 1u : 0u);   // 16 keys = 8 cells of P
            }
            if (t1 == 8) {
                umma_commit<1>(v_empty + 8 * st);
                if (j + 2 >= n_kv) umma_commit<1>(o_done + 8 * g);
            }
        };
        auto k_bar = [&](int j) { return k_full + 8 * (j % ATT_K_STAGES); };
        auto k_par = [&](int j) { return static_cast<uint32_t>((j / ATT_K_STAGES) & 1); };
        // rows of the last V tile that lie behind the CTA's keys but inside the tensor (behind the tensor TMA has filled in zeros)
        const int last_rows = kv_hi - (kv_lo + (n_kv - 1) * ATT_BN);
        const bool clean_last = last_rows < ATT_BN && kv_hi < (TOKEN ? sp.prefix_len : sp.seq_k);
        // The waits of this warp are on every tile's path, and it shares its scheduler with two busy softmax warps: barriers that
        // are normally complete are tested in pairs, and products that follow each other are issued from one election.
        for (int j0 = 0; ok && j0 < 2 && j0 < n_kv; ++j0) {
            bool w = att_wait(k_bar(j0), k_par(j0), wctx, 0x52000000u);
            ok = __all_sync(0xFFFFFFFFu, w);
            if (!ok) break;
            tcgen05_fence_after();
            if (elect_one_sync()) qk_mmas(j0);
            __syncwarp();
            issued_any = true;
        }
        for (int j = 0; ok && j < n_kv; ++j) {
            const uint32_t g = j & 1, bph = (j >> 1) & 1;
            const uint32_t vst = j % ATT_V_STAGES, vph = (j / ATT_V_STAGES) & 1;
            const bool more = j + 2 < n_kv;
            bool w = att_wait2(v_full + 8 * vst, vph, p_lo + 8 * g, bph, wctx, 0x54000000u, 0x55000000u);   // keys 0-63 of P_j are in TMEM
            ok = __all_sync(0xFFFFFFFFu, w);
            if (!ok) break;
            if (clean_last && j == n_kv - 1) sa_zero_rows<D>(v_tiles + vst * Cfg::V_BYTES, last_rows, lane);
            tcgen05_fence_after();
            if (elect_one_sync()) pv_mmas(j, 0, 4);
            __syncwarp();
            if (more) w = att_wait2(p_hi + 8 * g, bph, k_bar(j + 2), k_par(j + 2), wctx, 0x55000000u, 0x52000000u);
            else w = att_wait(p_hi + 8 * g, bph, wctx, 0x55000000u);
            ok = __all_sync(0xFFFFFFFFu, w);
            if (!ok) break;
            tcgen05_fence_after();
            if (elect_one_sync()) {
                pv_mmas(j, 4, 8);
                if (more) qk_mmas(j + 2);
            }
            __syncwarp();
        }
        if (*abort_flag != 0u && issued_any) {
            if (elect_one_sync()) umma_commit<1>(drain_bar);
            __syncwarp();
            att_wait(drain_bar, 0u, wctx, 0x57000000u, false);
        }
    } else if (warp >= 4) {
        // ------------------------------ softmax and output ------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(ATT_REGS_HIGH));
        const int lane_group = warp & 3;                       // TMEM lanes [32 * lane_group, +32)
        const int g = (warp - 4) >> 2;                         // group: key tiles j % 2 == g, S buffer g, accumulator O_g
        const int row = lane_group * 32 + lane;                // this thread's query row inside the tile
        // this row: where its result goes, which keys it sees, where it stands, its bias
        int64_t out_row;                                       // element offset of the output row
        int64_t lse_row;
        bool live;
        int lo, hi, pos;
        float slope_log2 = 0.0f;
        int side_first, side_last;                             // positions of the CTA's first and last row, for the bias formula
        if (TOKEN) {
            const int e = b0 + row / sp.group, hq = kvh * sp.group + row % sp.group;
            live = row < p.batch_per_tile * sp.group && e < sp.batch;
            const int ec = min(e, sp.batch - 1);
            lse_row = static_cast<int64_t>(ec) * sp.heads + hq;
            out_row = (static_cast<int64_t>(blockIdx.z) * sp.batch * sp.heads + lse_row) * sp.head_dim;
            lo = kv_lo;
            hi = kv_hi;
            pos = sp.prefix_len - 1;
            if (BIAS) {
                slope_log2 = __ldg(sp.slopes + hq) * SA_LOG2E;
                pos += min(max(__ldg(sp.key_lengths + ec), 0), sp.seq_k);
            }
            side_first = side_last = 0x7FFFFFFF;               // no key lies behind any of the queries
        } else {
            const int q = q0 + row;
            live = q < sp.seq_q;
            out_row = 0;                                       // the tensor map knows
            lse_row = (static_cast<int64_t>(b) * sp.heads + h) * sp.seq_q + q;
            sa_row_range(sp, b, min(q, sp.seq_q - 1), lo, hi);
            pos = q + first_pos;
            if (BIAS) slope_log2 = __ldg(sp.slopes + h) * SA_LOG2E;
            side_first = q0 + first_pos;
            side_last = side_first + ATT_BM - 1;
            // behind a purely causal diagonal everything is masked, whatever its bias
            if (sp.causal && sp.prefix_lengths == nullptr) side_first = side_last = 0x7FFFFFFF;
        }
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(lane_group * 32) << 16);
        const uint32_t t_s = t_lane + g * ATT_BN;              // S_j, and P_j in its last 64 cells
        const uint32_t t_o = t_lane + Cfg::TMEM_O + g * D;
        const bool bf16 = p.out_bf16 != 0;
        const float scale_log2 = p.scale_log2;
        float m_ref = -CUDART_INF_F, l_run = 0.0f;             // reference maximum (log2 units) and row sum relative to it
        bool ok = true;
        for (int j = g; j < n_kv; j += 2) {
            const int key0 = kv_lo + j * ATT_BN;
            ok = att_wait(s_full + 8 * g, (j >> 1) & 1, wctx, 0x61000000u);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tcgen05_fence_after();
            // the row's 128 scores -> registers
            uint32_t s[ATT_BN];
            __syncwarp();
#pragma unroll
            for (int c = 0; c < ATT_BN / 32; ++c) tmem_ld_32x32(t_s + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
#pragma unroll
            for (int c = 0; c < ATT_BN / 32; ++c) tmem_ld_wait_regs(*reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
            // some of the tile's keys do not count for some row of this warp
            const bool edge = __any_sync(0xFFFFFFFFu, key0 < lo || key0 + ATT_BN > hi);
            if constexpr (MODIFIED) {
                const float rel = static_cast<float>(key0 - pos);
                const bool before = !BIAS || key0 + ATT_BN - 1 <= side_first, mixed = BIAS && !before && key0 < side_last;
                const float sl = before ? slope_log2 : -slope_log2;
                if constexpr (CAP) {
                    float top;
                    if (mixed) top = sa_modify_small<BIAS, true>(s, p.cap_u, p.cap_log2, sl, rel);
                    else top = sa_modify_small<BIAS, false>(s, p.cap_u, p.cap_log2, sl, rel);
                    if (!__all_sync(0xFFFFFFFFu, top <= SA_TANH_RANGE * SA_TANH_RANGE)) {
                        // a score of this warp's rows is too large: once more from the products, which still lie in TMEM
#pragma unroll
                        for (int c = 0; c < ATT_BN / 32; ++c) tmem_ld_32x32(t_s + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
#pragma unroll
                        for (int c = 0; c < ATT_BN / 32; ++c) tmem_ld_wait_regs(*reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
                        // key by key holds on every side
                        sa_modify<true, BIAS, true>(s, scale_log2, p.cap_in, p.cap_log2, -slope_log2, rel);
                    }
                } else {
                    if (mixed) sa_modify<false, BIAS, true>(s, scale_log2, p.cap_in, p.cap_log2, sl, rel);
                    else sa_modify<false, BIAS, false>(s, scale_log2, p.cap_in, p.cap_log2, sl, rel);
                }
            }
            // a tile at the border of some row's range is masked here once; what follows is the same for every tile
            float factor = MODIFIED ? 1.0f : scale_log2;
            if (edge) {
                sa_mask<!MODIFIED>(s, scale_log2, lo - key0, hi - key0);
                factor = 1.0f;
            }
            float m_tile;
            if constexpr (MODIFIED) m_tile = sa_extreme<false>(s);
            else m_tile = (factor >= 0.0f ? sa_extreme<false>(s) : sa_extreme<true>(s)) * factor;
            if (j < 2) {
                m_ref = m_tile;                                 // the group's first tile: O_g does not exist yet
            } else {
                // move the reference only when the tile exceeds it by more than ATT_RESCALE_STEP.  O_g may be rewritten
                // here: its last product (tile j - 2) was issued before S_j, which is complete.
                const bool moves = m_tile > m_ref + ATT_RESCALE_STEP;
                if (__any_sync(0xFFFFFFFFu, moves)) {
                    const float alpha = moves ? att_exp2(m_ref - m_tile) : 1.0f;     // 0 when the row had no key so far
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t oc[16];
                        tmem_ld_32x16_sync(t_o + c * 16, oc);
#pragma unroll
                        for (int i = 0; i < 16; ++i) oc[i] = __float_as_uint(__uint_as_float(oc[i]) * alpha);
                        tmem_st_32x32(t_o + c * 16, oc);
                    }
                    l_run *= alpha;
                    if (moves) m_ref = m_tile;
                }
            }
            const float m_use = m_ref == -CUDART_INF_F ? 0.0f : m_ref;      // a row without any key so far
            // p = exp2(z - m), row sum, P (16-bit pairs) -> cells [64, 128) of the S buffer, whose scores are in registers by now
            const uint64_t scale2 = f32x2(factor, factor), neg_m2 = f32x2(-m_use, -m_use);
            uint64_t l2 = f32x2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                // 64 keys at a time: one long run of independent exponentials, then one store; when half of P_j is
                // written its four MMAs may start
                uint32_t packed[32];
                const uint32_t(&sc)[64] = *reinterpret_cast<const uint32_t(*)[64]>(&s[c * 64]);
                sa_exp_pack<64, MODIFIED>(sc, packed, scale2, neg_m2, l2, bf16);
                tmem_st_32x32(t_s + ATT_BN / 2 + c * 32, packed);
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive((c == 0 ? p_lo : p_hi) + 8 * g);
            }
            float l_a, l_b;
            f32x2_split(l2, l_a, l_b);
            l_run += l_a + l_b;
        }
        // both accumulators complete (a group without tiles has none: its weight below is 0 and its O is not read)
        const bool has0 = n_kv > 0, has1 = n_kv > 1;
        if (ok && has0) {
            ok = att_wait(o_done, 0u, wctx, 0x64000000u);
            ok = __all_sync(0xFFFFFFFFu, ok);
        }
        if (ok && has1) {
            ok = att_wait(o_done + 8, 0u, wctx, 0x64000000u);
            ok = __all_sync(0xFFFFFFFFu, ok);
        }
        // the row's true reference is the larger of the groups'; weights w_g = 2^(m_g - m), sum = w_0 l_0 + w_1 l_1
        float m_other = -CUDART_INF_F, lw_other = 0.0f;
        if (ok) ok = pair_exchange(xchg, xseq, g, row, 1, m_ref, m_other, wctx);
        const float m_all = fmaxf(m_ref, m_other);
        const float m_fin = m_all == -CUDART_INF_F ? 0.0f : m_all;
        const float w_mine = att_exp2(m_ref - m_fin), w_other = att_exp2(m_other - m_fin);      // 0 for a group without keys
        const float lw_mine = l_run * w_mine;
        if (ok) ok = pair_exchange(xchg, xseq, g, row, 2, lw_mine, lw_other, wctx);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (ok) {
            constexpr int HD = D / 2;                           // this thread writes columns [g * HD, +HD) of its row
            const float l_row = g == 0 ? lw_mine + lw_other : lw_other + lw_mine;     // the same bits in both threads
            const bool none = n_kv == 0 || l_row == 0.0f;       // the row saw no key
            const float lse = none ? -CUDART_INF_F : m_fin + log2f(l_row);
            if (live && g == 0) {
                if (TOKEN) p.part_lse[static_cast<int64_t>(blockIdx.z) * sp.batch * sp.heads + lse_row] = lse;
                else if (sp.lse != nullptr) sp.lse[lse_row] = lse * SA_LN2;
            }
            const float inv = none ? 0.0f : 1.0f / l_row;
            const float w0 = (g == 0 ? w_mine : w_other) * inv, w1 = (g == 0 ? w_other : w_mine) * inv;
            tcgen05_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                float r[32];
                if (n_kv > 0) {
                    uint32_t o0[32], o1[32];
                    __syncwarp();
                    tmem_ld_32x32_sync(t_lane + Cfg::TMEM_O + g * HD + c * 32, o0);
                    if (has1) tmem_ld_32x32_sync(t_lane + Cfg::TMEM_O + D + g * HD + c * 32, o1);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        r[i] = __uint_as_float(o0[i]) * w0;
                        if (has1) r[i] = fmaf(__uint_as_float(o1[i]), w1, r[i]);
                        if (none) r[i] = 0.0f;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = 0.0f;
                }
                const int col = g * HD + c * 32;
                if (TOKEN) {
                    if (live) {
#pragma unroll
                        for (int v = 0; v < 8; ++v)
                            if (col + v * 4 < sp.head_dim)              // head_dim is a multiple of 8
                                *reinterpret_cast<float4*>(p.part_out + out_row + col + v * 4) = make_float4(r[v * 4], r[v * 4 + 1], r[v * 4 + 2], r[v * 4 + 3]);
                    }
                } else {
                    // every score product is complete (o_done): Q's place takes the block's rows, in the swizzle of a TMA box
                    const uint32_t dst = q_smem + (col >> 6) * (ATT_BM * 128) + row * 128;
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        st_shared_v4(dst + (((((col & 63) >> 3) + v) ^ (row & 7)) << 4), pack16(r[v * 8], r[v * 8 + 1], bf16),
                                     pack16(r[v * 8 + 2], r[v * 8 + 3], bf16), pack16(r[v * 8 + 4], r[v * 8 + 5], bf16), pack16(r[v * 8 + 6], r[v * 8 + 7], bf16));
                }
            }
            tcgen05_fence_before();
        }
        if (!TOKEN) {
            fence_proxy_async_smem();
            // at D = 64 the two warps of a lane group fill the two halves of the same 128-byte rows; every warp comes here, aborted or not
            if (D == 64) asm volatile("bar.sync %0, 64;" ::"r"(1 + lane_group) : "memory");
            else __syncwarp();
            const int first = q0 + lane_group * 32;
            if (ok && first < sp.seq_q && (D == 128 || g == 0) && elect_one_sync()) {
                const int block = D == 128 ? g : 0;             // this warp's 64 columns
                if (block * 64 < sp.head_dim) tma_store_4d(&tmap_o, q_smem + block * (ATT_BM * 128) + lane_group * (32 * 128), block * 64, first, h, b);
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

// One variant's launch.  The register hand-over inside the kernel balances only if the kernel starts with ATT_REGS_LAUNCH
// registers, so a build that compiled to another count is refused.
template <int D, bool CAP, bool BIAS, bool TOKEN>
cudaError_t sa_fwd_variant(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, const SaFwdParams& p, dim3 grid,
                           int device, cudaStream_t stream) {
    static std::atomic<uint64_t> attr_done{0};
    auto kern = sm120_score_attention_kernel<D, CAP, BIAS, TOKEN>;
    const uint64_t bit = 1ull << (device & 63);
    if ((attr_done.load(std::memory_order_acquire) & bit) == 0) {
        cudaFuncAttributes fa{};
        cudaError_t e = cudaFuncGetAttributes(&fa, kern);
        if (e != cudaSuccess) return e;
        if (fa.numRegs != ATT_REGS_LAUNCH) return cudaErrorLaunchOutOfResources;
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SaCfg<D>::SMEM));
        if (e != cudaSuccess) return e;
        attr_done.fetch_or(bit, std::memory_order_release);
    }
    kern<<<grid, ATT_THREADS, SaCfg<D>::SMEM, stream>>>(tq, tk, tv, to, p);
    return cudaGetLastError();
}

// the variants are compiled in score_attention_tcgen05_d64.cu and _d128.cu
template <int D>
cudaError_t sa_fwd_launch_d(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, const SaFwdParams& p, bool token,
                            dim3 grid, int device, cudaStream_t stream);

#define SA_FWD_INSTANTIATE(D)                                                                                                         \
    template <>                                                                                                                       \
    cudaError_t sa_fwd_launch_d<D>(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to,        \
                                   const SaFwdParams& p, bool token, dim3 grid, int device, cudaStream_t stream) {                    \
        const bool cap = p.s.softcap > 0.0f, bias = p.s.slopes != nullptr;                                                            \
        auto pick = [&](auto tok) {                                                                                                   \
            constexpr bool T = decltype(tok)::value;                                                                                  \
            if (cap) return bias ? sa_fwd_variant<D, true, true, T>(tq, tk, tv, to, p, grid, device, stream)                          \
                                 : sa_fwd_variant<D, true, false, T>(tq, tk, tv, to, p, grid, device, stream);                        \
            return bias ? sa_fwd_variant<D, false, true, T>(tq, tk, tv, to, p, grid, device, stream)                                  \
                        : sa_fwd_variant<D, false, false, T>(tq, tk, tv, to, p, grid, device, stream);                                \
        };                                                                                                                            \
        return token ? pick(std::true_type{}) : pick(std::false_type{});                                                              \
    }

}  // namespace sm120
