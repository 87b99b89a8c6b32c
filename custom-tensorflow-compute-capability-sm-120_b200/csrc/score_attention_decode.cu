// Single-token attention over a cache, and over a prefix that the batch shares (16-bit types, head
// dimension up to 128).  Bound by HBM: every valid row of K and V is read once, 4 head_dim operations
// per query head and 4 head_dim bytes.
//
// Parts.  The keys of one (entry, key head) are cut into parts so that short batches fill the GPU and ragged ones
// balance; each part is one block.  Where two, four or eight parts of at most CLUSTER_KEYS keys do and all blocks run at once, the parts of a row are one
// cluster: the blocks leave their normalised rows and log2 denominators in shared memory and each joins a share of the columns from
// all of them, in ascending order, in the same launch (1 x 32/8 heads x 700 x 128: 5.9 us and no workspace instead of 5.8 + 5.3 us in two launches).
// Otherwise they go to the workspace and a second kernel joins them the same way.  A single part writes the result itself.
// Caches that offer more work than the GPU holds at once are STREAMED: the lengths live on the device, so the blocks (as many as run at
// once) count the 64-key units of all entries themselves and each takes an even, consecutive share of them, whatever the lengths
// are.  A share begins and ends inside some (entry, key head); those two pieces go to the block's two slots of the workspace, whole ones are
// written out at once, and the join finds the slots from the same arithmetic (what it brings: DIRECT_KEYS).
//
// Block.  Four warps, each with its own ring of 16-key tiles (K and V rows by 16-byte cp.async, rows behind the
// valid ones never touched: zero fill), so no barrier orders the loop: three tiles of 8 KB per warp and two blocks per SM keep
// ~190 KB of loads in flight per SM, four times what HBM latency asks for.  The query rows that share the keys (the heads of a
// group; for the prefix, all entries' heads) are the 16 rows of mma.sync.m16n8k16: the products need a tenth of the
// legacy tensor rate at full HBM speed, and 16 rows are what one token per request offers, so tcgen05's 128-row tiles would
// be 7/8 padding.  Both operands come from the swizzled tile by ldmatrix; P goes from the first product's accumulators
// straight into the second's operand.
//
// Rounding.  P is split into two 16-bit pieces (P = hi + lo to 2^-17 relative) that both multiply V: the second product is free
// under the memory time and the result then carries only its own final rounding.
//
// The shared prefix, when the batch has many rows, runs as 128-row tiles on the tcgen05 kernel instead (TOKEN variant of
// score_attention_tcgen05.cuh) and joins here in the same way.  The caches' launch needs nothing of it and begins while it runs, on the SMs
// that its last wave leaves idle (programmatic launch); only its first block waits for the prefix's grid before it ends, so
// that this grid's end, on which the join waits, is the end of both (128 x 32/8 heads, 16384 + up to 640 keys x 128: 96 -> 92 us).

#include <math_constants.h>

#include "attention_common.cuh"
#include "score_attention.h"

namespace sm120 {

constexpr int DEC_WARPS = 4;
constexpr int DEC_ROWS = 16;                  // query rows per block (M of the product)
constexpr int DEC_KEYS = 16;                  // keys per warp tile
constexpr int DEC_STAGES = 3;
// rows x keys x key heads of the prefix from which it runs on the tcgen05 kernel, whose 128-row tiles start slower but read the keys
// once per 128 rows instead of 16.  Measured, us (here / tcgen05): head size 128, 8 key heads, 4096 keys: 32 rows 14.2 / 16.4, 64 rows
// 19.4 / 17.2, 256 rows 50 / 27; 1 key head, 16384 keys: 64 rows 16.5 / 18.7, 256 rows 25 / 21; head size 64 crosses half as far again
// (8 key heads, 4096 keys: 64 rows 13.6 / 14.6, 128 rows 22.1 / 15.9)
constexpr int64_t PREFIX_TC_WORK_128 = 2ll << 20, PREFIX_TC_WORK_64 = 3ll << 20;
constexpr int PREFIX_MAX_PARTS = 64;
constexpr int JOIN_WARP_PARTS = 8;            // parts up to which one warp joins a row
constexpr int CLUSTER_KEYS = 1024;            // keys per part up to which a cluster joins its parts itself
constexpr int DEC_STEP = DEC_WARPS * DEC_KEYS;     // keys per turn of the block; parts are multiples of it

// One source of keys: rows [0, rows) of it belong to one key head; row tile t holds rows [16 t, 16 t + 16)
struct DecodeSide {
    const void *k, *v;
    int64_t k_st[3], v_st[3];
    int row_tiles;                            // per (entry, key head) or, for the prefix, per key head
    int part_keys, parts;
    int first_part;                           // index of its first part in the workspace
    int blocks;                               // row_tiles * parts * key heads (* batch)
};

struct DecodeParams {
    ScoreParams s;
    DecodeSide prefix, own;
    float scale_log2, cap_in, cap_log2;
    float* part_out;                          // [part][batch][heads][head_dim]
    float* part_lse;                          // [part][batch][heads], log2 units
    int stream;                               // > 0: the caches are streamed by this many blocks (own.blocks); own.parts is 1: a whole segment's row
    float* slot_out;                          // [stream][2][16][head_dim]
    float* slot_lse;                          // [stream][2][16]
    int direct;                               // one part in all: write the result itself
    int cluster;                              // > 1: this many parts are one cluster and join in it; parts vary fastest over the blocks
    int prefix_tiles;                         // the prefix runs on the tcgen05 kernel, this many key tiles per part (0: it runs here)
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    const int bytes = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool BF16>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// reads from another block's shared memory (shared::cluster address)
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// {a, b} = hi + lo, both packed in the 16-bit type
template <bool BF16>
__device__ __forceinline__ void split16(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack16(a, b, BF16);
    float ha, hb;
    if constexpr (BF16) {
        ha = __uint_as_float(hi << 16);
        hb = __uint_as_float(hi & 0xFFFF0000u);
    } else {
        const __half2 h = *reinterpret_cast<const __half2*>(&hi);
        ha = __low2float(h);
        hb = __high2float(h);
    }
    lo = pack16(a - ha, b - hb, BF16);
}

// The end of a block.  The first one waits until the grid before this one, if the launch was allowed to overlap it, has ended and its
// writes are visible.
__device__ __forceinline__ void wait_for_prefix() {
    if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Units (64 keys) of the entries before `b` and of all of them, times key heads and row tiles.  One warp.
__device__ __forceinline__ int units_of(const DecodeParams& p, int b) {
    return (min(max(__ldg(p.s.key_lengths + b), 0), p.s.seq_k) + DEC_STEP - 1) / DEC_STEP;
}
__device__ __forceinline__ void count_units(const DecodeParams& p, int b, int lane, int& before, int& all) {
    before = all = 0;
    for (int i = lane; i < p.s.batch; i += 32) {
        const int u = units_of(p, i);
        all += u;
        if (i < b) before += u;
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        before += __shfl_xor_sync(0xFFFFFFFFu, before, s);
        all += __shfl_xor_sync(0xFFFFFFFFu, all, s);
    }
    const int each = p.s.kv_heads * p.own.row_tiles;     // the plan keeps all units below 2^31
    before *= each;
    all *= each;
}

template <int D, bool BF16, bool CAP, bool BIAS>
__global__ void __launch_bounds__(DEC_WARPS * 32, D > 64 ? 2 : 3)
sm120_score_decode_kernel(const __grid_constant__ DecodeParams p) {
    constexpr int CH = D / 8;                            // 16-byte pieces per row
    constexpr uint32_t TILE = DEC_KEYS * D * 2;          // bytes of one K (or V) tile
    constexpr int KSTEPS = D / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    const ScoreParams& sp = p.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // blocks: the prefix's first, then the caches'; parts vary slowest, so the blocks that leave at once (a part behind an entry's
    // length) do not crowd together at one place of the grid
    int idx = static_cast<int>(blockIdx.x);
    const bool common = idx < p.prefix.blocks;
    if (!common) idx -= p.prefix.blocks;
    const DecodeSide& side = common ? p.prefix : p.own;
    const bool stream = p.stream > 0 && !common;
    int part = 0, rt, kvh, b;
    int unit = 0, unit_end = 0, seg_units = 0, seg_at = 0;       // streaming: this block's units, the segment's, and the first one's place in it
    if (stream) {
        const int block = idx;
        int before, all;
        count_units(p, 0, lane, before, all);
        const int blocks = min(p.stream, all);           // never more than units: no block between two others is without work
        if (block >= blocks) return wait_for_prefix();
        unit = static_cast<int>(static_cast<int64_t>(all) * block / blocks);
        unit_end = static_cast<int>(static_cast<int64_t>(all) * (block + 1) / blocks);
        // the entry that holds the first unit: 32 entries at a time
        const int each = sp.kv_heads * side.row_tiles;
        int cum = 0;
        for (b = 0; b < sp.batch; b += 32) {
            const int u = b + lane < sp.batch ? units_of(p, b + lane) * each : 0;
            int scan = u;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const int o = __shfl_up_sync(0xFFFFFFFFu, scan, s);
                if (lane >= s) scan += o;
            }
            const unsigned behind = __ballot_sync(0xFFFFFFFFu, cum + scan > unit);
            if (behind != 0u) {
                const int first = __ffs(behind) - 1;
                cum += __shfl_sync(0xFFFFFFFFu, scan - u, first);
                b += first;
                break;
            }
            cum += __shfl_sync(0xFFFFFFFFu, scan, 31);
        }
        // (lengths that another stream rewrites meanwhile give a wrong result, but no entry behind the last and no endless walk)
        seg_units = b < sp.batch ? units_of(p, b) : 0;
        if (seg_units == 0) return wait_for_prefix();
        const int seg = (unit - cum) / seg_units;
        seg_at = (unit - cum) % seg_units;
        kvh = seg / side.row_tiles;
        rt = seg % side.row_tiles;
        idx = block;
    } else {
        if (p.cluster > 1) {
            part = idx % p.cluster;
            idx /= p.cluster;
        }
        rt = idx % side.row_tiles;
        idx /= side.row_tiles;
        kvh = idx % sp.kv_heads;
        idx /= sp.kv_heads;
        b = common ? 0 : idx % sp.batch;
        if (p.cluster <= 1) part = common ? idx : idx / sp.batch;
    }
    for (;;) {
        const int row0 = rt * DEC_ROWS, n_rows = min(DEC_ROWS, (common ? sp.batch * sp.group : sp.group) - row0);
        const int total = common ? sp.prefix_len : min(max(__ldg(sp.key_lengths + b), 0), sp.seq_k);
        int lo, hi;
        int slot = -1, taken = 0;                            // streaming: where a piece of a segment goes, its units
        if (stream) {
            const int left = seg_units - seg_at;
            taken = min(left, unit_end - unit);
            lo = seg_at * DEC_STEP;
            hi = min(total, lo + taken * DEC_STEP);
            if (seg_at > 0) slot = 2 * idx;                  // begun by another block
            else if (taken < left) slot = 2 * idx + 1;       // left to another block
        } else {
            lo = part * side.part_keys;
            hi = min(total, lo + side.part_keys);
            if (lo >= hi && p.cluster <= 1 && !(p.direct && part == 0)) return wait_for_prefix();      // the join does not read this part
        }

        // query fragments: rows lane / 4 and lane / 4 + 8, columns 2 (lane % 4) + {0, 1, 8, 9} of each K step
        auto row_entry = [&](int r) { return common ? (row0 + r) / sp.group : b; };
        auto row_head = [&](int r) { return kvh * sp.group + (common ? (row0 + r) % sp.group : row0 + r); };
        uint32_t qf[KSTEPS][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = (lane >> 2) + 8 * half;
            const bool live = r < n_rows;
            const uint16_t* q = static_cast<const uint16_t*>(sp.q) + (live ? row_entry(r) * sp.q_st[0] + row_head(r) * sp.q_st[1] : 0);
#pragma unroll
            for (int t = 0; t < KSTEPS; ++t)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int col = t * 16 + c * 8 + (lane & 3) * 2;
                    qf[t][c * 2 + half] = live && col < sp.head_dim ? *reinterpret_cast<const uint32_t*>(q + col) : 0u;
                }
        }
        float slope[2] = {0.0f, 0.0f}, pos[2] = {0.0f, 0.0f};
        if constexpr (BIAS) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = min((lane >> 2) + 8 * half, n_rows - 1);
                slope[half] = __ldg(sp.slopes + row_head(r)) * SA_LOG2E;
                // keys of the cache follow the prefix: both count from the side's own first key here
                const int len = min(max(__ldg(sp.key_lengths + row_entry(r)), 0), sp.seq_k);
                pos[half] = static_cast<float>(len - 1 + (common ? sp.prefix_len : 0));
            }
        }

        const uint32_t ring = smem_u32(smem) + warp * (DEC_STAGES * 2 * TILE);
        const char* kp = reinterpret_cast<const char*>(static_cast<const uint16_t*>(side.k) + b * side.k_st[0] + kvh * side.k_st[1]);
        const char* vp = reinterpret_cast<const char*>(static_cast<const uint16_t*>(side.v) + b * side.v_st[0] + kvh * side.v_st[1]);
        const int64_t k_row = side.k_st[2] * 2, v_row = side.v_st[2] * 2;
        const int n_tiles = hi > lo ? (hi - lo + DEC_KEYS - 1) / DEC_KEYS : 0;          // of the block; warp w takes w, w + 4, ...
        auto load = [&](int tile, int stage) {
            const uint32_t dst = ring + stage * (2 * TILE);
#pragma unroll
            for (int i = 0; i < DEC_KEYS * CH / 32; ++i) {
                const int piece = i * 32 + lane, r = piece / CH, c = piece % CH;
                const int key = lo + tile * DEC_KEYS + r;
                const bool valid = key < hi && c * 8 < sp.head_dim;
                const uint32_t at = r * (D * 2) + ((c ^ (r & 7)) << 4);
                const int64_t src = valid ? key : 0;
                cp_async16(dst + at, kp + src * k_row + (valid ? c * 16 : 0), valid);
                cp_async16(dst + TILE + at, vp + src * v_row + (valid ? c * 16 : 0), valid);
            }
        };
        float o[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
        float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < DEC_STAGES - 1; ++st) {
            if (warp + st * DEC_WARPS < n_tiles) load(warp + st * DEC_WARPS, st);
            cp_async_commit();
        }
        int stage = 0;
        for (int tile = warp; tile < n_tiles; tile += DEC_WARPS) {
            {
                const int ahead = tile + (DEC_STAGES - 1) * DEC_WARPS;
                const int into = stage == 0 ? DEC_STAGES - 1 : stage - 1;
                if (ahead < n_tiles) load(ahead, into);
                cp_async_commit();
            }
            cp_async_wait<DEC_STAGES - 1>();
            __syncwarp();
            const uint32_t ks = ring + stage * (2 * TILE), vs = ks + TILE;
            // S = Q K^T: matrices (keys 0-7, 8-15) x (K columns 0-7, 8-15 of the step)
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
            const int kr = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
            for (int t = 0; t < KSTEPS; ++t) {
                uint32_t f[4];
                const int c = t * 2 + ((lane >> 3) & 1);
                ldmatrix4(ks + kr * (D * 2) + ((c ^ (kr & 7)) << 4), f);
                mma16<BF16>(s[0], qf[t], f[0], f[1]);
                mma16<BF16>(s[1], qf[t], f[2], f[3]);
            }
            // scores in log2 units; keys behind the part's end count as nothing
            const int key0 = lo + tile * DEC_KEYS + (lane & 3) * 2;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + n * 8 + (i & 1);
                    float z = s[n][i];
                    if constexpr (CAP) z = fmaf(att_rcp(att_exp2(z * p.cap_in) + 1.0f), -2.0f * p.cap_log2, p.cap_log2);
                    else z *= p.scale_log2;
                    if constexpr (BIAS) z = fmaf(slope[i >> 1], static_cast<float>(key) - pos[i >> 1], z);
                    s[n][i] = key < hi ? z : -CUDART_INF_F;
                }
            uint32_t hi_f[4], lo_f[4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float mx = fmaxf(fmaxf(s[0][2 * half], s[0][2 * half + 1]), fmaxf(s[1][2 * half], s[1][2 * half + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
                const float m_new = fmaxf(m[half], mx), m_use = m_new == -CUDART_INF_F ? 0.0f : m_new;
                if (__any_sync(0xFFFFFFFFu, m_new != m[half])) {
                    const float fade = att_exp2(m[half] - m_use);
                    l[half] *= fade;
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        o[n][2 * half] *= fade;
                        o[n][2 * half + 1] *= fade;
                    }
                    m[half] = m_new;
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float p0 = att_exp2(s[n][2 * half] - m_use), p1 = att_exp2(s[n][2 * half + 1] - m_use);
                    l[half] += p0 + p1;
                    split16<BF16>(p0, p1, hi_f[n * 2 + half], lo_f[n * 2 + half]);
                }
            }
            // O += P V: V matrices (keys 0-7, 8-15) x (two blocks of 8 columns), transposed on the way
            const int vr = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                uint32_t f[4];
                const int c = n * 2 + (lane >> 4);
                ldmatrix4_trans(vs + vr * (D * 2) + ((c ^ (vr & 7)) << 4), f);
                mma16<BF16>(o[2 * n], hi_f, f[0], f[1]);
                mma16<BF16>(o[2 * n + 1], hi_f, f[2], f[3]);
                mma16<BF16>(o[2 * n], lo_f, f[0], f[1]);
                mma16<BF16>(o[2 * n + 1], lo_f, f[2], f[3]);
            }
            __syncwarp();                                    // every lane has read the stage that the next turn's load overwrites
            if (++stage == DEC_STAGES) stage = 0;
        }
        cp_async_wait<0>();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 1);
            l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 2);
        }
        // join the four warps in shared memory (the rings are done): rows of D floats, then {m, l} per warp and row
        __syncthreads();
        float* rows = reinterpret_cast<float*>(smem);                                     // [warp][16][D]
        float2* ml = reinterpret_cast<float2*>(smem + DEC_WARPS * DEC_ROWS * D * 4);      // [warp][16]
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = (lane >> 2) + 8 * half;
            float* dst = rows + (warp * DEC_ROWS + r) * D + (lane & 3) * 2;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
            if ((lane & 3) == 0) ml[warp * DEC_ROWS + r] = make_float2(m[half], l[half]);
        }
        __syncthreads();
        float* done = reinterpret_cast<float*>(ml + DEC_WARPS * DEC_ROWS);                // [16][D]: this part's rows, and their denominators
        float* done_lse = done + DEC_ROWS * D;
        for (int i = threadIdx.x; i < n_rows * (D / 4); i += DEC_WARPS * 32) {
            const int r = i / (D / 4), col = i % (D / 4) * 4;
            float top = -CUDART_INF_F;
#pragma unroll
            for (int w = 0; w < DEC_WARPS; ++w) top = fmaxf(top, ml[w * DEC_ROWS + r].x);
            const float base = top == -CUDART_INF_F ? 0.0f : top;
            float sum = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < DEC_WARPS; ++w) {
                const float2 x = ml[w * DEC_ROWS + r];
                const float f = att_exp2(x.x - base);
                const float4 y = *reinterpret_cast<const float4*>(rows + (w * DEC_ROWS + r) * D + col);
                sum = fmaf(f, x.y, sum);
                acc.x = fmaf(f, y.x, acc.x);
                acc.y = fmaf(f, y.y, acc.y);
                acc.z = fmaf(f, y.z, acc.z);
                acc.w = fmaf(f, y.w, acc.w);
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const float lse = sum == 0.0f ? -CUDART_INF_F : base + log2f(sum);
            const int e = row_entry(r), h = row_head(r);
            const int64_t row = static_cast<int64_t>(e) * sp.heads + h;
            if (slot >= 0) {
                const int at = slot * DEC_ROWS + r;
                if (col < sp.head_dim)
                    *reinterpret_cast<float4*>(p.slot_out + static_cast<int64_t>(at) * sp.head_dim + col) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                if (col == 0) p.slot_lse[at] = lse;
            } else if (p.cluster > 1) {
                *reinterpret_cast<float4*>(done + r * D + col) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                if (col == 0) done_lse[r] = lse;
            } else if (p.direct) {
                if (col < sp.head_dim)
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(sp.out) + e * sp.o_st[0] + h * sp.o_st[1] + col) =
                        make_uint2(pack16(acc.x * inv, acc.y * inv, BF16), pack16(acc.z * inv, acc.w * inv, BF16));
                if (col == 0 && sp.lse != nullptr) sp.lse[row] = lse * SA_LN2;
            } else {
                const int64_t at = static_cast<int64_t>(side.first_part + part) * sp.batch * sp.heads + row;
                if (col < sp.head_dim)
                    *reinterpret_cast<float4*>(p.part_out + at * sp.head_dim + col) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                if (col == 0) p.part_lse[at] = lse;
            }
        }
        if (p.cluster > 1) {
            cluster_arrive();
            cluster_wait();
            const uint32_t done_at = smem_u32(done), lse_at = smem_u32(done_lse);
            for (int i = part * DEC_WARPS * 32 + threadIdx.x; i < n_rows * (D / 4); i += p.cluster * DEC_WARPS * 32) {
                const int r = i / (D / 4), col = i % (D / 4) * 4;
                float lse[8], top = -CUDART_INF_F;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    lse[c] = -CUDART_INF_F;
                    if (c < p.cluster) lse[c] = ld_cluster(map_to_cta(lse_at + r * 4, c));
                    top = fmaxf(top, lse[c]);
                }
                const float base = top == -CUDART_INF_F ? 0.0f : top;
                float sum = 0.0f;
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    if (c >= p.cluster) continue;
                    const float w = att_exp2(lse[c] - base);
                    const float4 y = ld_cluster4(map_to_cta(done_at + (r * D + col) * 4, c));
                    sum += w;
                    acc.x = fmaf(w, y.x, acc.x);
                    acc.y = fmaf(w, y.y, acc.y);
                    acc.z = fmaf(w, y.z, acc.z);
                    acc.w = fmaf(w, y.w, acc.w);
                }
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int e = row_entry(r), h = row_head(r);
                if (col < sp.head_dim)
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(sp.out) + e * sp.o_st[0] + h * sp.o_st[1] + col) =
                        make_uint2(pack16(acc.x * inv, acc.y * inv, BF16), pack16(acc.z * inv, acc.w * inv, BF16));
                if (col == 0 && sp.lse != nullptr) sp.lse[static_cast<int64_t>(e) * sp.heads + h] = sum == 0.0f ? -CUDART_INF_F : (base + log2f(sum)) * SA_LN2;
            }
            cluster_arrive();                                // no block leaves while another may still read its rows
            cluster_wait();
        }
        if (!stream) break;
        unit += taken;
        if (unit >= unit_end) break;
        // the next segment begins at its first unit: the next row tile, key head, or entry that has keys
        seg_at = 0;
        if (++rt == side.row_tiles) {
            rt = 0;
            if (++kvh == sp.kv_heads) {
                kvh = 0;
                seg_units = 0;
                while (seg_units == 0 && ++b < sp.batch) seg_units = units_of(p, b);
                if (seg_units == 0) break;                   // not reached: units are left
            }
        }
        __syncthreads();                                     // the join's rows lie where the next loads go
    }
    wait_for_prefix();
}

// WARPS warps per row: warp w sums the parts w, w + WARPS, ... with weights 2^(lse - max), the sums are added in order.  A row has up to
// hundreds of parts when few rows share long keys: four warps and four loads in flight keep that a matter of microseconds; rows with
// few parts (and then many rows) take one warp each (4096 rows x 5 parts x 128: 7.7 us instead of 12.5).
template <bool BF16, int WARPS>
__global__ void __launch_bounds__(128)
sm120_score_decode_join_kernel(const __grid_constant__ DecodeParams p) {
    __shared__ float4 part[4][32];
    __shared__ float part_sum[4];
    const ScoreParams& sp = p.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w0 = warp % WARPS;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (4 / WARPS) + warp / WARPS, all = static_cast<int64_t>(sp.batch) * sp.heads;
    if (WARPS == 1 && row >= all) return;                // with four warps per row the grid is exact
    const int e = static_cast<int>(row / sp.heads), h = static_cast<int>(row % sp.heads);
    const int len = min(max(__ldg(sp.key_lengths + e), 0), sp.seq_k);
    // the parts that were written: all of the prefix's, and the cache's up to the entry's length
    int own_parts = p.own.parts > 0 ? (len + p.own.part_keys - 1) / p.own.part_keys : 0;
    int64_t slot = -1;                                   // streamed: the first piece's row among the slots; the others' are in the next blocks' slots 0
    if (p.stream > 0) {
        own_parts = 0;
        if (len > 0) {
            int begin, units;
            count_units(p, e, lane, begin, units);
            const int mine = units_of(p, e);
            const int hg = h % sp.group;
            begin += (h / sp.group * p.own.row_tiles + hg / DEC_ROWS) * mine;
            // block c of n holds the units from floor(units c / n)
            const int blocks = min(p.stream, units);
            const int64_t first = (static_cast<int64_t>(begin + 1) * blocks - 1) / units, last = (static_cast<int64_t>(begin + mine) * blocks - 1) / units;
            own_parts = static_cast<int>(last - first) + 1;
            if (own_parts > 1) slot = (2 * first + 1) * DEC_ROWS + hg % DEC_ROWS;
            else if (p.prefix.parts == 0) return;        // one block had all of it and wrote the result
        }
    }
    const int parts = p.prefix.parts + own_parts;
    // Part i's denominator and row: pieces of a streamed segment lie in slot 1 of the first block and slot 0 of the following ones.  Selected
    // by address, not by branch: the loads of several parts stay in flight together.
    auto in_slot = [&](int i) { return slot >= 0 && i >= p.prefix.parts; };
    auto row_of = [&](int i) {
        const int k = i - p.prefix.parts;
        return in_slot(i) ? slot + (k > 0 ? (2 * k - 1) * DEC_ROWS : 0) : i * all + row;
    };
    auto lse_of = [&](int i) { return (in_slot(i) ? p.slot_lse : p.part_lse)[row_of(i)]; };
    float top = -CUDART_INF_F;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, lse_of(i));
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
    const float base = top == -CUDART_INF_F ? 0.0f : top;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
    const int col = lane * 4;
    const bool mine = col < sp.head_dim;
#pragma unroll 4
    for (int i = w0; i < parts; i += WARPS) {
        const float w = att_exp2(lse_of(i) - base);
        const float* from = (in_slot(i) ? p.slot_out : p.part_out) + row_of(i) * sp.head_dim;
        const float4 y = *reinterpret_cast<const float4*>(from + (mine ? col : 0));
        sum += w;
        acc.x = fmaf(w, y.x, acc.x);
        acc.y = fmaf(w, y.y, acc.y);
        acc.z = fmaf(w, y.z, acc.z);
        acc.w = fmaf(w, y.w, acc.w);
    }
    if (WARPS > 1) {
        part[warp][lane] = acc;
        if (lane == 0) part_sum[warp] = sum;
        __syncthreads();
        if (warp != 0) return;
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
            const float4 y = part[w][lane];
            sum += part_sum[w];
            acc.x += y.x;
            acc.y += y.y;
            acc.z += y.z;
            acc.w += y.w;
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (mine)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(sp.out) + e * sp.o_st[0] + h * sp.o_st[1] + col) =
            make_uint2(pack16(acc.x * inv, acc.y * inv, BF16), pack16(acc.z * inv, acc.w * inv, BF16));
    if (lane == 0 && sp.lse != nullptr) sp.lse[row] = sum == 0.0f ? -CUDART_INF_F : (base + log2f(sum)) * SA_LN2;
}

// How a call is cut.  A part is at least one turn of a block (64 keys) and at most PART_KEYS: long caches of ragged length then
// balance by themselves, and the workspace's traffic stays below 2 / PART_KEYS of the cache's per query row.
constexpr int64_t PART_KEYS = 1024;
// Caches longer than this are streamed.  Measured, us (a block per segment or 1024-key parts / streamed): 64 x 8 key heads x 128, half-ragged
// lengths up to 512: 22.2 / 29.6, 1024: 49 / 44, 2048: 84 / 76, 4096: 144 / 134; 16 x 16 x 64: 512: 8.3 / 14.3, 4096: 48 / 39
constexpr int64_t DIRECT_KEYS = 768;
struct DecodePlan {
    DecodeParams p;
    int64_t parts;
};

static bool plan_side(DecodeSide& s, int64_t keys, int64_t row_tiles, int64_t heads_and_entries, int64_t fill) {
    s.row_tiles = static_cast<int>(row_tiles);
    s.parts = 0;
    s.blocks = 0;
    s.part_keys = DEC_STEP;
    if (keys == 0) return true;
    const int64_t base = row_tiles * heads_and_entries;
    int64_t parts = fill > base ? fill / base : 1;                              // parts that fill the GPU
    int64_t part = (keys + parts - 1) / parts;
    part = (part + DEC_STEP - 1) / DEC_STEP * DEC_STEP;
    if (part > PART_KEYS) part = PART_KEYS;
    parts = (keys + part - 1) / part;
    if (parts * base > (1ll << 30)) return false;
    s.part_keys = static_cast<int>(part);
    s.parts = static_cast<int>(parts);
    s.blocks = static_cast<int>(parts * base);
    return true;
}

static bool make_plan(const ScoreParams& p, int sms, DecodePlan* plan) {
    DecodeParams& dp = plan->p;
    dp = DecodeParams{};
    dp.s = p;
    dp.scale_log2 = p.scale * SA_LOG2E;
    dp.cap_in = p.softcap > 0.0f ? 2.0f * SA_LOG2E * p.scale / p.softcap : 0.0f;
    dp.cap_log2 = p.softcap * SA_LOG2E;
    const int64_t fill = 2ll * sms;                                             // two blocks per SM
    const int64_t rows = static_cast<int64_t>(p.batch) * p.group;
    if (rows * p.prefix_len * p.kv_heads >= (p.head_dim > 64 ? PREFIX_TC_WORK_128 : PREFIX_TC_WORK_64) && p.group <= ATT_BM) {
        // one block per SM: parts that even out the last wave, a block's start and end counted as four key tiles
        const int64_t tiles = (p.prefix_len + ATT_BN - 1) / ATT_BN, per_tile = ATT_BM / p.group;
        const int64_t base = (p.batch + per_tile - 1) / per_tile * p.kv_heads;
        int64_t best = INT64_MAX;
        for (int64_t parts = 1; parts <= tiles && parts <= PREFIX_MAX_PARTS; ++parts) {
            const int64_t each = (tiles + parts - 1) / parts, cost = (base * parts + sms - 1) / sms * (each + 4);
            if (cost < best && (parts - 1) * each < tiles) {
                best = cost;
                dp.prefix.parts = static_cast<int>(parts);
                dp.prefix_tiles = static_cast<int>(each);
            }
        }
        dp.prefix.row_tiles = 1;
        dp.prefix.part_keys = dp.prefix_tiles * ATT_BN;
    } else if (!plan_side(dp.prefix, p.prefix_len, (rows + DEC_ROWS - 1) / DEC_ROWS, p.kv_heads, fill)) {
        return false;
    }
    if (!plan_side(dp.own, p.seq_k, (p.group + DEC_ROWS - 1) / DEC_ROWS, static_cast<int64_t>(p.kv_heads) * p.batch, fill)) return false;
    dp.prefix.k = p.prefix_k; dp.prefix.v = p.prefix_v;
    dp.prefix.k_st[1] = p.pk_st[0]; dp.prefix.k_st[2] = p.pk_st[1];
    dp.prefix.v_st[1] = p.pv_st[0]; dp.prefix.v_st[2] = p.pv_st[1];
    dp.own.k = p.k; dp.own.v = p.v;
    for (int a = 0; a < 3; ++a) {
        dp.own.k_st[a] = p.k_st[a];
        dp.own.v_st[a] = p.v_st[a];
    }
    dp.own.first_part = dp.prefix.parts;
    if (p.prefix_len == 0) {
        // one cluster per (entry, key head, row tile), if all of them run at once
        const int64_t base = static_cast<int64_t>(dp.own.row_tiles) * p.kv_heads * p.batch;
        int64_t size = 8;
        while (size > 1 && (size * base > fill || (size - 1) * DEC_STEP >= p.seq_k)) size >>= 1;
        const int64_t part = (p.seq_k + size * DEC_STEP - 1) / (size * DEC_STEP) * DEC_STEP;
        if (size > 1 && part <= CLUSTER_KEYS) {
            dp.cluster = static_cast<int>(size);
            dp.own.parts = static_cast<int>(size);
            dp.own.part_keys = static_cast<int>(part);
            dp.own.blocks = static_cast<int>(size * base);
            plan->parts = 1;                             // nothing left to join, no workspace
            dp.direct = 1;
            return true;
        }
    }
    // more units than blocks that run at once: stream long caches, and without a prefix give short ones a block per segment, which needs no join
    const int64_t base = static_cast<int64_t>(dp.own.row_tiles) * p.kv_heads * p.batch;
    const int64_t units = base * ((p.seq_k + DEC_STEP - 1) / DEC_STEP);
    if (p.seq_k > 0 && units > fill && units < (1ll << 31) && p.seq_k > DIRECT_KEYS) {
        dp.stream = static_cast<int>((p.head_dim > 64 ? 2 : 3) * sms);          // registers: two blocks per SM at 128, three at 64
        dp.own.blocks = dp.stream;
        dp.own.parts = p.prefix_len > 0 ? 1 : 0;                                // whole segments wait for the prefix in a part of their own
        dp.own.part_keys = DEC_STEP;
    } else if (p.seq_k > 0 && p.prefix_len == 0 && base >= fill) {
        dp.own.parts = 1;
        dp.own.part_keys = (p.seq_k + DEC_STEP - 1) / DEC_STEP * DEC_STEP;
        dp.own.blocks = static_cast<int>(base);
    }
    plan->parts = static_cast<int64_t>(dp.prefix.parts) + dp.own.parts;
    dp.direct = plan->parts <= 1 && dp.prefix_tiles == 0 && (dp.stream == 0 || p.prefix_len == 0);
    return static_cast<int64_t>(dp.prefix.blocks) + dp.own.blocks < (1ll << 31) && static_cast<int64_t>(p.batch) * p.heads < (1ll << 31);
}

// workspace: parts' rows, slots' rows, parts' denominators, slots' denominators
static size_t part_rows(const DecodePlan& plan) { return plan.p.direct && plan.p.stream == 0 ? 0 : static_cast<size_t>(plan.parts) * plan.p.s.batch * plan.p.s.heads; }
static size_t slot_rows(const DecodePlan& plan) { return static_cast<size_t>(plan.p.stream) * 2 * DEC_ROWS; }
static size_t plan_floats(const DecodePlan& plan) { return (part_rows(plan) + slot_rows(plan)) * (plan.p.s.head_dim + 1); }

bool sa_tc_decode_supported(const ScoreParams& p) {
    if (!sa_tc_types_ok(p) || (p.seq_k < 1 && p.prefix_len < 1)) return false;
    const int64_t qe[2] = {p.batch, p.heads}, ke[3] = {p.batch, p.kv_heads, p.seq_k}, pe[2] = {p.kv_heads, p.prefix_len};
    if (!sa_tma_ok(p.q, p.q_st, qe, 2) || !sa_tma_ok(p.out, p.o_st, qe, 2)) return false;
    if (p.seq_k > 0 && (!sa_tma_ok(p.k, p.k_st, ke, 3) || !sa_tma_ok(p.v, p.v_st, ke, 3))) return false;
    return p.prefix_len < 1 || (sa_tma_ok(p.prefix_k, p.pk_st, pe, 2) && sa_tma_ok(p.prefix_v, p.pv_st, pe, 2));
}

size_t sa_tc_decode_workspace(const ScoreParams& p, int sms) {
    DecodePlan plan;
    if (!make_plan(p, sms, &plan)) return 0;
    return plan_floats(plan) * sizeof(float);
}

template <int D, bool BF16>
static cudaError_t decode_launch(const DecodeParams& dp, int device, cudaStream_t stream) {
    constexpr int SMEM = DEC_WARPS * DEC_STAGES * 2 * DEC_KEYS * D * 2;
    static_assert((DEC_WARPS + 1) * DEC_ROWS * (D * 4 + 8) <= SMEM, "the joins' rows fit the rings");
    const bool cap = dp.s.softcap > 0.0f, bias = dp.s.slopes != nullptr;
    auto kern = cap ? (bias ? sm120_score_decode_kernel<D, BF16, true, true> : sm120_score_decode_kernel<D, BF16, true, false>)
                    : (bias ? sm120_score_decode_kernel<D, BF16, false, true> : sm120_score_decode_kernel<D, BF16, false, false>);
    static std::atomic<uint64_t> attr_done[4];
    std::atomic<uint64_t>& done = attr_done[(cap ? 2 : 0) + (bias ? 1 : 0)];
    const uint64_t bit = 1ull << (device & 63);
    if ((done.load(std::memory_order_acquire) & bit) == 0) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return e;
        done.fetch_or(bit, std::memory_order_release);
    }
    const unsigned blocks = static_cast<unsigned>(dp.prefix.blocks + dp.own.blocks);
    const bool overlap = dp.prefix_tiles > 0;            // the launch before this one is the prefix's
    if (dp.cluster <= 1 && !overlap) {
        kern<<<blocks, DEC_WARPS * 32, SMEM, stream>>>(dp);
        return cudaGetLastError();
    }
    cudaLaunchAttribute attr{};
    if (overlap) {                                       // never with a cluster, which has no prefix
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
    } else {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = static_cast<unsigned>(dp.cluster);
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks, 1, 1);
    cfg.blockDim = dim3(DEC_WARPS * 32, 1, 1);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, dp);
}

cudaError_t sa_tc_decode(const ScoreParams& p, void* workspace, int device, int sms, cudaStream_t stream, int* launches) {
    DecodePlan plan;
    if (!make_plan(p, sms, &plan)) return cudaErrorInvalidValue;
    DecodeParams& dp = plan.p;
    dp.part_out = static_cast<float*>(workspace);
    dp.slot_out = dp.part_out + part_rows(plan) * p.head_dim;
    dp.part_lse = dp.slot_out + slot_rows(plan) * p.head_dim;
    dp.slot_lse = dp.part_lse + part_rows(plan);
    const bool bf16 = p.dtype == SM120_DTYPE_BFLOAT16;
    *launches = 0;
    cudaError_t e = cudaSuccess;
    if (dp.prefix_tiles > 0) {
        e = sa_tc_prefix(p, dp.prefix.parts, dp.prefix_tiles, dp.part_out, dp.part_lse, device, stream);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    if (dp.prefix.blocks + dp.own.blocks > 0) {
        e = p.head_dim > 64 ? (bf16 ? decode_launch<128, true>(dp, device, stream) : decode_launch<128, false>(dp, device, stream))
                            : (bf16 ? decode_launch<64, true>(dp, device, stream) : decode_launch<64, false>(dp, device, stream));
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    if (dp.direct && dp.stream == 0) return e;
    const unsigned rows = static_cast<unsigned>(p.batch) * p.heads;
    const int64_t segments = static_cast<int64_t>(dp.own.row_tiles) * p.kv_heads * p.batch;
    if (plan.parts + dp.stream / segments > JOIN_WARP_PARTS) {
        if (bf16) sm120_score_decode_join_kernel<true, 4><<<rows, 128, 0, stream>>>(dp);
        else sm120_score_decode_join_kernel<false, 4><<<rows, 128, 0, stream>>>(dp);
    } else {
        if (bf16) sm120_score_decode_join_kernel<true, 1><<<(rows + 3) / 4, 128, 0, stream>>>(dp);
        else sm120_score_decode_join_kernel<false, 1><<<(rows + 3) / 4, 128, 0, stream>>>(dp);
    }
    ++*launches;
    return cudaGetLastError();
}

}  // namespace sm120
