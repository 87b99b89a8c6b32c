#pragma once
// Device helpers shared by the tcgen05 attention kernels: bounded waits that are safe after a register
// hand-over, tensor-memory loads and stores, packed fp32 arithmetic, and the register budget of a
// 384-thread block whose first warp group feeds two softmax groups.

#include <cuda.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>
#include <atomic>

#include "gemm_tcgen05_kernel.cuh"

namespace sm120 {

constexpr int ATT_BM = 128;          // query rows per CTA
constexpr int ATT_BN = 128;          // keys per tile
constexpr int ATT_K_STAGES = 3;
constexpr int ATT_V_STAGES = 2;
constexpr int ATT_THREADS = 384;           // warp group 0: TMA, MMA and two idle warps; warp groups 1 and 2: softmax
constexpr int ATT_REGS_LOW = 40;            // registers per thread of warp group 0 after the hand-over
constexpr int ATT_REGS_HIGH = 232;          // ... of the softmax warp groups
constexpr int ATT_REGS_LAUNCH = 168;        // what the kernel must be compiled to (65536 / 384, rounded down to 8)
// setmaxnreg.inc waits, without a limit, for registers that warps of the SAME CTA have released: the eight softmax warps
// may only ask for what the four warps of group 0 give back
static_assert(8 * (ATT_REGS_HIGH - ATT_REGS_LAUNCH) <= 4 * (ATT_REGS_LAUNCH - ATT_REGS_LOW), "register hand-over does not balance");
constexpr float ATT_RESCALE_STEP = 8.0f;   // the reference maximum follows a tile's maximum only beyond this (log2 units)

// 2^x by the hardware unit (MUFU.EX2); -inf gives 0
__device__ __forceinline__ float att_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 / x by the hardware unit (MUFU.RCP); +inf gives 0
__device__ __forceinline__ float att_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Tiled TMA load of one 4-D box into this CTA's shared memory, counted on `bar`
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, uint32_t bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// Tiled TMA store of one 4-D box from shared memory; what lies outside the tensor is clipped
__device__ __forceinline__ void tma_store_4d(const void* tmap, uint32_t src, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
        ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(src), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// two floats rounded to the 16-bit type and packed, the first in the low half
__device__ __forceinline__ uint32_t pack16(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The two threads that share a query row (one per group) hand each other one float per step.  Thread (g, row)
// publishes value and step number; it then waits, bounded like every other wait of the kernel, until its partner has
// published the same step.  Values alternate between two slots, so a thread that is one step ahead never overwrites
// what its partner still has to read.
__device__ __forceinline__ bool pair_exchange(volatile float* vals, volatile int* seq, int g, int row, int step, float v,
                                              float& from_partner, const WaitCtx& w) {
    volatile float* slot = vals + (step & 1) * (2 * ATT_BM);
    const int mine = g * ATT_BM + row, other = (g ^ 1) * ATT_BM + row;
    slot[mine] = v;
    __threadfence_block();
    seq[mine] = step;
    if (seq[other] < step) {
        const unsigned long long t0 = global_timer_ns();
        uint32_t spins = 0;
        while (seq[other] < step) {
            if ((++spins & 63u) == 0u) {
                if (*w.abort_flag != 0u) return false;
                if (global_timer_ns() - t0 > w.limit_ns) {
                    raise_abort(w, 0x65000000u);
                    return false;
                }
            }
        }
    }
    __threadfence_block();
    from_partner = slot[other];
    return true;
}

// The bounded mbarrier wait of the GEMM kernel, fully inlined: a warp whose register count was changed by
// setmaxnreg must not call a function that was compiled for the kernel's launch-time count.
__device__ __forceinline__ bool att_wait(uint32_t bar, uint32_t parity, const WaitCtx& w, uint32_t code, bool watch_abort = true) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = global_timer_ns();
    uint32_t spins = 0;
    for (;;) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((++spins & 31u) == 0u) {
            if (watch_abort && *w.abort_flag != 0u) return false;
            if (global_timer_ns() - t0 > w.limit_ns) {
                raise_abort(w, code);
                return false;
            }
        }
    }
}

// Two barriers that are both expected to be complete already: the two tests are in flight together, so the usual case
// costs one round trip to the barrier unit instead of two (the MMA-issuing thread's waits are on every tile's path)
__device__ __forceinline__ bool att_wait2(uint32_t bar_a, uint32_t parity_a, uint32_t bar_b, uint32_t parity_b, const WaitCtx& w,
                                          uint32_t code_a, uint32_t code_b) {
    const bool a = mbar_try_wait(bar_a, parity_a), b = mbar_try_wait(bar_b, parity_b);
    if (a && b) return true;
    if (!a && !att_wait(bar_a, parity_a, w, code_a)) return false;
    return b || att_wait(bar_b, parity_b, w, code_b);
}

// D[tmem] (+)= A[tmem] * B[smem]: the A operand (M = 128 lanes x 16 K elements, two 16-bit elements per 32-bit cell)
// comes from tensor memory
__device__ __forceinline__ void umma_ts_f16(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// 32 TMEM lanes x 16 consecutive 32-bit columns -> 16 registers per thread; the registers are valid when it returns
__device__ __forceinline__ void tmem_ld_32x16_sync(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 32 (16) registers per thread -> 32 TMEM lanes x 32 (16) consecutive 32-bit columns (thread i of the warp owns
// lane i); complete after tmem_st_wait()
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
           "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
           "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
           "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
           "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// Two fp32 values in one 64-bit register pair, and the packed fp32 arithmetic of sm_100 on them: one issue slot for
// two results
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f32x2_split(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// tanh(u) / u for |u| <= SA_TANH_RANGE as a polynomial in v = u^2 on the FMA pipe: the interpolant of degree 5 at the Chebyshev nodes of
// [0, 0.64], off by at most 4e-8; with the roundings of an fp32 evaluation tanh is off by 1.1e-7, what 1 - 2 / (1 + e^2u) from the
// MUFU unit gives as well.  Capped scores are rarely beyond: 0.8 is a score of 0.8 caps.
constexpr float SA_TANH_RANGE = 0.8f;
__device__ __forceinline__ uint64_t sa_tanh_ratio2(uint64_t v2) {
    uint64_t r = fma2(v2, f32x2(-4.34973891e-3f, -4.34973891e-3f), f32x2(1.90843537e-2f, 1.90843537e-2f));
    r = fma2(r, v2, f32x2(-5.3109269e-2f, -5.3109269e-2f));
    r = fma2(r, v2, f32x2(0.133209318f, 0.133209318f));
    r = fma2(r, v2, f32x2(-0.333326655f, -0.333326655f));
    return fma2(r, v2, f32x2(0.999999941f, 0.999999941f));
}

// the three-input maximum / minimum of sm_100: half the instructions and half the chain length of a row's search
__device__ __forceinline__ float att_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float att_min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

}  // namespace sm120
