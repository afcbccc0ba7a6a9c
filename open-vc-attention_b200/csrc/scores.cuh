// What the attention kernels share on the CUDA cores: bounded barrier waits, and arithmetic on rows of scores held in
// registers.
#pragma once

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace ovc {
namespace {

// A wait on a barrier that ends.  The hardware suspends the thread inside try_wait while the phase is pending, so a
// waiting warp issues almost nothing; the abort flag and the clock are looked at only every 16th wake-up.  Returns false
// when the barrier did not complete within `limit` clock ticks (after `give_up()`) or another thread of the CTA already
// gave up; the caller then leaves its loop and the CTA tears down.
constexpr long long kWaitCycles = 400000000LL;  // ~0.2 s
constexpr uint32_t kSleepHintNs = 100000;       // one hardware-suspended try_wait lasts at most this

template <class GiveUp>
__device__ __forceinline__ bool wait_bounded(volatile uint32_t* abort_flag, uint64_t* bar, uint32_t parity, long long limit,
                                             GiveUp give_up) {
    const uint32_t addr = ptx::smem_addr(bar);
    if (ptx::mbar_try_wait(addr, parity)) return true;
    long long start = 0;
#pragma unroll 1
    for (uint32_t tries = 1;; ++tries) {
        if (ptx::mbar_try_wait_sleep(addr, parity, kSleepHintNs)) return true;
        if ((tries & 15u) == 0) {
            if (*abort_flag) return false;
            const long long now = clock64();
            if (start == 0) start = now;
            if (now - start > limit) {
                give_up();
                return false;
            }
        }
    }
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pack_u2(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
// Row max of 128 scores: a three-input max tree per 32 columns (the order in which a tensor-memory load fills
// the registers), then the four partial results; 64 instructions.
__device__ __forceinline__ float max32(const uint32_t* s) {
    float a[11];
#pragma unroll
    for (int c = 0; c < 10; ++c)
        a[c] = fmax3(__uint_as_float(s[3 * c]), __uint_as_float(s[3 * c + 1]), __uint_as_float(s[3 * c + 2]));
    a[10] = fmaxf(__uint_as_float(s[30]), __uint_as_float(s[31]));
    const float b0 = fmax3(a[0], a[1], a[2]), b1 = fmax3(a[3], a[4], a[5]), b2 = fmax3(a[6], a[7], a[8]);
    return fmax3(fmax3(b0, b1, b2), a[9], a[10]);
}
__device__ __forceinline__ float max128(const uint32_t (&s)[128]) {
    return fmaxf(fmax3(max32(s), max32(s + 32), max32(s + 64)), max32(s + 96));
}

__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace
}  // namespace ovc
