// Rows of 128 channels held eight channels to a thread: 16-byte loads, exact widening, E4M3 codes with one scale,
// and the maximum over a CTA.  Shared by the preparation kernels and the rotary kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace ovc {
namespace {

constexpr float kQMax = 448.0f;
constexpr float kFloor = 1e-12f;

__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}

// Eight 16-bit floats (one uint4) widened exactly to float32.
template <int DT>
__device__ __forceinline__ void widen8(const uint4& raw, float (&f)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == OVC_BF16) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
}

__device__ __forceinline__ float absmax8(const float (&f)[8], float m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));
    return m;
}

__device__ __forceinline__ float clamp448(float x) { return fminf(fmaxf(x, -kQMax), kQMax); }

// Four float32 -> four E4M3 bytes (a in the lowest byte), RNE.
__device__ __forceinline__ uint32_t cast4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

__device__ __forceinline__ uint2 quantize8(const float (&f)[8], float scale) {
    uint2 out;
    out.x = cast4(clamp448(__fmul_rn(f[0], scale)), clamp448(__fmul_rn(f[1], scale)),
                  clamp448(__fmul_rn(f[2], scale)), clamp448(__fmul_rn(f[3], scale)));
    out.y = cast4(clamp448(__fmul_rn(f[4], scale)), clamp448(__fmul_rn(f[5], scale)),
                  clamp448(__fmul_rn(f[6], scale)), clamp448(__fmul_rn(f[7], scale)));
    return out;
}

__device__ __forceinline__ float warp_max(float m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    return m;
}

// Max over the 256 threads of a CTA; every thread gets the result.  `part` is caller-provided shared
// memory (8 floats) so that consecutive reductions can alternate between two buffers.
__device__ __forceinline__ float cta256_max(float m, float* part) {
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    return fmaxf(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])),
                 fmaxf(fmaxf(part[4], part[5]), fmaxf(part[6], part[7])));
}

}  // namespace
}  // namespace ovc
