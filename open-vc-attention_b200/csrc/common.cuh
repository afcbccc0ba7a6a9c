// Shared helpers for the libovc.so translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "ovc.h"

namespace ovc {

// Last CUDA error code seen by a failing entry point (per host thread).
void set_last_cuda_error(int code);

inline int check_launch() {
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) {
        set_last_cuda_error(static_cast<int>(err));
        return OVC_ERR_CUDA;
    }
    return OVC_OK;
}

#ifdef __CUDACC__
// A kernel launched behind another of its stream without the gap between them: its CTAs may start as soon as all CTAs of the
// one before have called release_next() (or have ended) and leave room.  Until wait_for_previous() it may only read what
// neither of the two writes, and write nothing.  In a kernel launched in the ordinary way both are empty.
// A preparation with rotation and norm in a graph, [32768, 8, 128]: 86 -> 79 us, [1024, 2, 128]: 14.2 -> 12.1,
// [73397, 14, 128]: 0 to 4 % from run to run; without rotation [32768, 8, 128] 86 -> 82, [73397, 56, 128] 1054 -> 1048.
template <class... Parameters, class... Arguments>
int launch_behind(void (*kernel)(Parameters...), dim3 grid, unsigned threads, cudaStream_t stream, Arguments... arguments) {
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid, config.blockDim = dim3(threads), config.stream = stream;
    config.attrs = &early, config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...);
    if (err != cudaSuccess) {
        cudaGetLastError();
        set_last_cuda_error(static_cast<int>(err));
        return OVC_ERR_CUDA;
    }
    return OVC_OK;
}
__device__ __forceinline__ void release_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

// The V part of the fused preparation (prep.cu): per-head max |v| into amax_ws (which an earlier kernel on the stream has
// reset), then the cast with the packed layout.  Arguments are the callers' to check.
int launch_amax_cast_pack_v(const void* v, int dtype, int64_t S, int64_t H, float* amax_ws, void* v_packed, float* v_descale,
                            void* stream);

// The same with row-major codes, for a batch.
int launch_amax_cast_v(const void* v, int dtype, int64_t B, int64_t S, int64_t H, float* amax_ws, void* codes, float* v_descale,
                       void* stream);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kTile = 128;  // tokens per quantisation block and per key tile
constexpr int kDim = 128;   // head dimension

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

#ifdef __CUDACC__
// a / b as the reference's Triton kernels compute it on a GPU: div.full.f32, the dividend times the
// hardware's approximate reciprocal of b, rounded once (not the IEEE quotient).
__device__ __forceinline__ float div_full(float a, float b) {
    float q;
    asm("div.full.f32 %0, %1, %2;" : "=f"(q) : "f"(a), "f"(b));
    return q;
}
#endif

}  // namespace ovc
