// Rotary positions with several axes (time, height, width, ...) on query and key heads of 128 channels, with the RMS
// norm of the head in front, in 16 bits (rotary_kernel) or straight to E4M3 codes with one scale for each head and 128
// tokens (rotary_quant_kernel).
//
//   y = turn(x * w / sqrt(mean(x^2) + eps)),   (a, b) -> (a cos t - b sin t, a sin t + b cos t) for each pair of channels,
//   t = position[axis of the pair] * frequency of the pair.
//
// Angles.  A float32 product position * frequency is off by 2^-24 of itself: 2e-3 radians at position 30000.  So the
// product is taken in float64 in units of whole turns, its fractional part (exact) rounded to float32, and sincospif gives
// both functions: off by about 2e-7 whatever the position.  A head is 64 pairs, so a token costs 64 double products and
// 64 sincospif, shared by all its heads; everything else is float32, rounded once when it is stored.

#include <math.h>

#include "common.cuh"
#include "rows.cuh"

namespace ovc {
namespace {

constexpr int kPairs = kDim / 2;

struct Angles {
    const void* positions;  // [S, axes] or [B, S, axes]
    long long batch_stride; // in elements; 0: the same positions for every batch item
    int type, axes;
    float eps;
    double turns[kPairs];   // frequency / 2 pi of each pair; 0 leaves the pair as it is
    uint8_t axis[kPairs];
};

// cos and sin of one pair at one token.
__device__ __forceinline__ float2 pair_turn(const Angles& a, long long row, int pair) {
    const double f = a.turns[pair];
    const long long at = row + a.axis[pair];
    double pos;
    if (a.type == OVC_POSITIONS_I32) pos = static_cast<double>(__ldg(static_cast<const int*>(a.positions) + at));
    else if (a.type == OVC_POSITIONS_I64) pos = static_cast<double>(__ldg(static_cast<const long long*>(a.positions) + at));
    else pos = static_cast<double>(__ldg(static_cast<const float*>(a.positions) + at));
    const double turns = f == 0.0 ? 0.0 : pos * f;
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    return make_float2(c, s);
}

// Eight channels 8 * c16 .. of one head, sixteen lanes to a head.  kHalf: channel i is paired with channel i + 64, held
// by lane c16 ^ 8, and cs[e] belongs to channel 8 * (c16 & 7) + e; otherwise neighbours are paired and cs[0..3] are used.
// `lanes`: the sixteen lanes of the head.
template <bool kHalf>
__device__ __forceinline__ void norm_turn(float (&x)[8], const float* w, float eps, const float2* cs, int c16, uint32_t lanes) {
    if (w != nullptr) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(lanes, sum, o);
        const float r = rsqrtf(fmaf(sum, 1.0f / kDim, eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
    }
    if (kHalf) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float other = __shfl_xor_sync(lanes, x[i], 8);
            x[i] = fmaf(x[i], cs[i].x, (c16 < 8 ? -other : other) * cs[i].y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = fmaf(a, cs[i].x, -b * cs[i].y);
            x[2 * i + 1] = fmaf(a, cs[i].y, b * cs[i].x);
        }
    }
}

template <int DT>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
    if (DT == OVC_BF16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}

struct Source {
    const uint16_t* x;
    void* y;
    const float* weight;                 // [128] or null: no norm
    long long batch, token, head;        // strides of x in elements
    int heads;
    float* descale;                      // rotary_quant_kernel only
    long long descale_stride;
};
struct RotaryArgs {
    Angles angles;
    Source src[2];
    long long S, tokens;                 // tokens = B * S
    float* amax_init;                    // rotary_quant_kernel: optional [H], set to 0
};

constexpr int kRowsAhead = 4;  // heads that a half warp has in flight

// HBM bound: 4 bytes per element (2 read, 2 written).  Sixteen lanes hold a head (16 bytes each), a CTA is sixteen such
// half warps: `token_tile` of them on tokens of their own, the others on further heads of the same tokens, so that a lane
// computes its four (or eight) angles once and keeps them in registers for all heads it visits.  gridDim.y splits the heads
// where there are few tokens.
template <int DT, bool kHalf>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs a, int token_tile, int rows_per_cta) {
    const int c16 = threadIdx.x & 15, half_warp = threadIdx.x >> 4;
    const uint32_t lanes = 0xFFFFu << (threadIdx.x & 16);
    const long long token = static_cast<long long>(blockIdx.x) * token_tile + half_warp % token_tile;
    if (token >= a.tokens) return;
    const int step = 16 / token_tile;
    const long long b = token / a.S, s = token - b * a.S;

    float2 cs[kHalf ? 8 : 4];
#pragma unroll
    for (int i = 0; i < (kHalf ? 8 : 4); ++i)
        cs[i] = pair_turn(a.angles, b * a.angles.batch_stride + s * a.angles.axes, kHalf ? 8 * (c16 & 7) + i : 4 * c16 + i);

    // The heads of q and then those of k are one list; this CTA has [first, last) of it.
    const int first = blockIdx.y * rows_per_cta;
    const int last = min(first + rows_per_cta, a.src[0].heads + a.src[1].heads);
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const Source& t = a.src[which];
        const int before = which == 0 ? 0 : a.src[0].heads;
        const int end = min(last - before, t.heads);
        const uint16_t* x = t.x + b * t.batch + s * t.token + c16 * 8;
        uint4* y = reinterpret_cast<uint4*>(t.y) + token * t.heads * (kDim / 8) + c16;
        float w[8];
        if (t.weight != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __ldg(t.weight + c16 * 8 + i);
        }
        for (int h = max(first - before, 0) + half_warp / token_tile; h < end; h += kRowsAhead * step) {
            uint4 raw[kRowsAhead];
#pragma unroll
            for (int u = 0; u < kRowsAhead; ++u)
                if (h + u * step < end) raw[u] = ld_stream(x + (h + u * step) * t.head);
#pragma unroll
            for (int u = 0; u < kRowsAhead; ++u) {
                if (h + u * step >= end) break;
                float f[8];
                widen8<DT>(raw[u], f);
                norm_turn<kHalf>(f, t.weight != nullptr ? w : nullptr, a.angles.eps, cs, c16, lanes);
                y[static_cast<long long>(h + u * step) * (kDim / 8)] =
                    make_uint4(narrow2<DT>(f[0], f[1]), narrow2<DT>(f[2], f[3]), narrow2<DT>(f[4], f[5]), narrow2<DT>(f[6], f[7]));
            }
        }
    }
}

// The Q/K quantiser with the rotation in front: the turned values stay in float32 registers until their block's maximum
// is known, so they are rounded once, to E4M3.  A CTA holds the angles of one block of 128 tokens in shared memory (64 KB)
// and walks `rows_per_cta` heads of the list (heads of q, heads of k), 256 threads, eight tokens of sixteen bytes per thread,
// the next head's loads issued before this head's maximum is reduced.  3 bytes per element (2 read, 1 written).
template <int DT, bool kHalf>
__global__ void __launch_bounds__(256, 2) rotary_quant_kernel(const __grid_constant__ RotaryArgs a, int blocks, int rows_per_cta) {
    extern __shared__ __align__(16) float2 table[];  // [128][64]
    __shared__ float part[2][8];
    const int c16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const uint32_t lanes = 0xFFFFu << (threadIdx.x & 16);
    const int blk = blockIdx.x;
    const long long b = blockIdx.z;
    const long long row0 = static_cast<long long>(blk) * kTile;
    for (int i = threadIdx.x; i < kTile * kPairs; i += 256) {
        const long long s = row0 + i / kPairs;
        if (s < a.S) table[i] = pair_turn(a.angles, b * a.angles.batch_stride + s * a.angles.axes, i % kPairs);
        else table[i] = make_float2(1.0f, 0.0f);
    }
    const int heads = a.src[0].heads;
    const int first = blockIdx.y * rows_per_cta, last = min(first + rows_per_cta, 2 * heads);
    uint4 raw[8];
    const auto load = [&](int row) {
        const Source& t = a.src[row >= heads];
        const uint16_t* x = t.x + b * t.batch + (row >= heads ? row - heads : row) * t.head + c16 * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long long s = row0 + r0 + 16 * i;
            raw[i] = s < a.S ? ld_stream(x + s * t.token) : make_uint4(0, 0, 0, 0);
        }
    };
    load(first);
    __syncthreads();
    for (int row = first; row < last; ++row) {
        const Source& t = a.src[row >= heads];
        const int head = row >= heads ? row - heads : row;
        float w[8];
        if (t.weight != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __ldg(t.weight + c16 * 8 + i);
        }
        float y[8][8], m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float2 cs[kHalf ? 8 : 4];
            const float4* from = reinterpret_cast<const float4*>(table + (r0 + 16 * i) * kPairs + (kHalf ? 8 * (c16 & 7) : 4 * c16));
#pragma unroll
            for (int e = 0; e < (kHalf ? 4 : 2); ++e) {
                const float4 two = from[e];
                cs[2 * e] = make_float2(two.x, two.y), cs[2 * e + 1] = make_float2(two.z, two.w);
            }
            widen8<DT>(raw[i], y[i]);
            norm_turn<kHalf>(y[i], t.weight != nullptr ? w : nullptr, a.angles.eps, cs, c16, lanes);
            m = absmax8(y[i], m);
        }
        if (row + 1 < last) load(row + 1);
        const float amax = fmaxf(cta256_max(m, part[row & 1]), kFloor);
        const float scale = div_full(kQMax, amax);
        if (threadIdx.x == 0) {
            float* descale = t.descale + (b * heads + head) * t.descale_stride;
            descale[blk] = div_full(amax, kQMax);
            if (blk == 0 && t.descale_stride > blocks) descale[blocks] = 1.0f;
            if (blk == 0 && row < heads && a.amax_init != nullptr) a.amax_init[b * heads + head] = 0.0f;
        }
        uint8_t* dst = static_cast<uint8_t*>(t.y) + ((b * a.S + row0) * heads + head) * kDim + c16 * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = r0 + 16 * i;
            if (row0 + r < a.S) *reinterpret_cast<uint2*>(dst + static_cast<long long>(r) * heads * kDim) = quantize8(y[i], scale);
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

bool take_angles(const ovc_rotary* r, Angles* out) {
    if (!r || !r->positions || !r->turns || !r->pair_axis || r->axes < 1 || r->axes > 64 || !(r->eps >= 0.0f) || !isfinite(r->eps) ||
        (r->position_type != OVC_POSITIONS_I32 && r->position_type != OVC_POSITIONS_I64 && r->position_type != OVC_POSITIONS_F32) ||
        r->position_batch_stride < 0 || (reinterpret_cast<uintptr_t>(r->positions) & (r->position_type == OVC_POSITIONS_I64 ? 7u : 3u)))
        return false;
    out->positions = r->positions, out->batch_stride = r->position_batch_stride;
    out->type = r->position_type, out->axes = r->axes, out->eps = r->eps;
    for (int i = 0; i < kPairs; ++i) {
        if (!isfinite(r->turns[i]) || r->pair_axis[i] >= r->axes) return false;
        out->turns[i] = r->turns[i], out->axis[i] = r->pair_axis[i];
    }
    return true;
}

bool take_source(const void* x, void* y, const float* weight, const int64_t* strides, int64_t heads, uintptr_t out_mask, Source* out) {
    if (!x || !y || !strides || !aligned16(x) || (reinterpret_cast<uintptr_t>(y) & out_mask) || (reinterpret_cast<uintptr_t>(weight) & 3u) ||
        strides[0] < 0 || strides[1] < 0 || strides[2] < 0 || strides[0] % 8 || strides[1] % 8 || strides[2] % 8)
        return false;
    out->x = static_cast<const uint16_t*>(x), out->y = y, out->weight = weight;
    out->batch = strides[0], out->token = strides[1], out->head = strides[2], out->heads = static_cast<int>(heads);
    return true;
}

bool bad_shape(int dtype, int64_t B, int64_t S, int64_t Hq, int64_t Hk) {
    return (dtype != OVC_F16 && dtype != OVC_BF16) || B < 1 || S < 1 || Hq < 1 || Hk < 1 || Hq > 65535 || Hk > 65535 || B > 32767 ||
           S > (1LL << 30) || B * S > 0x7FFFFFFFLL;
}

}  // namespace
}  // namespace ovc

using namespace ovc;

extern "C" int ovc_rotary_qk(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype, int64_t B,
                             int64_t S, int64_t Hq, int64_t Hk, const ovc_rotary* rotary, void* q_out, void* k_out, void* stream) {
    RotaryArgs a{};
    if (bad_shape(dtype, B, S, Hq, Hk) || !take_angles(rotary, &a.angles) ||
        !take_source(q, q_out, rotary->q_weight, q_strides, Hq, 15, &a.src[0]) ||
        !take_source(k, k_out, rotary->k_weight, k_strides, Hk, 15, &a.src[1]))
        return OVC_ERR_ARGUMENT;
    a.S = S, a.tokens = B * S;
    // As many tokens per CTA (up to sixteen) as leave a few CTAs per SM, more where a token has fewer heads than the CTA's
    // half warps; with one token per CTA and still too few CTAs, the heads are split.
    const int rows = static_cast<int>(Hq + Hk);
    int tile = 16;
    while (tile > 1 && (ceil_div(a.tokens, tile) < 4 * 148 && 16 / tile < rows)) tile /= 2;
    int splits = 1;
    while (ceil_div(a.tokens, tile) * splits < 2 * 148 && splits * (16 / tile) < rows) ++splits;
    const int per_cta = static_cast<int>(ceil_div(rows, splits));
    const dim3 grid(static_cast<unsigned>(ceil_div(a.tokens, tile)), static_cast<unsigned>(ceil_div(rows, per_cta)));
    auto s = static_cast<cudaStream_t>(stream);
    if (dtype == OVC_BF16 && rotary->half_split) rotary_kernel<OVC_BF16, true><<<grid, 256, 0, s>>>(a, tile, per_cta);
    else if (dtype == OVC_BF16) rotary_kernel<OVC_BF16, false><<<grid, 256, 0, s>>>(a, tile, per_cta);
    else if (rotary->half_split) rotary_kernel<OVC_F16, true><<<grid, 256, 0, s>>>(a, tile, per_cta);
    else rotary_kernel<OVC_F16, false><<<grid, 256, 0, s>>>(a, tile, per_cta);
    return check_launch();
}

namespace {

int launch_rotary_quant(const void* q, const void* k, int dtype, int64_t B, int64_t S, int64_t H, const ovc_rotary* rotary, void* q8,
                        void* k8, float* q_descale, int64_t q_stride, float* k_descale, int64_t k_stride, float* amax_init, void* stream) {
    const int64_t blocks = ceil_div(S, kTile);
    const int64_t strides[3] = {S * H * kDim, H * kDim, kDim};
    RotaryArgs a{};
    if (bad_shape(dtype, B, S, H, H) || !q_descale || !k_descale || q_stride < blocks || k_stride < blocks || !take_angles(rotary, &a.angles) ||
        !take_source(q, q8, rotary->q_weight, strides, H, 7, &a.src[0]) || !take_source(k, k8, rotary->k_weight, strides, H, 7, &a.src[1]))
        return OVC_ERR_ARGUMENT;
    a.S = S, a.tokens = B * S, a.amax_init = amax_init;
    a.src[0].descale = q_descale, a.src[0].descale_stride = q_stride;
    a.src[1].descale = k_descale, a.src[1].descale_stride = k_stride;
    // A CTA computes its block's angles once, so it takes as many heads as leave a few CTAs per SM.
    const int rows = static_cast<int>(2 * H);
    const int64_t splits = ceil_div(4 * 2 * 148, blocks * B);
    const int per_cta = static_cast<int>(splits >= rows ? 1 : ceil_div(rows, splits));
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(ceil_div(rows, per_cta)), static_cast<unsigned>(B));
    constexpr int smem = kTile * kPairs * static_cast<int>(sizeof(float2));
    auto s = static_cast<cudaStream_t>(stream);
    const auto launch = [&](auto kernel) {
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (err != cudaSuccess) { set_last_cuda_error(err); return static_cast<int>(OVC_ERR_CUDA); }
        kernel<<<grid, 256, smem, s>>>(a, static_cast<int>(blocks), per_cta);
        return check_launch();
    };
    if (dtype == OVC_BF16) return rotary->half_split ? launch(rotary_quant_kernel<OVC_BF16, true>) : launch(rotary_quant_kernel<OVC_BF16, false>);
    return rotary->half_split ? launch(rotary_quant_kernel<OVC_F16, true>) : launch(rotary_quant_kernel<OVC_F16, false>);
}

}  // namespace

extern "C" int ovc_quantize_qk_rotary(const void* q, const void* k, int dtype, int64_t B, int64_t S, int64_t H, const ovc_rotary* rotary,
                                      void* q8, void* k8, float* q_descale, int64_t q_stride, float* k_descale, int64_t k_stride, void* stream) {
    return launch_rotary_quant(q, k, dtype, B, S, H, rotary, q8, k8, q_descale, q_stride, k_descale, k_stride, nullptr, stream);
}

extern "C" int ovc_prepare_fused_rotary(const void* q, const void* k, const void* v, int dtype, int64_t S, int64_t H, const ovc_rotary* rotary,
                                        void* q8, void* k8, void* v_packed, float* q_descale, float* k_descale, float* v_descale,
                                        float* amax_ws, void* stream) {
    if (!v || !v_packed || !v_descale || !amax_ws || !aligned16(v) || !aligned16(v_packed)) return OVC_ERR_ARGUMENT;
    const int64_t blocks = ceil_div(S, kTile);
    const int rc = launch_rotary_quant(q, k, dtype, 1, S, H, rotary, q8, k8, q_descale, (blocks + 1) / 2 * 2, k_descale, blocks, amax_ws, stream);
    return rc != OVC_OK ? rc : launch_amax_cast_pack_v(v, dtype, S, H, amax_ws, v_packed, v_descale, stream);
}
