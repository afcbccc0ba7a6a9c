// Rotary positions with several axes (time, height, width, ...) on query and key heads of 128 channels, with the RMS
// norm of the head in front, in 16 bits (rotary_kernel) or straight to E4M3 codes with one scale for each head and 128
// tokens (rotary_quant_kernel).
//
//   y = turn(x * w / sqrt(mean(x^2) + eps)),   (a, b) -> (a cos t - b sin t, a sin t + b cos t) for each pair of channels,
//   t = position[axis of the pair] * frequency of the pair.
//
// Angles.  A float32 product position * frequency is off by 2^-24 of itself: 2e-3 radians at position 30000.  Only the
// fraction of a turn counts, so a frequency is an integer in units of 2^-64 turns and the product with a position is
// taken modulo 2^64, which drops the whole turns exactly; its upper 32 bits go to sincospif.  The angle is off by about
// 2e-7 for positions up to 2^28, without an instruction in float64; behind those the 53 bits of the frequency that a plan
// gives count (2^-55 turns a position).  Whole turns of a frequency matter to fractional positions only, whose type carries
// them in a second word.  A token has 64 pairs, shared by all its heads; everything else is float32, rounded once when it
// is stored.
//
// A lane holds four pairs of one head and sixteen lanes a head, in both layouts of the pairs (neighbours: 16 bytes in a
// row; halves: 8 bytes from each half of the head), so no value of a pair crosses lanes and both pair members are
// computed two at a time (f32x2).

#include <math.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "rows.cuh"
#include "scores.cuh"

namespace ovc {
namespace {

constexpr int kPairs = kDim / 2;

struct Angles {
    const void* positions;  // [S, axes] or [B, S, axes]
    long long batch_stride; // in elements; 0: the same positions for every batch item
    int type, axes;
    float eps;
    unsigned long long turns[kPairs];  // per position, in units of 2^-64 turns, without the whole turns
    int whole[kPairs];                 // the whole turns, rounded down; 0 unless the positions are float32
    unsigned long long still;          // bit p: pair p is not turned
    uint8_t axis[kPairs];
};

// position * (whole + turns * 2^-64) modulo one turn, in units of 2^-64, for a float32 position m * 2^e.
__device__ __forceinline__ unsigned long long float_turns(float position, unsigned long long turns, int whole) {
    const uint32_t bits = __float_as_uint(position);
    const int field = (bits >> 23) & 255;
    if (field == 0) return 0;  // zero (a subnormal position turns nothing)
    const unsigned long long m = (bits & 0x7FFFFFu) | 0x800000u;
    const unsigned long long lo = m * turns, hi = __umul64hi(m, turns);
    const int e = field - 150;
    const long long n = static_cast<long long>(m) * whole;  // below 2^55
    unsigned long long x;
    if (e >= 0) x = e < 64 ? lo << e : 0;
    else if (e > -64) x = ((lo >> -e) | (hi << (64 + e))) + (static_cast<unsigned long long>(n) << (64 + e));
    else x = (e > -128 ? hi >> (-e - 64) : 0) + static_cast<unsigned long long>(n >> min(-e - 64, 63));
    return bits >> 31 ? 0 - x : x;
}

// The frequencies in shared memory: lanes want different pairs, and the parameters' constant bank serves one address at
// a time (read from there, the angles took twice as long as everything else).
struct Pairs {
    unsigned long long turns[kPairs];
    int whole[kPairs];
    uint8_t axis[kPairs];
};
__device__ __forceinline__ void stage_pairs(const Angles& a, Pairs& pairs) {
    const int i = threadIdx.x;
    if (i < kPairs) pairs.turns[i] = a.turns[i], pairs.whole[i] = a.whole[i], pairs.axis[i] = a.axis[i];
}

// cos and sin of one pair at one token, whose positions start at `row`.
__device__ __forceinline__ float2 pair_turn(const Angles& a, const Pairs& pairs, long long row, int pair) {
    const unsigned long long f = pairs.turns[pair];
    const long long at = row + pairs.axis[pair];
    unsigned long long x;
    bool finite = true;
    if (a.type == OVC_POSITIONS_I32) {
        x = static_cast<unsigned long long>(static_cast<long long>(__ldg(static_cast<const int*>(a.positions) + at))) * f;
    } else if (a.type == OVC_POSITIONS_I64) {
        x = static_cast<unsigned long long>(__ldg(static_cast<const long long*>(a.positions) + at)) * f;
    } else {
        const float position = __ldg(static_cast<const float*>(a.positions) + at);
        const int whole = pairs.whole[pair];
        const bool still = f == 0 && whole == 0;
        finite = isfinite(position) || still;
        x = still ? 0 : float_turns(position, f, whole);
    }
    float s, c;
    sincospif(static_cast<float>(static_cast<int>((x + 0x80000000ull) >> 32)) * 4.656612873077393e-10f, &s, &c);  // 2^-31 half turns
    return finite ? make_float2(c, s) : make_float2(NAN, NAN);
}

__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void split2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }

// Four pairs (a, b): first members a01, a23, second members b01, b23.
struct Four {
    uint64_t a[2], b[2];
};

// 16-bit words: with kHalf x and y are the first members, z and w the second; otherwise a word is a pair.
template <int DT, bool kHalf>
__device__ __forceinline__ Four widen_pairs(const uint4& raw) {
    float f[8];
    widen8<DT>(raw, f);
    Four v;
    if (kHalf) v.a[0] = pack2(f[0], f[1]), v.a[1] = pack2(f[2], f[3]), v.b[0] = pack2(f[4], f[5]), v.b[1] = pack2(f[6], f[7]);
    else v.a[0] = pack2(f[0], f[2]), v.a[1] = pack2(f[4], f[6]), v.b[0] = pack2(f[1], f[3]), v.b[1] = pack2(f[5], f[7]);
    return v;
}
// The values in the order of the stored channels.
template <bool kHalf>
__device__ __forceinline__ void in_order(const Four& v, float (&f)[8]) {
    float a[4], b[4];
    split2(v.a[0], a[0], a[1]), split2(v.a[1], a[2], a[3]), split2(v.b[0], b[0], b[1]), split2(v.b[1], b[2], b[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[kHalf ? i : 2 * i] = a[i];
        f[kHalf ? 4 + i : 2 * i + 1] = b[i];
    }
}
template <bool kHalf>
__device__ __forceinline__ Four load_weights(const float* weight, int c16) {
    const float4 x = reinterpret_cast<const float4*>(weight)[kHalf ? c16 : 2 * c16];
    const float4 y = reinterpret_cast<const float4*>(weight)[kHalf ? c16 + 16 : 2 * c16 + 1];
    Four v;
    if (kHalf) v.a[0] = pack2(x.x, x.y), v.a[1] = pack2(x.z, x.w), v.b[0] = pack2(y.x, y.y), v.b[1] = pack2(y.z, y.w);
    else v.a[0] = pack2(x.x, x.z), v.a[1] = pack2(y.x, y.z), v.b[0] = pack2(x.y, x.w), v.b[1] = pack2(y.y, y.w);
    return v;
}
__device__ __forceinline__ float squares(const Four& v) {
    uint64_t sum = fmul2(v.a[0], v.a[0]);
    sum = ffma2(v.a[1], v.a[1], sum);
    sum = ffma2(v.b[0], v.b[0], sum);
    sum = ffma2(v.b[1], v.b[1], sum);
    float x, y;
    split2(sum, x, y);
    return x + y;
}
__device__ __forceinline__ void times(Four& v, const Four& w) {
#pragma unroll
    for (int i = 0; i < 2; ++i) v.a[i] = fmul2(v.a[i], w.a[i]), v.b[i] = fmul2(v.b[i], w.b[i]);
}
struct Turns {
    uint64_t c[2], s[2], minus_s[2];
};
// The rotation and the weights of the norm in one: a' = aa a + ab b, b' = ba a + bb b.
struct Mix {
    uint64_t aa[2], ab[2], ba[2], bb[2];
};
__device__ __forceinline__ Mix make_mix(const Turns& t, const Four& w) {
    Mix m;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        m.aa[i] = fmul2(w.a[i], t.c[i]), m.ab[i] = fmul2(w.b[i], t.minus_s[i]), m.ba[i] = fmul2(w.a[i], t.s[i]), m.bb[i] = fmul2(w.b[i], t.c[i]);
    return m;
}
__device__ __forceinline__ void turn(Four& v, const Mix& t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t a = v.a[i], b = v.b[i];
        v.a[i] = ffma2(a, t.aa[i], fmul2(b, t.ab[i]));
        v.b[i] = ffma2(a, t.ba[i], fmul2(b, t.bb[i]));
    }
}
__device__ __forceinline__ Turns make_turns(const float4& c, const float4& s) {
    return Turns{{pack2(c.x, c.y), pack2(c.z, c.w)}, {pack2(s.x, s.y), pack2(s.z, s.w)}, {pack2(-s.x, -s.y), pack2(-s.z, -s.w)}};
}
__device__ __forceinline__ void turn(Four& v, const Turns& t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t a = v.a[i], b = v.b[i];
        v.a[i] = ffma2(a, t.c[i], fmul2(b, t.minus_s[i]));
        v.b[i] = ffma2(a, t.s[i], fmul2(b, t.c[i]));
    }
}

// Pairs that are not turned keep their values whatever the other member holds: zero times an infinity is NaN, so their members
// enter each other's products as zero.  `moving` has a bit for each of the lane's pairs that turns.
__device__ __forceinline__ uint64_t moving_mask(uint32_t moving, int i) {
    return pack_u2(moving >> 2 * i & 1 ? ~0u : 0u, moving >> 2 * i & 2 ? ~0u : 0u);
}
__device__ __forceinline__ void turn_moving(Four& v, const Turns& t, uint32_t moving) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t a = v.a[i], b = v.b[i], mask = moving_mask(moving, i);
        v.a[i] = ffma2(a, t.c[i], fmul2(b & mask, t.minus_s[i]));
        v.b[i] = ffma2(a & mask, t.s[i], fmul2(b, t.c[i]));
    }
}
__device__ __forceinline__ void turn_moving(Four& v, const Mix& t, uint32_t moving) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t a = v.a[i], b = v.b[i], mask = moving_mask(moving, i);
        v.a[i] = ffma2(a, t.aa[i], fmul2(b & mask, t.ab[i]));
        v.b[i] = ffma2(a & mask, t.ba[i], fmul2(b, t.bb[i]));
    }
}

// Sums over the sixteen lanes of a head for N = 2, 4 or 8 heads at once: steps in which a lane gives half of its sums away and
// adds up the other half, so that 4 sums cost 5 exchanges instead of 16.  Lane lane_of_sum<N>(i) is left with sum i.
template <int N>
__device__ __forceinline__ constexpr int lane_of_sum(int i) { return i * (16 / N); }
template <int N>
__device__ __forceinline__ float sums_of_heads(float (&v)[N], int c16) {
    int o = 8;
#pragma unroll
    for (int n = N / 2; n >= 1; n >>= 1, o >>= 1) {
        const bool up = c16 & o;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
            v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
        }
    }
    float sum = v[0];
#pragma unroll
    for (int last = 8 / N; last > 0; last >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, last);
    return sum;
}
// 1 / sqrt(mean(x^2) + eps) of N heads.
template <int N>
__device__ __forceinline__ void norm_factors(const Four (&v)[N], float eps, int c16, float (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = squares(v[i]);
    const float mine = rsqrtf(fmaf(sums_of_heads<N>(r, c16), 1.0f / kDim, eps));
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = __shfl_sync(0xFFFFFFFFu, mine, lane_of_sum<N>(i), 16);
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
    int32_t* bounds;                     // rotary_quant_kernel: optional [2], set to 0 and S
};

constexpr int kGroupRows = 8, kUnitGroups = 4, kUnitWarps = 4;

// 16 bytes to shared memory behind the thread's back: what is in flight takes no registers.
__device__ __forceinline__ void copy16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copy8(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
template <int kPending>
__device__ __forceinline__ void wait_copies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// HBM bound: 4 bytes per element (2 read, 2 written).  The heads of a token's q and then of its k are groups of eight, a unit
// is up to four groups of one token.  A warp asks for all heads of its unit at once, computes the token's angles meanwhile -
// four pairs to a lane, kept in registers - and then works through the groups as they arrive, two heads side by side.  With
// norm, the angles are multiplied by the weights once per tensor.  [4, 8191, 24 + 24, 128] with norm, at the clock that the
// power limit leaves after some hundred calls (1.61 GHz): 125 us (805 MB; a copy of that size takes 123 us); with the weights
// loaded and multiplied head by head 131, and with the unit's place found by a 64-bit division 138.  (Groups of one tensor:
// heads of either in a row, which cost every head a choice of pointers and weights, took 143 us where this took 122.)
// kStill, where the plan has pairs that are not turned and a tensor without norm: such pairs keep their values beside an
// infinity.  It costs nothing without norm, 10 % (registers) where only one of the tensors has it.  (A normalised head that holds
// an infinity has nothing but zeros and NaN left.)
template <int DT, bool kHalf, bool kNorm, bool kStill>
__global__ void __launch_bounds__(32 * kUnitWarps, 7)
rotary_kernel(const __grid_constant__ RotaryArgs a, int unit_groups) {
    extern __shared__ __align__(16) uint8_t staged[];
    __shared__ Pairs pairs;
    const int lane = threadIdx.x & 31, c16 = lane & 15, side = lane >> 4;
    const uint32_t wanted = blockIdx.x * kUnitWarps + (threadIdx.x >> 5), tokens = static_cast<uint32_t>(a.tokens);
    const long long token = min(wanted, tokens - 1);
    const int groups0 = (a.src[0].heads + kGroupRows - 1) / kGroupRows, all = groups0 + (a.src[1].heads + kGroupRows - 1) / kGroupRows;
    const int first = blockIdx.y * unit_groups;
    const int count = wanted < tokens ? min(unit_groups, all - first) : 0;
    const long long b = static_cast<uint32_t>(token) / static_cast<uint32_t>(a.S), s = token - b * a.S;
    uint8_t* const mine = staged + (threadIdx.x >> 5) * unit_groups * kGroupRows * 256;

#pragma unroll
    for (int j = 0; j < kUnitGroups; ++j) {
        if (j < count) {
            const Source& t = a.src[first + j >= groups0];
            const int head = (first + j >= groups0 ? first + j - groups0 : first + j) * kGroupRows + side;
            const uint16_t* x = t.x + b * t.batch + s * t.token + head * t.head + 8 * c16;
#pragma unroll
            for (int i = 0; i < kGroupRows; i += 2, x += 2 * t.head)
                if (head + i < t.heads) copy16(mine + (j * kGroupRows + i + side) * 256 + 16 * c16, x);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    stage_pairs(a.angles, pairs);
    __syncthreads();
    if (count == 0) return;
    // Either half of the warp computes two of a lane's four angles.
    float cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 t = pair_turn(a.angles, pairs, b * a.angles.batch_stride + s * a.angles.axes, 4 * c16 + 2 * side + i);
        const float c = __shfl_xor_sync(0xFFFFFFFFu, t.x, 16), s = __shfl_xor_sync(0xFFFFFFFFu, t.y, 16);
        cs[i] = side ? c : t.x, cs[2 + i] = side ? t.x : c;
        sn[i] = side ? s : t.y, sn[2 + i] = side ? t.y : s;
    }
    Turns turns = make_turns(make_float4(cs[0], cs[1], cs[2], cs[3]), make_float4(sn[0], sn[1], sn[2], sn[3]));
    const uint32_t moving = kStill ? ~static_cast<uint32_t>(a.angles.still >> 4 * c16) : 0u;
    if (kStill)  // zero times minus zero added to either member keeps the sign of a zero
#pragma unroll
        for (int i = 0; i < 2; ++i) turns.s[i] |= pack_u2(moving >> 2 * i & 1 ? 0u : 0x80000000u, moving >> 2 * i & 2 ? 0u : 0x80000000u);

    Mix mix;
    for (int j = 0; j < count; ++j) {
        // Every warp has four groups of copies, the last ones empty where it has fewer; those behind j may be under way.
        // Lanes read what other lanes copied, hence the __syncwarp.
        if (j == 0) wait_copies<3>();
        else if (j == 1) wait_copies<2>();
        else if (j == 2) wait_copies<1>();
        else wait_copies<0>();
        __syncwarp();
        const Source& t = a.src[first + j >= groups0];
        const int head = (first + j >= groups0 ? first + j - groups0 : first + j) * kGroupRows + side;
        constexpr int kRows = kGroupRows / 2;
        Four v[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {  // (what lies behind the last head is computed on, and not stored)
            const uint8_t* from = mine + (j * kGroupRows + 2 * i + side) * 256;
            uint4 raw;
            if (kHalf) {
                const uint2 lo = *reinterpret_cast<const uint2*>(from + 8 * c16), hi = *reinterpret_cast<const uint2*>(from + 8 * c16 + 128);
                raw = make_uint4(lo.x, lo.y, hi.x, hi.y);
            } else {
                raw = *reinterpret_cast<const uint4*>(from + 16 * c16);
            }
            v[i] = widen_pairs<DT, kHalf>(raw);
        }
        if (kNorm && t.weight != nullptr) {
            float r[kRows];
            norm_factors<kRows>(v, a.angles.eps, c16, r);
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const uint64_t r2 = pack2(r[i], r[i]);
                times(v[i], Four{{r2, r2}, {r2, r2}});
            }
        }
        if (kNorm && (j == 0 || first + j == groups0)) {
            const uint64_t one = pack2(1.0f, 1.0f);
            mix = make_mix(turns, t.weight != nullptr ? load_weights<kHalf>(t.weight, c16) : Four{{one, one}, {one, one}});
        }
        uint16_t* const y = static_cast<uint16_t*>(t.y) + (token * t.heads + head) * kDim + (kHalf ? 4 : 8) * c16;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (kNorm && kStill && t.weight == nullptr) turn_moving(v[i], mix, moving);
            else if (kNorm) turn(v[i], mix);
            else if (kStill) turn_moving(v[i], turns, moving);
            else turn(v[i], turns);
            float f[8];
            in_order<kHalf>(v[i], f);
            const uint2 lo = make_uint2(narrow2<DT>(f[0], f[1]), narrow2<DT>(f[2], f[3]));
            const uint2 hi = make_uint2(narrow2<DT>(f[4], f[5]), narrow2<DT>(f[6], f[7]));
            if (head + 2 * i < t.heads) {
                if (kHalf) {
                    *reinterpret_cast<uint2*>(y + 2 * i * kDim) = lo;
                    *reinterpret_cast<uint2*>(y + 2 * i * kDim + 64) = hi;
                } else {
                    *reinterpret_cast<uint4*>(y + 2 * i * kDim) = make_uint4(lo.x, lo.y, hi.x, hi.y);
                }
            }
        }
    }
}

// The Q/K quantiser with the rotation in front: the turned values stay in float32 registers until their block's maximum
// is known, so they are rounded once, to E4M3.  A CTA holds the angles of one block of 128 tokens in shared memory (64 KB)
// and walks `rows_per_cta` heads of the list (heads of q, heads of k), 512 threads, four tokens of four pairs per thread, the
// next head's values copied to shared memory (32 KB) meanwhile.  3 bytes per element (2 read, 1 written).  The norm's factor
// of a row is not multiplied into its values but into the row's maximum and scale.
// [73397, 14 + 14, 128]: 146 us, with norm 162 us (789 MB: 120 us at the rate of a copy); with norm it issues on two of three
// cycles.  Next head in registers: 155 / 185 us.  Max |v| found on the way, instead of by the kernel behind it: 17 us more in
// all.  kStill as above, 1 % and 7 %.
constexpr int kQuantThreads = 512, kQuantRows = kTile * 16 / kQuantThreads, kQuantStep = kQuantThreads / 16;

template <int DT, bool kHalf, bool kNorm, bool kStill>
__global__ void __launch_bounds__(kQuantThreads, 2) rotary_quant_kernel(const __grid_constant__ RotaryArgs a, int blocks, int rows_per_cta) {
    extern __shared__ __align__(16) float table[];  // cos [128][64], sin [128][64]
    __shared__ uint32_t part[2][kQuantThreads / 32];
    __shared__ Pairs pairs;
    const int c16 = threadIdx.x & 15, r0 = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blk = blockIdx.x;
    const long long b = blockIdx.z;
    const long long row0 = static_cast<long long>(blk) * kTile;
    const int tokens = static_cast<int>(min(static_cast<long long>(kTile), a.S - row0));
    const int heads = a.src[0].heads;
    const int first = blockIdx.y * rows_per_cta, last = min(first + rows_per_cta, 2 * heads);
    const uint32_t pitch = static_cast<uint32_t>(heads) * kDim;  // inputs and codes are dense: elements from token to token
    // A thread's tokens, in elements from the block's first (128 tokens stay below 2^31).  Behind the sequence's end the last
    // token is done again: it changes no maximum and stores the same codes.
    uint32_t at[kQuantRows];
#pragma unroll
    for (int i = 0; i < kQuantRows; ++i) at[i] = min(r0 + kQuantStep * i, tokens - 1) * pitch + (kHalf ? 4 : 8) * c16;
    const long long block_at = (b * a.S + row0) * heads * kDim;
    // The next head's values wait in shared memory, sixteen bytes of each token where the thread that copies them reads them.
    uint8_t* const staged = reinterpret_cast<uint8_t*>(table + 2 * kTile * kPairs) + threadIdx.x * 16;
    const auto load = [&](int row) {
        const uint16_t* const x = (row >= heads ? a.src[1].x + (row - heads) * kDim : a.src[0].x + row * kDim) + block_at;
#pragma unroll
        for (int i = 0; i < kQuantRows; ++i) {
            uint8_t* const to = staged + i * kQuantThreads * 16;
            if (kHalf) copy8(to, x + at[i]), copy8(to + 8, x + at[i] + kPairs);
            else copy16(to, x + at[i]);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const uint32_t moving = kStill ? ~static_cast<uint32_t>(a.angles.still >> 4 * c16) : 0u;
    release_next();  // the kernel behind may read V where this one leaves room
    load(first);
    stage_pairs(a.angles, pairs);
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * kPairs; i += kQuantThreads) {
        const long long s = row0 + min(i / kPairs, tokens - 1);
        const float2 t = pair_turn(a.angles, pairs, b * a.angles.batch_stride + s * a.angles.axes, i % kPairs);
        table[i] = t.x, table[kTile * kPairs + i] = t.y;
    }
    __syncthreads();
    if (a.bounds != nullptr && blk == 0 && first == 0 && b == 0 && threadIdx.x < 2) a.bounds[threadIdx.x] = threadIdx.x * static_cast<int>(a.S);
    for (int row = first; row < last; ++row) {
        const Source& t = a.src[row >= heads];
        const int head = row >= heads ? row - heads : row;
        Four v[kQuantRows];
        float r[kQuantRows];
        wait_copies<0>();
#pragma unroll
        for (int i = 0; i < kQuantRows; ++i) v[i] = widen_pairs<DT, kHalf>(*reinterpret_cast<const uint4*>(staged + i * kQuantThreads * 16));
        if (row + 1 < last) load(row + 1);
        const bool norm = kNorm && t.weight != nullptr;
        if (norm) {
            norm_factors<kQuantRows>(v, a.angles.eps, c16, r);
            const Four w = load_weights<kHalf>(t.weight, c16);
#pragma unroll
            for (int i = 0; i < kQuantRows; ++i) times(v[i], w);
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < kQuantRows; ++i) {
            const float* from = table + (r0 + kQuantStep * i) * kPairs + 4 * c16;
            const Turns turns = make_turns(*reinterpret_cast<const float4*>(from), *reinterpret_cast<const float4*>(from + kTile * kPairs));
            if (kStill && !norm) turn_moving(v[i], turns, moving);
            else turn(v[i], turns);
            float f[8];
            in_order<kHalf>(v[i], f);
            float top = fmax3(fabsf(f[0]), fabsf(f[1]), fabsf(f[2]));
            top = fmax3(top, fabsf(f[3]), fabsf(f[4]));
            top = fmax3(top, fabsf(f[5]), fmaxf(fabsf(f[6]), fabsf(f[7])));
            m = fmaxf(m, norm ? top * r[i] : top);
        }
        // (The order of non-negative floats is that of their bits.)
        const uint32_t warp_top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m));
        if (lane == 0) part[row & 1][warp] = warp_top;
        __syncthreads();
        const float amax = fmaxf(__uint_as_float(__reduce_max_sync(0xFFFFFFFFu, part[row & 1][lane & (kQuantThreads / 32 - 1)])), kFloor);
        const float scale = div_full(kQMax, amax);
        if (threadIdx.x == 0) {
            float* descale = t.descale + (b * heads + head) * t.descale_stride;
            descale[blk] = div_full(amax, kQMax);
            if (blk == 0 && t.descale_stride > blocks) descale[blocks] = 1.0f;
            if (blk == 0 && row < heads && a.amax_init != nullptr) a.amax_init[b * heads + head] = 0.0f;
        }
        uint8_t* dst = static_cast<uint8_t*>(t.y) + block_at + head * kDim;
#pragma unroll
        for (int i = 0; i < kQuantRows; ++i) {
            const float k = norm ? scale * r[i] : scale;
            const uint64_t k2 = pack2(k, k);
            times(v[i], Four{{k2, k2}, {k2, k2}});
            float f[8];
            in_order<kHalf>(v[i], f);
            const uint32_t lo = cast4(f[0], f[1], f[2], f[3]), hi = cast4(f[4], f[5], f[6], f[7]);  // (saturates at 448)
            uint8_t* const to = dst + at[i];
            if (kHalf) {
                *reinterpret_cast<uint32_t*>(to) = lo;
                *reinterpret_cast<uint32_t*>(to + kPairs) = hi;
            } else {
                *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
            }
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

constexpr double kMostTurns = 1 << 30;  // per float32 position

bool take_angles(const ovc_rotary* r, Angles* out) {
    if (!r || !r->positions || !r->turns || !r->pair_axis || r->axes < 1 || r->axes > 64 || !(r->eps >= 0.0f) || !isfinite(r->eps) ||
        (r->position_type != OVC_POSITIONS_I32 && r->position_type != OVC_POSITIONS_I64 && r->position_type != OVC_POSITIONS_F32) ||
        r->position_batch_stride < 0 || (reinterpret_cast<uintptr_t>(r->positions) & (r->position_type == OVC_POSITIONS_I64 ? 7u : 3u)))
        return false;
    out->positions = r->positions, out->batch_stride = r->position_batch_stride;
    out->type = r->position_type, out->axes = r->axes, out->eps = r->eps;
    for (int i = 0; i < kPairs; ++i) {
        if (!isfinite(r->turns[i]) || r->pair_axis[i] >= r->axes) return false;
        // Sign and size apart: both parts of the size are exact, and so is their negation (rounded down, a fraction above zero).
        const bool negative = r->turns[i] < 0.0;
        const double size = fabs(r->turns[i]), whole = floor(size);
        const auto fraction = static_cast<unsigned long long>(ldexp(size - whole, 64));
        out->turns[i] = negative ? 0 - fraction : fraction;
        if (r->position_type == OVC_POSITIONS_F32) {
            if (!(size < kMostTurns)) return false;
            out->whole[i] = negative ? -static_cast<int>(whole) - (fraction != 0) : static_cast<int>(whole);
        }
        if (fraction == 0 && out->whole[i] == 0) out->still |= 1ull << i;
        out->axis[i] = r->pair_axis[i];
    }
    return true;
}

bool take_source(const void* x, void* y, const float* weight, const int64_t* strides, int64_t heads, uintptr_t out_mask, Source* out) {
    if (!x || !y || !strides || !aligned16(x) || (reinterpret_cast<uintptr_t>(y) & out_mask) || !aligned16(weight) ||
        strides[0] < 0 || strides[1] < 0 || strides[2] < 0 || strides[0] % 8 || strides[1] % 8 || strides[2] % 8)
        return false;
    out->x = static_cast<const uint16_t*>(x), out->y = y, out->weight = weight;
    out->batch = strides[0], out->token = strides[1], out->head = strides[2], out->heads = static_cast<int>(heads);
    return true;
}

// launch(bf16, half, norm, still) with the four as compile-time constants.
template <class Launch>
int by_variant(int dtype, const ovc_rotary* r, const Angles& angles, Launch launch) {
    const auto by_still = [&](auto bf16, auto half, auto norm) {
        const bool both = r->q_weight && r->k_weight;
        return angles.still && !both ? launch(bf16, half, norm, std::true_type{}) : launch(bf16, half, norm, std::false_type{});
    };
    const auto by_norm = [&](auto bf16, auto half) {
        return r->q_weight || r->k_weight ? by_still(bf16, half, std::true_type{}) : by_still(bf16, half, std::false_type{});
    };
    const auto by_half = [&](auto bf16) { return r->half_split ? by_norm(bf16, std::true_type{}) : by_norm(bf16, std::false_type{}); };
    return dtype == OVC_BF16 ? by_half(std::true_type{}) : by_half(std::false_type{});
}

bool bad_shape(int dtype, int64_t B, int64_t S, int64_t Hq, int64_t Hk) {
    return (dtype != OVC_F16 && dtype != OVC_BF16) || B < 1 || S < 1 || Hq < 1 || Hk < 1 || Hq > 65535 || Hk > 65535 ||
           B > 0x7FFFFFFFLL || S > (1LL << 30) || B * S > 0x7FFFFFFFLL;
}

}  // namespace
}  // namespace ovc

using namespace ovc;

namespace {

int launch_rotary(const RotaryArgs& a, int dtype, const ovc_rotary* rotary, void* stream) {
    // A unit has up to four groups of eight heads, fewer where that would leave SMs without a few warps each.
    const int64_t groups = ceil_div(a.src[0].heads, kGroupRows) + ceil_div(a.src[1].heads, kGroupRows), share = a.tokens * groups / (8 * 148);
    int64_t unit_groups = share > kUnitGroups ? kUnitGroups : share < 1 ? 1 : share;
    const int64_t units = ceil_div(groups, unit_groups);
    unit_groups = ceil_div(groups, units);
    const dim3 grid(static_cast<unsigned>(ceil_div(a.tokens, kUnitWarps)), static_cast<unsigned>(units));
    const size_t smem = static_cast<size_t>(kUnitWarps * unit_groups * kGroupRows * 256);
    auto s = static_cast<cudaStream_t>(stream);
    return by_variant(dtype, rotary, a.angles, [&](auto bf16, auto half, auto norm, auto still) {
        rotary_kernel<bf16.value ? OVC_BF16 : OVC_F16, half.value, norm.value, still.value>
            <<<grid, 32 * kUnitWarps, smem, s>>>(a, static_cast<int>(unit_groups));
        return check_launch();
    });
}

}  // namespace

extern "C" int ovc_rotary_qk(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype, int64_t B,
                             int64_t S, int64_t Hq, int64_t Hk, const ovc_rotary* rotary, void* q_out, void* k_out, void* stream) {
    RotaryArgs a{};
    if (bad_shape(dtype, B, S, Hq, Hk) || !take_angles(rotary, &a.angles) ||
        !take_source(q, q_out, rotary->q_weight, q_strides, Hq, 15, &a.src[0]) ||
        !take_source(k, k_out, rotary->k_weight, k_strides, Hk, 15, &a.src[1]))
        return OVC_ERR_ARGUMENT;
    a.S = S, a.tokens = B * S;
    return launch_rotary(a, dtype, rotary, stream);
}

namespace {

int launch_rotary_quant(const void* q, const void* k, int dtype, int64_t B, int64_t S, int64_t H, const ovc_rotary* rotary, void* q8,
                        void* k8, float* q_descale, int64_t q_stride, float* k_descale, int64_t k_stride, float* amax_init, int32_t* bounds,
                        void* stream) {
    const int64_t blocks = ceil_div(S, kTile);
    const int64_t strides[3] = {S * H * kDim, H * kDim, kDim};
    RotaryArgs a{};
    if (bad_shape(dtype, B, S, H, H) || B > 32767 || !q_descale || !k_descale || q_stride < blocks || k_stride < blocks || !take_angles(rotary, &a.angles) ||
        !take_source(q, q8, rotary->q_weight, strides, H, 7, &a.src[0]) || !take_source(k, k8, rotary->k_weight, strides, H, 7, &a.src[1]))
        return OVC_ERR_ARGUMENT;
    a.S = S, a.tokens = B * S, a.amax_init = amax_init, a.bounds = bounds;
    a.src[0].descale = q_descale, a.src[0].descale_stride = q_stride;
    a.src[1].descale = k_descale, a.src[1].descale_stride = k_stride;
    // Two CTAs run per SM.  Heads per CTA: the count whose rounds of CTAs, each of its heads and the block's angles (which
    // cost about as much as two heads), are the shortest in all.
    const int rows = static_cast<int>(2 * H);
    // (With hundreds of heads the angles are shared by many, so the grid's second index stays far below its limit.)
    int per_cta = 1;
    int64_t best = 0;
    for (int n = 1; n <= rows; ++n) {
        const int64_t cost = ceil_div(blocks * B * ceil_div(rows, n), 2 * 148) * (n + 2);
        if (n == 1 || cost <= best) best = cost, per_cta = n;
    }
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(ceil_div(rows, per_cta)), static_cast<unsigned>(B));
    constexpr int smem = kTile * kPairs * static_cast<int>(sizeof(float2)) + kTile * kDim * 2;
    auto s = static_cast<cudaStream_t>(stream);
    const auto launch = [&](auto bf16, auto half, auto norm, auto still) {
        const auto kernel = rotary_quant_kernel<bf16.value ? OVC_BF16 : OVC_F16, half.value, norm.value, still.value>;
        static std::atomic<unsigned long long> ready;  // devices on which the kernel may take that much
        int device = 0;
        cudaError_t err = cudaGetDevice(&device);
        if (err == cudaSuccess && (device >= 64 || !(ready.load(std::memory_order_acquire) >> device & 1))) {
            err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (err == cudaSuccess && device < 64) ready.fetch_or(1ull << device, std::memory_order_release);
        }
        if (err != cudaSuccess) { set_last_cuda_error(err); return static_cast<int>(OVC_ERR_CUDA); }
        kernel<<<grid, kQuantThreads, smem, s>>>(a, static_cast<int>(blocks), per_cta);
        return check_launch();
    };
    return by_variant(dtype, rotary, a.angles, launch);
}

}  // namespace

extern "C" int ovc_prepare_rotary(const void* q, const void* k, const void* v, int dtype, int64_t B, int64_t S, int64_t H,
                                  const ovc_rotary* rotary, void* q8, void* k8, void* v8, float* q_descale, float* k_descale,
                                  float* v_descale, float* amax_ws, int32_t* cu_seqlens, void* stream) {
    if (!v || !v8 || !v_descale || !amax_ws || !aligned16(v) || (reinterpret_cast<uintptr_t>(v8) & 7u) || (cu_seqlens && B != 1))
        return OVC_ERR_ARGUMENT;
    const int64_t blocks = ceil_div(S, kTile);
    const int rc = launch_rotary_quant(q, k, dtype, B, S, H, rotary, q8, k8, q_descale, blocks, k_descale, blocks, amax_ws, cu_seqlens, stream);
    return rc != OVC_OK ? rc : launch_amax_cast_v(v, dtype, B, S, H, amax_ws, v8, v_descale, stream);
}

extern "C" int ovc_prepare_fused_rotary(const void* q, const void* k, const void* v, int dtype, int64_t S, int64_t H, const ovc_rotary* rotary,
                                        void* q8, void* k8, void* v_packed, float* q_descale, float* k_descale, float* v_descale,
                                        float* amax_ws, int32_t* cu_seqlens, void* stream) {
    if (!v || !v_packed || !v_descale || !amax_ws || !aligned16(v) || !aligned16(v_packed)) return OVC_ERR_ARGUMENT;
    const int64_t blocks = ceil_div(S, kTile);
    const int rc = launch_rotary_quant(q, k, dtype, 1, S, H, rotary, q8, k8, q_descale, (blocks + 1) / 2 * 2, k_descale, blocks, amax_ws,
                                       cu_seqlens, stream);
    return rc != OVC_OK ? rc : launch_amax_cast_pack_v(v, dtype, S, H, amax_ws, v_packed, v_descale, stream);
}
