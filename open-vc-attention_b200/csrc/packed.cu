// Attention over packed sequences of different lengths in 16 bits: grouped query heads, optional causal mask, keys split
// over CTAs where there are few query rows.  TMA -> shared memory -> tcgen05 (kind::f16) with accumulators in tensor
// memory; the softmax on the CUDA cores in float32, in one pass over the keys with a running maximum and sum.
//
// A row of the score tile is one query head of one token: the G query heads of a key head are packed behind each other
// (row = token * G + head in group), 128 / G tokens to a tile of 128 rows, so that a key tile is read once for all of them.
//
// A CTA runs two softmax stages of 128 rows each (one row per thread).
//   Whole: a CTA is two neighbouring tiles of rows with all their keys; both stages visit every key tile.
//   Split, where that would leave SMs without work: the key tiles of all row tiles of all key heads are one list that is
//   cut into equal shares, one to a CTA.  A share is one or a few segments (key tiles of one row tile), which the CTA
//   works off one after another; it writes unnormalised partial results that combine_kernel joins.  Wide split has the
//   stages of the whole form; narrow split (at most one tile of rows per sequence) gives both stages the same rows and every
//   other key tile, since with one tile of rows the time goes into reading keys.
//
// Warp roles (384 threads): warps 0-3 / 4-7 softmax of stage 0 / 1, warp 8 TMA loads, warp 9 the products, warps 10 and 11
// clear the CTA's share of the rows behind the last sequence, where asked to.  Warp 8 also clears the rows of a value tile
// behind the end of its sequence (another sequence's values may be infinite or NaN, and 0 times those is NaN).
//
// Tensor memory (512 columns): S0 0..127, S1 128..255, O0 256..383, O1 384..511.  The probabilities of a stage overwrite the
// first 64 columns of its scores: there is room for nothing else.  The SM's one tensor pipe runs the products of the issuing
// thread in the order of their issue, so S(n+1), issued behind O += P(n) V(n), cannot overtake the reads of P(n), and a
// stage that sees S(n+1) knows O to be complete up to n.
//
// Shared memory: Q 2 x 32 KB, a ring of five 32 KB tiles that holds K and V alternately.
//
// What bounds it.  Whole: a step (both stages, one key tile) is 2048 cycles of tensor pipe and as many of exponentials (128 x
// 128 x 2 at 16 a cycle); it takes about 3300.  A stage's step is a chain - scores read and their maximum found (350 cycles),
// two halves of exponentials (512 each and what the other stage takes of the unit), P V, Q K^T of the next tile (1120), a
// few hand-overs of 100 to 200 - and the two stages' chains interleave.  [32768, 8, 128]: 3.74 ms in a row (1.18 PFLOP/s at the
// power limit, where the library's matrix product reaches 1.4), 3.34 ms alone.  Tried on it, each right and slower: a warp
// for the products of each stage (they drift into step: 1.25 times the time), two threads to a row (1.13), part of the
// exponentials as polynomials on the FMA pipe (1.05 for an eighth to 1.3 for half: a pair costs 25 cycles of issue there and
// 16 on the special-function unit), the exponentials started with the maximum of the tile before (1.04), a relay that
// tells the issuing warp of landed tiles (1.03), CTAs that stay and take one row tile after another (1.03).
// Split, narrow: the rate at which keys are read; 81 us of kernel for 487 MB (6.0 TB/s), 7.2 TB/s once under way.
// The split forms spill 11 registers of the launch's 168 (44 bytes stored, 64 loaded), the whole form none.

#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "scores.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.cuh"

namespace ovc {
namespace {

using namespace ptx;

constexpr int kThreads = 384;
constexpr int kSlots = 5;
constexpr int kHalfBytes = kTile * 128;       // 128 rows of 64 values
constexpr int kTileBytes = 2 * kHalfBytes;    // 128 rows of 128 values, as two halves of the channels
constexpr uint32_t kColS = 0, kColO = 256, kTmemCols = 512;
constexpr int kMaxTiles = 160;                // row tiles of a key head that a split launch can plan (shared memory)

enum Mode { kWhole = 0, kSplitWide = 1, kSplitNarrow = 2 };

// The row tiles of a key head (all key heads have the same), made alike by every warp that asks, and what each costs: a unit
// for each of its key tiles and segment_cost more.  start[t] is the sum before tile t, start[count] of all.
struct PlanTiles {
    int count;
    int seq[kMaxTiles], token0[kMaxTiles], start[kMaxTiles + 1];
};

struct PackedParams {
    const int* cu_q;       // [B+1]
    const int* cu_k;       // [B+1]
    void* out;             // [Tq,Hq,128]
    float* lse;            // [Hq,Tq] or null
    PlanTiles* plan;       // split: for combine_kernel
    float* part_o;         // split: [segments * 2][slot_rows][128], unnormalised
    float2* part_ml;       // split: [segments * 2][slot_rows], (maximum in units of log2, sum)
    uint32_t* status;      // [1]: sticky word, or null
    volatile uint32_t* host_status;
    int B, Hq, Hk, G;
    int tokens;            // tokens of a tile of 128 rows: 128 / G
    int Tq, Tk;
    int ctas;              // split: shares
    int segment_cost;      // split: what it costs to begin and end a segment, in key tiles
    int max_tiles;         // split: row tiles of a key head that the workspace has room for
    int slot_rows;
    int heads_first;       // whole: the grid is (key heads, row tiles), not (row tiles, key heads)
    int zero_tail;         // rows behind the last sequence are set to zero
    float scale_log2;
};

// What a CTA works on: rows of one sequence, a key head and a range of the sequence's key tiles.
struct Item {
    int valid;             // 0: nothing
    int segment;           // split: where its partial results go
    int kv_head;
    int q0, lq, k0, lk;    // the sequence
    int token0;            // first token of the tile within the sequence
    int t0, t1;            // key tiles
    int units;             // split: how far it is along the list
};

__device__ __forceinline__ void bounds(const int* cu, int b, int total, int* start, int* length) {
    const int lo = max(0, min(cu[b], total));
    *start = lo;
    *length = max(lo, min(cu[b + 1], total)) - lo;
}

// Key tiles that tokens [token0, token0 + n) of a sequence see.  Causal: the last token sees every key, token t the keys
// below t + 1 + lk - lq.
template <bool kCausal>
__device__ __forceinline__ int visible_tiles(int lq, int lk, int token0, int n) {
    int keys = lk;
    if (kCausal) keys = max(0, min(lk, lk - lq + min(token0 + n, lq)));
    return (keys + kTile - 1) / kTile;
}

__device__ __forceinline__ int warp_sum_before(int x, int lane, int* all) {
    int s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= o) s += y;
    }
    *all = __shfl_sync(0xFFFFFFFFu, s, 31);
    return s - x;
}

// Row tile `which` of the launch (one warp).  Within a sequence the last tokens come first: under a causal mask theirs are
// the longest, and the short ones fill the SMs at the end.
template <bool kCausal>
__device__ void find_tile(const PackedParams& p, int per_tile, int which, int lane, Item* item) {
    constexpr int kEach = 4;  // sequences of a lane at a time: their bounds are loaded together
    int before = 0;
    bool found = false;
    for (int base = 0; base < p.B && !found; base += 32 * kEach) {
        const int b0 = base + kEach * lane;
        int q0[kEach], lq[kEach], n = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            q0[i] = lq[i] = 0;
            if (b0 + i < p.B) bounds(p.cu_q, b0 + i, p.Tq, &q0[i], &lq[i]);
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) n += (lq[i] + per_tile - 1) / per_tile;
        int all, at = before + warp_sum_before(n, lane, &all);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int mine = (lq[i] + per_tile - 1) / per_tile;
            if (which >= at && which < at + mine) {
                item->q0 = q0[i], item->lq = lq[i];
                bounds(p.cu_k, b0 + i, p.Tk, &item->k0, &item->lk);
                item->token0 = (mine - 1 - (which - at)) * per_tile;
                item->t0 = 0;
                item->t1 = visible_tiles<kCausal>(lq[i], item->lk, item->token0, per_tile);
            }
            at += mine;
        }
        found = which < before + all;
        before += all;
    }
    if (lane == 0) item->valid = found;
    __syncwarp();
}

__device__ __forceinline__ int tile_cost(const PackedParams& p, int key_tiles) { return key_tiles > 0 ? key_tiles + p.segment_cost : 0; }
template <bool kCausal>
__device__ void plan_tiles(const PackedParams& p, int per_tile, int lane, PlanTiles* plan) {
    int tiles = 0, total = 0;
    for (int base = 0; base < p.B; base += 32) {
        const int b = base + lane;
        int q0, lq = 0, k0, lk = 0;
        if (b < p.B) {
            bounds(p.cu_q, b, p.Tq, &q0, &lq);
            bounds(p.cu_k, b, p.Tk, &k0, &lk);
        }
        // (More tiles than there is room for come of bounds that are out of order only.)
        int all, all_costs, n = min((lq + per_tile - 1) / per_tile, kMaxTiles);
        const int at = tiles + warp_sum_before(n, lane, &all);
        n = max(0, min(n, p.max_tiles - at));
        int cost = 0;
        for (int i = 0; i < n; ++i) cost += tile_cost(p, visible_tiles<kCausal>(lq, lk, i * per_tile, per_tile));
        int start = total + warp_sum_before(cost, lane, &all_costs);
        for (int i = 0; i < n; ++i) {
            plan->seq[at + i] = b, plan->token0[at + i] = i * per_tile, plan->start[at + i] = start;
            start += tile_cost(p, visible_tiles<kCausal>(lq, lk, i * per_tile, per_tile));
        }
        tiles = min(tiles + all, p.max_tiles);
        total += all_costs;
    }
    if (lane == 0) plan->count = tiles, plan->start[tiles] = total;
    __syncwarp();
}
// The list of all units (key head by key head) is cut into `shares` pieces, share c from (c * total) / shares.
struct Shares {
    long long total;
    int shares;
    __device__ Shares(const PlanTiles& plan, const PackedParams& p) {
        total = static_cast<long long>(plan.start[plan.count]) * p.Hk;
        shares = static_cast<int>(max(1LL, min(static_cast<long long>(p.ctas), total / (2 + p.segment_cost))));  // of two tiles at least
    }
    __device__ long long first(int c) const { return c >= shares ? total : c * total / shares; }
    __device__ int owner(long long at) const { return static_cast<int>(((at + 1) * shares + total - 1) / total) - 1; }
};
// The first segment of share c from `at` of the list on.  Of a row tile's units the first segment_cost are no key tiles: a
// piece of those alone is no segment.  Segments are counted by the shares and the row tiles before them (each begins
// either).
__device__ void find_segment(const PackedParams& p, const PlanTiles& plan, const Shares& shares, int c, long long at, int lane, Item* item) {
    const int per_head = plan.start[plan.count];
    const long long end = shares.first(c + 1);
    long long pos = at;
    bool found = false;
    while (pos < end && !found) {
        const int kv_head = static_cast<int>(pos / per_head), r = static_cast<int>(pos - static_cast<long long>(kv_head) * per_head);
        int units = 0;
        for (int t = lane; t < plan.count; t += 32) {
            if (r < plan.start[t] || r >= plan.start[t + 1]) continue;
            units = static_cast<int>(min(static_cast<long long>(plan.start[t + 1] - r), end - pos));
            const int from = r - plan.start[t] - p.segment_cost, t0 = max(0, from), t1 = max(0, from + units);
            if (t1 <= t0) continue;
            found = true;
            item->kv_head = kv_head, item->segment = c + kv_head * plan.count + t;
            bounds(p.cu_q, plan.seq[t], p.Tq, &item->q0, &item->lq);
            bounds(p.cu_k, plan.seq[t], p.Tk, &item->k0, &item->lk);
            item->token0 = plan.token0[t], item->t0 = t0, item->t1 = t1;
        }
        found = __any_sync(0xFFFFFFFFu, found);
        pos += static_cast<int>(__reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned>(units)));
    }
    if (lane == 0) item->valid = found, item->units = static_cast<int>(pos - at);
    __syncwarp();
}

// Rows behind the last sequence, every `stride`th from the `first`th: zero, -inf.
__device__ __forceinline__ void clear_tail(const PackedParams& p, int first, int stride, int thread, int threads) {
    const int q_end = max(0, min(p.cu_q[p.B], p.Tq));
    for (long long t = q_end + static_cast<long long>(first); t < p.Tq; t += stride) {
        uint4* dst = reinterpret_cast<uint4*>(p.out) + t * p.Hq * 16;
        for (int i = thread; i < p.Hq * 16; i += threads) dst[i] = make_uint4(0, 0, 0, 0);
        for (int h = thread; p.lse != nullptr && h < p.Hq; h += threads) p.lse[static_cast<long long>(h) * p.Tq + t] = -INFINITY;
    }
}

// ---- operands ----------------------------------------------------------------------------------------------------

template <bool kBf16>
__host__ __device__ constexpr uint32_t idesc(bool b_mn_major) {
    return (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(kTile >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}

// The products are issued by one elected lane while the whole warp executes the (convergent) code, so that descriptors and
// addresses are warp-uniform values and need no moves between the products.
// S = Q K^T: both operands K-major, 64 channels to a half; eight steps of 16 channels (32 bytes).
__device__ __forceinline__ void product_qk(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t id) {
#define OVC_QK_STEP(offset, accumulate)                                                                  \
    "add.u32 al, %1, " #offset ";\n\tadd.u32 bl, %2, " #offset ";\n\tmov.b64 da, {al, %3};\n\tmov.b64 db, {bl, %3};\n\t" \
    "@leader tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, " #accumulate ";\n\t"
    static_assert((kHalfBytes >> 4) == 1024, "the second half's offset is written out below");
    asm volatile(
        "{\n\t.reg .pred leader;\n\t.reg .b64 da, db;\n\t.reg .b32 al, bl;\n\t"
        "elect.sync _|leader, 0xFFFFFFFF;\n\t"
        OVC_QK_STEP(0, 0) OVC_QK_STEP(2, 1) OVC_QK_STEP(4, 1) OVC_QK_STEP(6, 1)
        OVC_QK_STEP(1024, 1) OVC_QK_STEP(1026, 1) OVC_QK_STEP(1028, 1) OVC_QK_STEP(1030, 1) "}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(kSmemDescHi), "r"(id)
        : "memory");
#undef OVC_QK_STEP
}
// O (+)= P V: P in tensor memory (two values per column), V as the MN-major operand (a row of shared memory is a key);
// four steps of 16 keys, a half of a tile.
__device__ __forceinline__ void product_pv(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t id, uint32_t accumulate_first) {
#define OVC_PV_STEP(a_offset, b_offset, accumulate)                                                      \
    "add.u32 ta, %1, " #a_offset ";\n\tadd.u32 bl, %2, " #b_offset ";\n\tmov.b64 db, {bl, %3};\n\t"      \
    "@leader tcgen05.mma.cta_group::1.kind::f16 [%0], [ta], db, %4, " accumulate ";\n\t"
    asm volatile(
        "{\n\t.reg .pred leader, p;\n\t.reg .b64 db;\n\t.reg .b32 ta, bl;\n\t"
        "elect.sync _|leader, 0xFFFFFFFF;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        OVC_PV_STEP(0, 0, "p") OVC_PV_STEP(8, 128, "1") OVC_PV_STEP(16, 256, "1") OVC_PV_STEP(24, 384, "1") "}"
        ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(kSmemDescHi), "r"(id), "r"(accumulate_first)
        : "memory");
#undef OVC_PV_STEP
}

template <bool kBf16>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
    uint32_t r;
    if (kBf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float* a, float* b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(v));
}

// Row maximum that is not a number where a score is not.
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max128_nan(const uint32_t (&s)[128]) {
    const auto v = [&](int i) { return __uint_as_float(s[i]); };
    float m[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float a[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = fmax3_nan(v(32 * c + i), v(32 * c + 8 + i), v(32 * c + 16 + i));
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = fmax3_nan(a[i], a[i + 4], v(32 * c + 24 + i));
#pragma unroll
        for (int i = 0; i < 2; ++i) a[i] = fmax3_nan(a[i], a[i + 2], v(32 * c + 28 + i));
        m[c] = fmax3_nan(a[0], a[1], fmax3_nan(v(32 * c + 30), v(32 * c + 31), v(32 * c + 31)));
    }
    return fmax3_nan(fmax3_nan(m[0], m[1], m[2]), m[3], m[3]);
}

// Four lanes that hold four 16-byte pieces each of rows of their own exchange them: lane r of the four gets piece r of
// every row, so that a store covers 64 bytes of eight rows and not 16 bytes of thirty-two, which the store unit works
// through one by one (5500 cycles for the output of an item; prompts of 5000 to 1 tokens 354 -> 348 us).
__device__ __forceinline__ void exchange4(uint4 (&u)[4], int lane) {
    const auto swap = [](uint4& keep_low, uint4& keep_high, bool high, int mask) {
        uint4 give = high ? keep_low : keep_high;
        give.x = __shfl_xor_sync(0xFFFFFFFFu, give.x, mask), give.y = __shfl_xor_sync(0xFFFFFFFFu, give.y, mask);
        give.z = __shfl_xor_sync(0xFFFFFFFFu, give.z, mask), give.w = __shfl_xor_sync(0xFFFFFFFFu, give.w, mask);
        if (high) keep_low = give;
        else keep_high = give;
    };
    swap(u[0], u[1], lane & 1, 1), swap(u[2], u[3], lane & 1, 1);
    swap(u[0], u[2], lane & 2, 2), swap(u[1], u[3], lane & 2, 2);
}

struct Smem {
    alignas(1024) uint8_t q[2][kTileBytes];
    alignas(1024) uint8_t ring[kSlots][kTileBytes];
    alignas(8) uint64_t q_full[2];
    uint64_t full[kSlots], empty[kSlots];  // a tile has landed / its last reader is done
    uint64_t s_full[2];                    // the stage's scores are in tensor memory
    uint64_t p_full[2][2];                 // the stage's probabilities of the first, second 64 keys are, and O is rescaled
    uint64_t o_full[2];
    uint64_t v_clean;                      // the rows behind the sequence's end are cleared in its last value tile
    uint64_t drain;
    uint32_t tmem_base, gave_up;
    volatile uint32_t abort_flag;
    Item item;
    PlanTiles plan;
};

// The order in which a CTA visits key tiles.  Whole, wide: both stages every tile.  Narrow: stage s the tiles s, s + 2, ...
// A tile is slot indices 2 i (K) and 2 i + 1 (V) of the ring, i counting the segment's tiles.
template <int kMode>
__device__ __forceinline__ int tile_of(int stage, int n) {
    return kMode == kSplitNarrow ? 2 * n + stage : n;
}

// Steps of a stage.
template <bool kCausal, int kMode>
__device__ __forceinline__ int steps_of(const PackedParams& p, const Item& it, int stage) {
    if (kMode == kSplitNarrow) return (it.t1 - it.t0 - stage + 1) / 2;
    const int token = it.token0 + stage * p.tokens;
    return token >= it.lq ? 0 : max(0, min(it.t1, visible_tiles<kCausal>(it.lq, it.lk, token, p.tokens)) - it.t0);
}
// Rows of the last value tile that belong to the sequence, where that is the sequence's last tile and not full; else 0.
__device__ __forceinline__ int rows_to_keep(const Item& it) {
    return it.t1 == (it.lk + kTile - 1) / kTile ? it.lk % kTile : 0;
}

template <bool kBf16, bool kCausal, int kMode>
__global__ void __launch_bounds__(kThreads, 1)
packed_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
              const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PackedParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];  // the kernel's only shared memory, so at the start of it
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    constexpr bool kSplit = kMode != kWhole, kNarrow = kMode == kSplitNarrow;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_cta = (kNarrow ? 1 : 2) * p.tokens;  // tokens of a row tile
    const float nan = __int_as_float(0x7FC00000);
    const Item& item = sm.item;

    if (warp == 0) {
        // A barrier wait expired since the host last looked: start nothing, leave NaN, and report this launch as well (the
        // host may have taken note of the earlier one on another stream, and clears the word on its own).  (Nor could
        // anything be computed were the tiles not on the 1024-byte grid of their swizzle.)
        if (lane == 0) {
            const uint32_t expired = p.status != nullptr ? *reinterpret_cast<volatile uint32_t*>(p.status) : 0u;
            // (The end of the kernel makes it visible; a fence here, though never reached, takes 1.5 % of a long launch.)
            if (expired != 0 && p.host_status != nullptr) *p.host_status = OVC_STATUS_WAIT_EXPIRED;
            sm.gave_up = expired | (smem_addr(smem_raw) & 1023u);
            sm.abort_flag = 0;
        }
        if (kSplit) plan_tiles<kCausal>(p, per_cta, lane, &sm.plan);
    }
    if (warp == 9) {
        tmem_alloc(smem_addr(&sm.tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    const bool live = sm.gave_up == 0;

    const auto wait = [&](uint64_t* bar, uint32_t parity) {
        return wait_bounded(&sm.abort_flag, bar, parity, kWaitCycles, [&] {
            sm.abort_flag = 1;
            if (p.status != nullptr) atomicOr(p.status, OVC_STATUS_WAIT_EXPIRED);
            if (p.host_status != nullptr) {
                *p.host_status = OVC_STATUS_WAIT_EXPIRED;
                __threadfence_system();
            }
        });
    };
    if (kSplit && blockIdx.x == 0 && warp == 10) {
        const int* from = reinterpret_cast<const int*>(&sm.plan);
        for (int i = lane; i < static_cast<int>(sizeof(PlanTiles) / sizeof(int)); i += 32) reinterpret_cast<int*>(p.plan)[i] = from[i];
    }
    // Where this CTA is in the list of key tiles (split), or whether its only item is still to come.
    long long at = 0, end = 1, first_at = 0;
    if (kSplit) {
        const Shares shares(sm.plan, p);
        at = first_at = shares.first(blockIdx.x), end = shares.first(blockIdx.x + 1);
    }
    // The next segment, for the whole CTA: false behind the last.  All products and copies of the one before are done, and what
    // the softmax warps read of its accumulators comes before the next one's products.
    const auto next_segment = [&]() {
        if (at >= end) return false;
        if (kSplit) tc_fence_before();
        __syncwarp();
        asm volatile("bar.sync 0;" ::: "memory");
        if (warp == 0) {
            if (kSplit) {
                find_segment(p, sm.plan, Shares(sm.plan, p), blockIdx.x, at, lane, &sm.item);
            } else {
                find_tile<kCausal>(p, per_cta, p.heads_first ? blockIdx.y : blockIdx.x, lane, &sm.item);
                if (lane == 0) sm.item.kv_head = p.heads_first ? blockIdx.x : blockIdx.y;
            }
        }
        if (threadIdx.x == 32) {
            for (uint64_t* bar = sm.q_full; bar <= &sm.drain; ++bar) {
                if (kSplit && at != first_at) mbar_inval(smem_addr(bar));
                const bool by_stage = bar >= sm.p_full[0] && bar < sm.o_full;
                mbar_init(smem_addr(bar), by_stage ? 128 : 1);
            }
            mbar_init_fence();
        }
        fence_proxy_async_smem();
        __syncwarp();
        asm volatile("bar.sync 0;" ::: "memory");
        if (kSplit) tc_fence_after();
        at += kSplit ? item.units : 1;
        return item.valid != 0;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        while (next_segment()) {
            const int n_tiles = item.t1 - item.t0, kv_head = item.kv_head, group0 = kv_head * p.G, tail_rows = rows_to_keep(item);
            const int steps[2] = {steps_of<kCausal, kMode>(p, item, 0), steps_of<kCausal, kMode>(p, item, 1)};
            const bool cleans = tail_rows > 0, run = live && sm.abort_flag == 0 && n_tiles > 0;
            if (warp == 8 && run) {
                // ---------------- TMA loads ----------------
                const int q_tiles = kMode == kSplitNarrow ? 1 : 2;
                int issued = 0;
                if (lane == 0) {
                    tma_prefetch_desc(&tmap_k);
                    tma_prefetch_desc(&tmap_v);
                    const uint64_t keep = policy_evict_last(), stream = policy_evict_first();
                    const uint64_t kv_policy = kMode == kSplitNarrow ? stream : keep;
                    const uint32_t q_bytes = static_cast<uint32_t>(p.tokens * p.G) * 128;  // of one half
                    for (int s = 0; s < q_tiles; ++s) {
                        mbar_expect_tx(smem_addr(&sm.q_full[s]), 2 * q_bytes);
                        const int token = item.q0 + item.token0 + s * p.tokens;
                        for (int h = 0; h < 2; ++h)
                            tma_load_4d(smem_addr(sm.q[s]) + h * kHalfBytes, &tmap_q, smem_addr(&sm.q_full[s]), 0, group0, token, h, stream);
                    }
                    for (int i = 0; i < 2 * n_tiles; ++i) {
                        const int slot = i % kSlots;
                        if (i >= kSlots && !wait(&sm.empty[slot], (i / kSlots - 1) & 1)) break;
                        mbar_expect_tx(smem_addr(&sm.full[slot]), kTileBytes);
                        const int key = item.k0 + (item.t0 + (i >> 1)) * kTile;
                        tma_load_4d(smem_addr(sm.ring[slot]), (i & 1) ? &tmap_v : &tmap_k, smem_addr(&sm.full[slot]), 0, kv_head, key, 0, kv_policy);
                        issued = i + 1;
                    }
                }
                issued = __shfl_sync(0xFFFFFFFFu, issued, 0);
                // The last value tile: its rows behind the end of the sequence.  (The warp that issued the load may wait for
                // it: its slot's earlier phases are over, so the parity is unambiguous.)
                const int index = 2 * n_tiles - 1;
                if (cleans && issued == 2 * n_tiles && __all_sync(0xFFFFFFFFu, wait(&sm.full[index % kSlots], (index / kSlots) & 1))) {
                    for (int h = 0; h < 2; ++h) {
                        uint4* rows = reinterpret_cast<uint4*>(sm.ring[index % kSlots] + h * kHalfBytes);
                        for (int i = tail_rows * 8 + lane; i < kTile * 8; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_addr(&sm.v_clean));
                }
                // Every copy has landed before the CTA's shared memory goes away (it has, unless a wait expired).
                if (lane == 0) {
                    const long long t0 = clock64();
                    for (int i = max(0, issued - kSlots); i < issued; ++i)
                        while (!mbar_try_wait(smem_addr(&sm.full[i % kSlots]), (i / kSlots) & 1) && clock64() - t0 < kWaitCycles) {}
                    for (int s = 0; s < q_tiles; ++s)
                        while (!mbar_try_wait(smem_addr(&sm.q_full[s]), 0) && clock64() - t0 < kWaitCycles) {}
                }
            } else if (warp == 9 && run) {
                // ---------------- products ----------------
                // One warp issues for both stages, in a fixed order, which keeps them half a step apart (with a warp for each
                // stage they drift into step: 1.25 times the time).  The issuing lane is held until all but the last
                // products have run, so what lies between two issues is kept short: slots and descriptors are carried along,
                // the copies are waited for by the first stage that needs them (in the narrow form, where keys are what is
                // waited for, K of the next step only once V's slot is on its way back).
                constexpr uint32_t id_qk = idesc<kBf16>(false), id_pv = idesc<kBf16>(true);
                const auto uniform = [](int x) { return static_cast<int>(__reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned>(x))); };
                const int steps0 = uniform(steps[0]), steps1 = uniform(steps[1]), dirty = uniform(cleans ? n_tiles : 0) - 1;
                const uint32_t tm = static_cast<uint32_t>(uniform(static_cast<int>(tmem)));
                const auto all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, wait(bar, parity)) != 0; };
                struct Slot {
                    int i = 0;
                    uint32_t phase = 0;
                    __device__ __forceinline__ void advance() { if (++i == kSlots) i = 0, phase ^= 1; }
                };
                const uint32_t ring_lo = smem_desc_lo(smem_addr(sm.ring[0])), q_lo = smem_desc_lo(smem_addr(sm.q[0]));
                const uint32_t ring_lo_mn = smem_desc_lo_bmn(smem_addr(sm.ring[0]), kHalfBytes);
                const auto scores = [&](int s, const Slot& k, bool last_reader) {
                    product_qk(tm + kColS + 128 * s, q_lo + (kMode == kSplitNarrow ? 0 : s * (kTileBytes >> 4)), ring_lo + k.i * (kTileBytes >> 4), id_qk);
                    mma_commit_elect(smem_addr(&sm.s_full[s]));
                    if (last_reader) mma_commit_elect(smem_addr(&sm.empty[k.i]));
                };
                // Slots of K of a stage's next step and V of its present one.
                Slot k, v;
                v.advance();
                bool ok = true;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (ok && (s ? steps1 : steps0) > 0) {
                        ok = all(&sm.q_full[kMode == kSplitNarrow ? 0 : s], 0) && all(&sm.full[k.i], k.phase);
                        if (ok) scores(s, k, kMode == kSplitNarrow || s == 1 || steps1 == 0);
                    }
                    if (kMode == kSplitNarrow || s == 1) k.advance(), k.advance();
                }
                const int most = max(steps0, steps1);
                for (int n = 0; ok && n < most; ++n) {
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int mine = s ? steps1 : steps0;
                        if (n < mine) {
                            const uint32_t t_o = tm + kColO + 128 * s, t_p = tm + kColS + 128 * s, v_lo = ring_lo_mn + v.i * (kTileBytes >> 4);
                            const bool first = kMode == kSplitNarrow || s == 0 || n >= steps0, last = kMode == kSplitNarrow || s == 1 || n >= steps1;
                            const bool more = n + 1 < mine;
                            if (first) {
                                ok = all(&sm.full[v.i], v.phase) && (tile_of<kMode>(s, n) != dirty || all(&sm.v_clean, 0));
                                if (kMode != kSplitNarrow && more) ok = ok && all(&sm.full[k.i], k.phase);
                            } else if (more && n + 1 >= steps0) {
                                ok = all(&sm.full[k.i], k.phase);
                            }
                            // The first half of the keys is multiplied while the stage still works on the second.
                            ok = ok && all(&sm.p_full[s][0], n & 1);
                            if (!ok) break;
                            tc_fence_after();
                            product_pv(t_o, t_p, v_lo, id_pv, n > 0);
                            ok = all(&sm.p_full[s][1], n & 1);
                            if (!ok) break;
                            tc_fence_after();
                            product_pv(t_o, t_p + 32, v_lo + 512, id_pv, 1);
                            if (last) mma_commit_elect(smem_addr(&sm.empty[v.i]));
                            if (kMode == kSplitNarrow && more) ok = all(&sm.full[k.i], k.phase);
                            if (!ok) break;
                            if (more) scores(s, k, kMode == kSplitNarrow || s == 1 || n + 1 >= steps1);
                            else mma_commit_elect(smem_addr(&sm.o_full[s]));
                        }
                        if (kMode == kSplitNarrow || s == 1) k.advance(), k.advance(), v.advance(), v.advance();
                    }
                }
                if (!ok) {  // products in flight end before tensor memory is released
                    mma_commit_elect(smem_addr(&sm.drain));
                    const long long t0 = clock64();
                    while (!mbar_try_wait(smem_addr(&sm.drain), 0) && clock64() - t0 < kWaitCycles) {}
                }
            }
        }
        if (warp >= 10 && !kSplit && p.zero_tail)
            clear_tail(p, blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y, threadIdx.x - 320, 64);
    } else {
        // ---------------- softmax: one row per thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int stage = warp >> 2;
        const int row = (warp & 3) * 32 + lane;
        while (next_segment()) {
            const int group0 = item.kv_head * p.G;
            const int token = item.token0 + (kMode == kSplitNarrow ? 0 : stage * p.tokens) + row / p.G;  // within the sequence
            const int head = group0 + row % p.G;
            const bool real = row < p.tokens * p.G && token < item.lq;
            const int keys = kCausal ? max(0, min(item.lk, item.lk - item.lq + token + 1)) : item.lk;
            const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const uint32_t t_s = lane_base + kColS + 128 * stage, t_o = lane_base + kColO + 128 * stage;
            const bool go = live && sm.abort_flag == 0;
            const int my_steps = go ? steps_of<kCausal, kMode>(p, item, stage) : 0;

            float top = -INFINITY;     // the maximum that the accumulator is scaled by
            // Probabilities of fp16 are 2^7 times as large, so that what its exponents cannot hold is below 2^-32 of the row's
            // largest (2^-25 without; with hundreds of thousands of small ones that would be per cents of the row).
            constexpr float kLift = kBf16 ? 0.0f : 7.0f;
            float shift = 0.0f;        // kLift - top * scale_log2, 0 while there is no maximum
            float limit = -INFINITY;   // a scaled score above it moves the maximum
            // Steps whose tile every row of the warp sees in full.
            const int whole_tiles = static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, static_cast<unsigned>(keys))) / kTile - item.t0;
            const int whole_steps = kMode == kSplitNarrow ? (whole_tiles - stage + 1) / 2 : whole_tiles;
            uint64_t sum2 = 0;         // the running sum, even and odd columns
            bool ok = true;
            for (int n = 0; n < my_steps; ++n) {
                ok = __all_sync(0xFFFFFFFFu, wait(&sm.s_full[stage], n & 1));
                if (!ok) break;
                tc_fence_after();
                uint32_t s[128];
                tmem_ld32(t_s, s);
                tmem_ld32(t_s + 32, s + 32);
                tmem_ld32(t_s + 64, s + 64);
                tmem_ld32(t_s + 96, s + 96);
                tmem_wait_ld();
                if (n >= whole_steps) {
                    const int columns = keys - (item.t0 + tile_of<kMode>(stage, n)) * kTile;
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c >= columns) s[c] = 0xFF800000u;  // -inf, whatever the key holds
                }
                // The maximum moves only when it grows by more than 2^8: until then probabilities above 1 are as exact as those
                // below, and neither the sums (float32) nor the 16-bit probabilities (up to 2^15) overflow.  The
                // comparison is false where both are -inf (no key yet) and true where a score is not a number.  Rows that are none
                // of the sequence's have no vote, whatever the query tile holds there (another sequence's rows, or what was in
                // shared memory, where G does not divide 128): NaN in them had the accumulator reloaded at every step (9 rows of
                // 20000 keys, 148 heads: 371 us beside NaN, 331 beside finite rows).
                const float tile_top = max128_nan(s);
                if (__any_sync(0xFFFFFFFFu, real && !(tile_top * p.scale_log2 <= limit) && tile_top != -INFINITY)) {
                    float alpha = 1.0f;
                    if (tile_top * p.scale_log2 > limit) {
                        const float moved = fmaf(-tile_top, p.scale_log2, kLift);
                        alpha = top == -INFINITY ? 0.0f : ex2(moved - shift);
                        top = tile_top;
                        shift = moved;
                        limit = 8.0f + kLift - shift;
                    }
                    if (tile_top != tile_top) alpha = nan;  // a score is not a number: neither is the row
                    float a, b;
                    unpack2(sum2, &a, &b);
                    sum2 = pack2(a * alpha, b * alpha);
                    if (n > 0) {
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            uint32_t o[32];
                            tmem_ld32(t_o + 32 * c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            tmem_st32(t_o + 32 * c, o);
                        }
                    }
                }
                const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), shift2 = pack2(shift, shift);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pr[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        uint32_t* pair = s + 32 * c + 2 * e;
                        uint64_t x = ffma2(pack_u2(pair[0], pair[1]), scale2, shift2);
                        float a, b;
                        unpack2(x, &a, &b);
                        a = ex2(a), b = ex2(b);
                        pair[0] = __float_as_uint(a), pair[1] = __float_as_uint(b);
                        pr[e] = narrow2<kBf16>(a, b);
                    }
                    tmem_st16(t_s + 16 * c, pr);
                    if (c & 1) {
                        tmem_wait_st();
                        tc_fence_before();
                        mbar_arrive(smem_addr(&sm.p_full[stage][c >> 1]));
                    }
                }
                // The sum adds the probabilities before their rounding to 16 bits (which is unbiased), behind the hand-over: a
                // tile's first, so that many small ones are not lost one by one beside a large sum.
                uint64_t part[4];
#pragma unroll
                for (int e = 0; e < 64; ++e) {
                    const uint64_t pair = pack_u2(s[2 * e], s[2 * e + 1]);
                    part[e & 3] = e < 4 ? pair : fadd2(part[e & 3], pair);
                }
                sum2 = fadd2(sum2, fadd2(fadd2(part[0], part[1]), fadd2(part[2], part[3])));
            }
            if (ok && my_steps > 0) ok = __all_sync(0xFFFFFFFFu, wait(&sm.o_full[stage], 0));
            tc_fence_after();
            ok = ok && go;
            float a, b;
            unpack2(sum2, &a, &b);
            const float sum = ok ? a + b : nan;
            if (kMode == kWhole) {
                const bool none = top == -INFINITY && sum == sum;  // no key is visible
                const float factor = 1.0f / sum;
                const long long at = static_cast<long long>(item.q0 + token) * p.Hq + head;
                if (real && p.lse != nullptr)
                    p.lse[static_cast<long long>(head) * p.Tq + item.q0 + token] =
                        none ? -INFINITY : (__log2f(sum) - shift) * 0.69314718055994531f;  // (NaN where a wait expired)
                // After the exchange a lane stores its piece of the four rows of its group.
                uint4* to[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    to[i] = reinterpret_cast<uint4*>(p.out) + __shfl_sync(0xFFFFFFFFu, real ? at : -1LL, (lane & ~3) + i) * 16 + (lane & 3);
                const uint32_t reals = __ballot_sync(0xFFFFFFFFu, real) >> (lane & ~3);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t o[32];
                    if (my_steps > 0 && ok) {  // warp-uniform
                        tmem_ld32(t_o + 32 * c, o);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0;
                    }
                    uint4 u[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            // (Zero by choice: where a value is infinite or NaN, the sum of zero times the values is NaN.)
                            w[i] = none ? 0u : narrow2<kBf16>(__uint_as_float(o[8 * e + 2 * i]) * factor, __uint_as_float(o[8 * e + 2 * i + 1]) * factor);
                        u[e] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    exchange4(u, lane);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (reals >> i & 1) to[i][4 * c] = u[i];
                }
            } else {
                const long long slot = (static_cast<long long>(item.segment) * 2 + stage) * p.slot_rows + row;
                const bool none = top == -INFINITY && sum == sum;
                if (real) p.part_ml[slot] = make_float2(none ? -INFINITY : -shift, none ? 0.0f : sum);
                const uint32_t reals = __ballot_sync(0xFFFFFFFFu, real) >> (lane & ~3);
                const bool any_real = __any_sync(0xFFFFFFFFu, real);
                uint4* const to = reinterpret_cast<uint4*>(p.part_o) + (slot - (lane & 3)) * 32 + (lane & 3);
                if (my_steps > 0 && ok) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        tmem_ld32(t_o + 32 * c, o);
                        tmem_wait_ld();
                        if (!any_real) continue;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint4 u[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) u[e] = make_uint4(o[16 * h + 4 * e], o[16 * h + 4 * e + 1], o[16 * h + 4 * e + 2], o[16 * h + 4 * e + 3]);
                            exchange4(u, lane);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (reals >> i & 1) to[32 * i + 8 * c + 4 * h] = u[i];
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Joins the partial results of a split launch: a warp per row, four channels per lane.
//   M = max m_i,  out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i,  lse = ln 2 (M + log2 of that sum).
// A partial that saw no key has l = 0 and its O was not written.
// Bound by the chain of its loads from L2: plan, maxima and sums (a lane each), partials.  Narrow rows have many partials, of
// which four are asked for at once; wide rows two or three (in a row 4.9 us for 512 rows of 2 to 40 partials, 16 us for 25000
// rows; one partial after the other, each with its own maximum and sum: 6.2 and 18).
template <bool kBf16, bool kNarrow>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ PackedParams p) {
    const PlanTiles& plan = *p.plan;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv_head = blockIdx.y, group0 = kv_head * p.G;
    const int per_cta = (kNarrow ? 1 : 2) * p.tokens;
    if (p.zero_tail && kv_head == 0 && blockIdx.z == 0) clear_tail(p, blockIdx.x, gridDim.x, threadIdx.x, 256);
    const int tile = blockIdx.x;
    if (tile >= plan.count) return;
    int q0, lq;
    bounds(p.cu_q, plan.seq[tile], p.Tq, &q0, &lq);
    const Shares shares(plan, p);
    // The shares that the tile's keys lie in, none where it has none.
    const long long from = static_cast<long long>(kv_head) * plan.start[plan.count] + plan.start[tile];
    const int cost = plan.start[tile + 1] - plan.start[tile];
    const int share0 = cost > 0 ? shares.owner(from + p.segment_cost) : 0;
    const int segments = cost > 0 ? shares.owner(from + cost - 1) - share0 + 1 : 0;
    const int segment0 = share0 + kv_head * plan.count + tile;
    const int token0 = plan.token0[tile], rows = min(per_cta, lq - token0) * p.G;
    const int stage_rows = p.tokens * p.G;
    const uint32_t inverse = 65536u / p.G + 1;  // r / G is r * inverse >> 16 for r < 256, G < 256
    for (int r = blockIdx.z * 8 + warp; r < rows; r += 8 * gridDim.z) {
        // Row r of the row tile is row r of its only 128-row tile, or of the second one.
        const int stage = !kNarrow && r >= stage_rows, slot_row = r - stage * stage_rows;
        const int parts = segments * (kNarrow ? 2 : 1);
        const auto slot = [&](int i) {
            const int segment = segment0 + (kNarrow ? i >> 1 : i), s = kNarrow ? i & 1 : stage;
            return (static_cast<long long>(segment) * 2 + s) * p.slot_rows + slot_row;
        };
        const auto max_and_sum = [&](int i) { return i < parts ? __ldcg(p.part_ml + slot(i)) : make_float2(-INFINITY, 0.0f); };
        const float2 mine = max_and_sum(lane);
        float top = mine.x;
        for (int i = 32 + lane; i < parts; i += 32) top = fmaxf(top, max_and_sum(i).x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
        for (int base = 0; base < parts; base += 32) {  // a lane weighs a partial, all lanes add it
            const float2 ml = base == 0 ? mine : max_and_sum(base + lane);
            const float weight = ml.y == 0.0f ? 0.0f : ml.y != ml.y ? ml.y : ex2(ml.x - top);
            sum = fmaf(weight, ml.y, sum);
            const int n = min(32, parts - base);
            constexpr int kBatch = kNarrow ? 4 : 1;
            for (int j = 0; j < n; j += kBatch) {
                float w[kBatch];
                float4 o[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    w[i] = __shfl_sync(0xFFFFFFFFu, weight, (j + i) & 31);
                    if (j + i >= n) w[i] = 0.0f;
                    o[i] = w[i] != 0.0f ? __ldcg(reinterpret_cast<const float4*>(p.part_o) + slot(base + j + i) * 32 + lane)
                                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    acc.x = fmaf(w[i], o[i].x, acc.x), acc.y = fmaf(w[i], o[i].y, acc.y), acc.z = fmaf(w[i], o[i].z, acc.z), acc.w = fmaf(w[i], o[i].w, acc.w);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int token = static_cast<int>(r * inverse >> 16);
        const long long t = q0 + token0 + token;
        const int head = group0 + r - token * p.G;
        reinterpret_cast<uint2*>(p.out)[(t * p.Hq + head) * 32 + lane] =
            make_uint2(narrow2<kBf16>(acc.x * factor, acc.y * factor), narrow2<kBf16>(acc.z * factor, acc.w * factor));
        if (p.lse != nullptr && lane == 0)
            p.lse[static_cast<long long>(head) * p.Tq + t] = sum == 0.0f ? -INFINITY : (top + __log2f(sum)) * 0.69314718055994531f;
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

// [tokens, heads, 128] of 16-bit values, read as (64 channels, heads, tokens, half) with a 128-byte-swizzled box.
int make_map(CUtensorMap* map, const void* base, bool bf16, int64_t tokens, int64_t heads, int64_t token_stride, int64_t head_stride,
             int box_heads, int box_tokens, int box_halves) {
    const EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return OVC_ERR_DRIVER;
    const cuuint64_t dims[4] = {64, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens), 2};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(head_stride) * 2, static_cast<cuuint64_t>(token_stride) * 2, 128};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens), static_cast<cuuint32_t>(box_halves)};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims,
                          strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_last_cuda_error(static_cast<int>(r));
        return OVC_ERR_DRIVER;
    }
    return OVC_OK;
}

// The current device; whether the library's code runs there (asked for once per device).
int sm100_device(int* device) {
    static std::atomic<unsigned long long> known;
    cudaError_t err = cudaGetDevice(device);
    if (err == cudaSuccess && *device < 64 && known.load(std::memory_order_acquire) >> *device & 1) return OVC_OK;
    int major = 0, minor = 0;
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *device);
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, *device);
    if (err != cudaSuccess) { set_last_cuda_error(err); return OVC_ERR_CUDA; }
    if (major != 10 || minor != 0) return OVC_ERR_UNSUPPORTED;
    if (*device < 64) known.fetch_or(1ull << *device, std::memory_order_release);
    return OVC_OK;
}

// How a launch is laid out; from sizes alone (the lengths of the sequences are on the device).
struct Layout {
    int mode, tokens, slot_rows;
    int64_t tiles;     // at most so many row tiles per key head
    int64_t segments;  // split: at most so many segments
};

constexpr int64_t kSms = 148;
constexpr int64_t kMostSlots = 1 << 19;  // rows of partial results: 270 MB of workspace

Layout lay_out(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk) {
    Layout l{};
    const int64_t G = Hq / Hk;
    l.tokens = static_cast<int>(kTile / G);
    // n sequences of at least one token make at most Tq tiles, and at most one tile each that is not full.
    const auto tiles = [&](int64_t per_tile) { const int64_t t = Tq / per_tile + B; return t < Tq ? t : Tq; };
    l.mode = kWhole, l.tiles = tiles(2 * l.tokens);
    const int64_t key_tiles = ceil_div(Tk, kTile), rows = Tq * G;
    l.slot_rows = static_cast<int>(rows < kTile ? rows : kTile);
    // Narrow where a sequence has on average no more rows than one tile, however many sequences there are: the time goes into
    // reading keys, which two stages on alternate key tiles do faster than one, in equal shares.
    const int64_t narrow = tiles(l.tokens), slots = (kSms + narrow * Hk) * 2 * l.slot_rows;
    if (rows <= kTile * B && narrow <= kMaxTiles && key_tiles >= 2 * B && slots <= kMostSlots) l.mode = kSplitNarrow, l.tiles = narrow;
    // Wide where whole row tiles leave SMs without work and there are keys enough to share.
    else if (l.tiles * Hk < kSms && l.tiles <= kMaxTiles && key_tiles >= 4 * B) l.mode = kSplitWide;
    l.segments = l.mode == kWhole ? 0 : kSms + l.tiles * Hk;
    return l;
}

constexpr int64_t kPlanBytes = (sizeof(PlanTiles) + 255) / 256 * 256;
int64_t workspace_bytes(const Layout& l) {
    return l.mode == kWhole ? 0 : kPlanBytes + l.segments * 2 * l.slot_rows * (kDim + 2) * static_cast<int64_t>(sizeof(float));
}

bool bad_sizes(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk) {
    return B < 1 || Tq < 1 || Tk < 1 || Hk < 1 || Hk > 65535 || Hq < Hk || Hq % Hk != 0 || Hq / Hk > kTile || B > (1 << 20) ||
           Tq > (1LL << 30) || Tk > (1LL << 30) || Hq > (1 << 20);
}

}  // namespace
}  // namespace ovc

using namespace ovc;

extern "C" int64_t ovc_attention_packed_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk) {
    if (bad_sizes(B, Tq, Tk, Hq, Hk)) return 0;
    return workspace_bytes(lay_out(B, Tq, Tk, Hq, Hk));
}

extern "C" int ovc_attention_packed(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                    const int64_t* v_strides, int dtype, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                    int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int flags, float softmax_scale, void* out,
                                    float* lse, void* workspace, uint32_t* status, uint32_t* host_status, void* stream) {
    if (bad_sizes(B, Tq, Tk, Hq, Hk) || !q || !k || !v || !q_strides || !k_strides || !v_strides || !cu_seqlens_q || !cu_seqlens_k || !out ||
        (dtype != OVC_F16 && dtype != OVC_BF16) || (flags & ~(OVC_ATTN_CAUSAL | OVC_ATTN_ZERO_TAIL)) != 0 || !(softmax_scale > 0.0f) ||
        !isfinite(softmax_scale * 1.4426950408889634f) || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) ||
        ((reinterpret_cast<uintptr_t>(cu_seqlens_q) | reinterpret_cast<uintptr_t>(cu_seqlens_k) | reinterpret_cast<uintptr_t>(lse)) & 3u))
        return OVC_ERR_ARGUMENT;
    for (const int64_t* s : {q_strides, k_strides, v_strides})
        if (s[0] <= 0 || s[1] <= 0 || s[0] % 8 || s[1] % 8 || s[0] >= (1LL << 38) || s[1] >= (1LL << 38)) return OVC_ERR_ARGUMENT;
    const Layout l = lay_out(B, Tq, Tk, Hq, Hk);
    if (workspace_bytes(l) > 0 && (!workspace || !aligned16(workspace))) return OVC_ERR_ARGUMENT;

    int device = 0;
    const int supported = sm100_device(&device);
    if (supported != OVC_OK) return supported;

    const bool bf16 = dtype == OVC_BF16, causal = (flags & OVC_ATTN_CAUSAL) != 0;
    const int64_t G = Hq / Hk;
    CUtensorMap map_q, map_k, map_v;
    int rc = make_map(&map_q, q, bf16, Tq, Hq, q_strides[0], q_strides[1], static_cast<int>(G), l.tokens, 1);
    if (rc == OVC_OK) rc = make_map(&map_k, k, bf16, Tk, Hk, k_strides[0], k_strides[1], 1, kTile, 2);
    if (rc == OVC_OK) rc = make_map(&map_v, v, bf16, Tk, Hk, v_strides[0], v_strides[1], 1, kTile, 2);
    if (rc != OVC_OK) return rc;

    PackedParams p{};
    p.cu_q = cu_seqlens_q, p.cu_k = cu_seqlens_k, p.out = out, p.lse = lse;
    p.plan = static_cast<PlanTiles*>(workspace);
    p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + (l.mode == kWhole ? 0 : kPlanBytes));
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (l.mode == kWhole ? 0 : l.segments * 2 * l.slot_rows * kDim));
    p.status = status, p.host_status = host_status;
    p.B = static_cast<int>(B), p.Hq = static_cast<int>(Hq), p.Hk = static_cast<int>(Hk), p.G = static_cast<int>(G);
    p.tokens = l.tokens, p.Tq = static_cast<int>(Tq), p.Tk = static_cast<int>(Tk);
    // Narrow: a segment's beginning and end take as long as about four key tiles (with 0, 2, 4, 6 of them sixteen requests
    // of 129 to 32768 keys took 116, 104, 96, 97 us).  Wide: a key tile takes three times as long, and is cheaper where only
    // one stage has rows; no count was better than shares by key tiles alone by more than runs differ (0, 2 and 4: 212 to 233
    // us in changing order for chunks behind prefixes).
    p.segment_cost = l.mode == kSplitNarrow ? 4 : 0;
    p.ctas = static_cast<int>(kSms), p.max_tiles = static_cast<int>(l.tiles < kMaxTiles ? l.tiles : kMaxTiles), p.slot_rows = l.slot_rows;
    p.zero_tail = (flags & OVC_ATTN_ZERO_TAIL) != 0;
    p.scale_log2 = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);

    constexpr int smem = sizeof(Smem);
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    auto s = static_cast<cudaStream_t>(stream);
    // CTAs start in the order of the grid.  Row tile by row tile, with all key heads of each, the long ones of a causal launch
    // come before the short ones whatever their head (356 -> 334 us for prompts of 5000 to 1 tokens); but the keys and values
    // of all heads are in use at once, and where those do not stay in L2 head by head is better (32768 keys of 8 heads, 134 MB:
    // 3.74 against 3.83 ms; two clips of 24 heads, 134 MB as well: 0.89 against 0.91).  Half of L2 is the border.
    p.heads_first = l.mode == kWhole && Tk * Hk * 4 * kDim <= 63LL << 20 && l.tiles <= 65535;
    const dim3 grid = l.mode != kWhole ? dim3(static_cast<unsigned>(kSms))
                      : p.heads_first  ? dim3(static_cast<unsigned>(Hk), static_cast<unsigned>(l.tiles))
                                       : dim3(static_cast<unsigned>(l.tiles), static_cast<unsigned>(Hk));
    const auto launch = [&](auto kernel, auto* ready) {  // ready: the devices on which the kernel may take that much
        if (device >= 64 || !(ready->load(std::memory_order_acquire) >> device & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e != cudaSuccess) { set_last_cuda_error(e); return static_cast<int>(OVC_ERR_CUDA); }
            if (device < 64) ready->fetch_or(1ull << device, std::memory_order_release);
        }
        kernel<<<grid, kThreads, smem, s>>>(map_q, map_k, map_v, p);
        return check_launch();
    };
    const auto by_mask = [&](auto is_bf16, auto is_causal) {
        constexpr bool kB = decltype(is_bf16)::value, kC = decltype(is_causal)::value;
        static std::atomic<unsigned long long> ready[3];
        if (l.mode == kWhole) return launch(packed_kernel<kB, kC, kWhole>, &ready[kWhole]);
        const int r = l.mode == kSplitNarrow ? launch(packed_kernel<kB, kC, kSplitNarrow>, &ready[kSplitNarrow])
                                             : launch(packed_kernel<kB, kC, kSplitWide>, &ready[kSplitWide]);
        if (r != OVC_OK) return r;
        const int rows = (l.mode == kSplitNarrow ? 1 : 2) * l.tokens * static_cast<int>(G);
        const int64_t mean = ceil_div(Tq * G, B);  // rows of a sequence; a row tile has them, or is full
        const dim3 cgrid(static_cast<unsigned>(l.tiles), static_cast<unsigned>(Hk), static_cast<unsigned>(ceil_div(mean < rows ? mean : rows, 16)));
        if (l.mode == kSplitNarrow) combine_kernel<kB, true><<<cgrid, 256, 0, s>>>(p);
        else combine_kernel<kB, false><<<cgrid, 256, 0, s>>>(p);
        return check_launch();
    };
    if (bf16) return causal ? by_mask(std::true_type{}, std::true_type{}) : by_mask(std::true_type{}, std::false_type{});
    return causal ? by_mask(std::false_type{}, std::true_type{}) : by_mask(std::false_type{}, std::false_type{});
}
