// FP8 ExpCast forward attention for sm_100a: TMA -> shared memory -> tcgen05 FP8 MMA with
// accumulators in tensor memory, score -> FP8 probability conversion on CUDA cores.
//
// One CTA owns 256 query rows of one (batch, head): two 128-row stages that ping-pong through one
// score buffer in tensor memory.  Numerics follow the reference's packed kernel
// (src/open_vc_attn/_kernels/blackwell/flash_attn/cute/flash_fwd_sm100.py:3513-3911 with
// cute/softmax.py:203-248 and cute/utils.py:704-795): running max in the descaled domain,
// ExpCast codes from one FMA and an FP16-subnormal rounding, denominator summed by the tensor core
// through a block of ones appended to the V tile.
//
// Warp roles (384 threads): warps 0-3 convert the scores of stage 0 (one query row per thread),
// warps 4-7 those of stage 1, warp 8 issues TMA loads, warp 9 issues the score products QK^T, warp 10
// relays "tile landed" from the TMA barriers into the MMA barriers, warp 11 issues the PV products.
//
// Schedule.  The two stages share one score buffer, so the scores form a chain: S_0(n) -> copied out ->
// S_1(n) -> copied out -> S_0(n+1) ...  Everything on that chain is kept short.  A conversion thread of
// stage s arrives on gate[s] right after it has copied S_s(n) out of tensor memory; on gate[s] warp 9
// (descriptors built before the wait) issues S = Q_{1-s} K^T for the other stage and commits to
// s_full[1-s].  The PV products are off the chain: a conversion thread arrives on p_full[s] when it has
// stored P_s(n) (and rescaled O_s if the row max moved); warp 11 then issues O_s += P_s(n) [V(n) | 1]
// and commits to pv_done[s], which the stage waits for before it overwrites P_s one step later.  The
// relay adds "K(n+1) landed" to gate[1] and "V(n) landed" to p_full[0], the first users of those
// tiles.  Shared-memory slots are recycled from progress that the conversion warps publish, not from
// extra commits.
//
// Tensor memory map (512 columns): S 0..127 (shared by both stages), P0 128..159, P1 160..191,
// O0 192..327, O1 328..463; each O region is 128 output columns followed by 8 copies of the
// denominator (the PV product has N = 136).  V-Smooth variant: O0 192..335, O1 336..479, each 128 output
// columns followed by 16 columns that collect the probability masses of sixteen key blocks one by one (N = 144:
// the extension of a V tile is one row of ones, row = key block mod 16), and W0 480..495, W1 496..511: those
// masses as BF16 high parts (8 columns) and low parts (8), the A operand of the products with the block means.

#include <atomic>

#include <cuda_bf16.h>
#include <math.h>

#include "common.cuh"
#include "scores.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.cuh"

namespace ovc {
namespace {

using namespace ptx;

constexpr int kThreads = 384;
constexpr int kKStages = 4;
constexpr int kVStages = 4;
constexpr int kTileBytes = kTile * kDim;          // 16384: one FP8 tile, 128 rows of 128 bytes
constexpr int kMeanGroup = 32;                    // key blocks per tile of block means (V-Smooth)
constexpr int kMeanSlice = 16;                    // key blocks restored by one group of BF16 products
// Rows appended to a V tile so that the PV product also sums P: 8 rows of ones (one denominator, 8 copies), or for
// V-Smooth 16 rows of which one holds ones (a denominator per key block of a slice).
__host__ __device__ constexpr int ext_rows(bool vs) { return vs ? kMeanSlice : 8; }
__host__ __device__ constexpr int pv_n(bool vs) { return kDim + ext_rows(vs); }  // 136 / 144
constexpr uint32_t kColS = 0, kColP = 128, kColO = 192, kColW = 480, kTmemCols = 512;

template <bool kVS, bool kVNat>
struct SmemLayout {
    alignas(1024) uint8_t q[2][kTileBytes];
    alignas(1024) uint8_t k[kKStages][kTileBytes];
    alignas(1024) uint8_t v[kVStages][kTileBytes + ext_rows(kVS) * 128];
    alignas(8) uint64_t q_full[2];
    uint64_t k_full[kKStages], v_full[kVStages];
    uint64_t k_empty[kKStages], v_empty[kVStages];  // slot may be refilled (one arrival by a stage-1 thread)
    uint64_t s_full[2];   // scores of a stage are in tensor memory (commit)
    uint64_t gate[2];     // the stage has copied its scores out of tensor memory (+ K tile landed for gate[1])
    uint64_t p_full[2];   // the stage has stored its probabilities of the step (+ V tile landed for p_full[0])
    uint64_t pv_done[2];  // the stage's previous PV has been accumulated (commit)
    uint64_t o_full[2], drain[2];
    uint64_t m_full[2], m_free[2];  // V-Smooth: a tile of block means has landed / its last reader is done (commit)
    uint32_t tmem_base;
    volatile uint32_t abort_flag;
    // V-Smooth only (a stub in the other variants): two tiles of block means, 128 channels x 128 bytes = BF16 high
    // parts of 32 key blocks, then their low parts, in the 128-byte swizzle.
    alignas(1024) uint8_t means[kVS ? 2 : 1][kVS ? kTileBytes : 16];
    // V in its [S,H,128] layout only (a stub otherwise): 128 rows of E4M3 1.0, the continuation of every V tile
    // along N (the MN-major operand's next 128-byte column), which makes the PV product sum P.
    alignas(1024) uint8_t ones[kVNat ? kTileBytes : 16];
};

struct AttnParams {
    const float* q_descale;  // [B,H,q_blocks]
    const float* k_descale;  // [B,H,n_tiles]
    const float* v_descale;  // [B,H]
    const float* repair_kd;  // [H,repair_rows] or null
    const float* vs_means;   // V-Smooth: [n_tiles,H,128] block means in code units, else null
    const float* vs_scale;   // V-Smooth: [H,128] channel scales
    __nv_bfloat16* out;      // [B,Sq,H,128]
    float* lse;              // [B,H,Sq] log-sum-exp of the scaled scores, or null
    uint32_t* status;
    long long Sq, Sk;
    int H, B, q_blocks, n_tiles, first_tile, m_blocks, mid_window;
    float scale_log2;
};

// Key tile visited at step `it`: from j0 down to first_tile, then from the right edge down to
// j0 + 1, then the repair prefix from first_tile - 1 down to 0.
__device__ __forceinline__ int tile_at(int it, int j0, int first_tile, int n_tiles) {
    const int len1 = j0 - first_tile + 1;
    const int originals = n_tiles - first_tile;
    if (it < len1) return j0 - it;
    if (it < originals) return n_tiles - 1 - (it - len1);
    return first_tile - 1 - (it - originals);
}

__device__ __forceinline__ void give_up(volatile uint32_t* abort_flag, uint32_t* status) {
    *abort_flag = 1;
    if (status != nullptr) {
        atomicOr(status, OVC_STATUS_WAIT_EXPIRED);      // this launch: later CTAs do not start
        atomicOr(status + 1, OVC_STATUS_WAIT_EXPIRED);  // sticky: for the host to read and clear
    }
}

__device__ __forceinline__ bool wait_bar(volatile uint32_t* abort_flag, uint64_t* bar, uint32_t parity, uint32_t* status,
                                         long long limit) {
    return wait_bounded(abort_flag, bar, parity, limit, [&] { give_up(abort_flag, status); });
}

template <class Layout>
__device__ __forceinline__ bool wait_bar(Layout& sm, uint64_t* bar, uint32_t parity, uint32_t* status) {
    return wait_bar(&sm.abort_flag, bar, parity, status, kWaitCycles);
}

// The MMA warp's reaction time is on the critical path of the shared score buffer, and it shares its
// scheduler with two conversion warps: descriptors are built before the wait, and after it come only a
// fence, one election, the four K-steps and the commit.
__device__ __forceinline__ uint64_t desc64(uint32_t lo) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(ptx::kSmemDescHi));
    return d;
}
__device__ __forceinline__ void qk_issue(uint32_t d_tmem, const uint64_t (&da)[4], const uint64_t (&db)[4], uint32_t idesc,
                                         uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred leader;\n\t"
        "tcgen05.fence::after_thread_sync;\n\t"
        "elect.sync _|leader, 0xFFFFFFFF;\n\t"
        "@leader tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %5, %9, 0;\n\t"
        "@leader tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %2, %6, %9, 1;\n\t"
        "@leader tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %3, %7, %9, 1;\n\t"
        "@leader tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %4, %8, %9, 1;\n\t"
        "@leader tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%10];\n\t}"
        :
        : "r"(d_tmem), "l"(da[0]), "l"(da[1]), "l"(da[2]), "l"(da[3]), "l"(db[0]), "l"(db[1]), "l"(db[2]), "l"(db[3]),
          "r"(idesc), "r"(bar)
        : "memory");
}

// bias = RD(-row_max * code_scale + 119.65 * 2^-24)
__device__ __forceinline__ float expcast_bias(float row_max, float code_scale) {
    float b;
    asm("fma.rm.f32 %0, %1, %2, 0f36EF4CCD;" : "=f"(b) : "f"(-row_max), "f"(code_scale));
    return b;
}

// ExpCast codes of 128 scores: y = x*scale + bias in units of 2^-24 (one packed FMA per pair), rounded
// to an FP16 subnormal whose low byte is the integer code (ReLU supplies the clamp at zero), low bytes
// gathered four at a time.  Written stage by stage over 32 columns so that every stage is a run of
// independent instructions.
// Two FP16-subnormal conversions give (c2:c0) and (c3:c1) with each code in the low byte of a half;
// one integer multiply-add (the FMA pipe, which has room) merges them into c0|c1<<8|c2<<16|c3<<24.
__device__ __forceinline__ uint32_t codes4(uint64_t y01, uint64_t y23) {
    uint32_t y0, y1, y2, y3, a, b, r;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(y0), "=r"(y1) : "l"(y01));
    asm("mov.b64 {%0, %1}, %2;" : "=r"(y2), "=r"(y3) : "l"(y23));
    asm("cvt.rn.relu.f16x2.f32 %0, %1, %2;" : "=r"(a) : "f"(__uint_as_float(y2)), "f"(__uint_as_float(y0)));
    asm("cvt.rn.relu.f16x2.f32 %0, %1, %2;" : "=r"(b) : "f"(__uint_as_float(y3)), "f"(__uint_as_float(y1)));
    asm("mad.lo.u32 %0, %1, 256, %2;" : "=r"(r) : "r"(b), "r"(a));
    return r;
}
__device__ __forceinline__ void encode128(const uint32_t (&s)[128], uint64_t scale2, uint64_t bias2, uint32_t (&codes)[32]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint64_t y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = ffma2(pack_u2(s[32 * c + 2 * i], s[32 * c + 2 * i + 1]), scale2, bias2);
#pragma unroll
        for (int i = 0; i < 8; ++i) codes[8 * c + i] = codes4(y[2 * i], y[2 * i + 1]);
    }
}

// After a failed wait: let the MMAs this thread has issued finish (bounded) before tensor memory is released.
template <class Layout>
__device__ __forceinline__ void drain_mmas(Layout& sm, int which) {
    mma_commit_elect(smem_addr(&sm.drain[which]));
    const long long t0 = clock64();
    while (!mbar_try_wait(smem_addr(&sm.drain[which]), 0) && clock64() - t0 < kWaitCycles) {}
}

// A launch that gave up (or found the status word already set) leaves NaN in the rows it owns, and -inf
// in their log-sum-exp, so that a caller that never reads the status word cannot mistake the buffer for a
// result.
__device__ __forceinline__ void poison_row(const AttnParams& p, int batch, int head, long long row) {
    if (row >= p.Sq) return;
    uint4* dst = reinterpret_cast<uint4*>(p.out + ((static_cast<long long>(batch) * p.Sq + row) * p.H + head) * kDim);
    const uint4 nan4 = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u);
#pragma unroll
    for (int i = 0; i < 16; ++i) dst[i] = nan4;
    if (p.lse != nullptr) p.lse[(static_cast<long long>(batch) * p.H + head) * p.Sq + row] = -INFINITY;
}

// kVS: V-Smooth variant (VC-Attention baseline): V holds residual codes; (sum of a key block's probabilities) x
// (the block's mean) is added to the accumulator for sixteen key blocks at a time by BF16 tensor-core products
// (cute/flash_fwd_sm100.py:4111-4206,4482-4526 of the reference), and the output is scaled per channel
// (cute/flash_fwd_sm100.py:4857-4863).
// The tensor map of the block means is a kernel parameter of the V-Smooth variant only.
template <bool kVS>
struct MeansMap {
    CUtensorMap map;
};
template <>
struct MeansMap<false> {
    int unused;
};

template <bool kVS, bool kCausal, bool kRepair, bool kVNat>
__global__ void __launch_bounds__(kThreads, 1)
attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                 const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ MeansMap<kVS> means_map,
                 const AttnParams p) {
    extern __shared__ uint8_t smem_raw[];
    using Layout = SmemLayout<kVS, kVNat>;
    Layout& sm = *reinterpret_cast<Layout*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m_block = blockIdx.x % p.m_blocks;
    const int bh = blockIdx.x / p.m_blocks;
    const int head = bh % p.H, batch = bh / p.H;

    // A barrier wait already expired in this launch (the entry point clears the word before the launch): do
    // not start more work.  One thread reads the word so that the whole CTA takes the same decision.
    __shared__ uint32_t skip_cta;
    if (threadIdx.x == 0) skip_cta = p.status != nullptr ? *reinterpret_cast<volatile uint32_t*>(p.status) : 0u;
    __syncthreads();
    if (skip_cta != 0) {
        if (threadIdx.x < 2 * kTile) poison_row(p, batch, head, static_cast<long long>(m_block) * (2 * kTile) + threadIdx.x);
        return;
    }
    // Causal (bottom-right aligned, cute/mask.py:186-199): key column c is visible to query row r iff
    // c < r + 1 + Sk - Sq, so this CTA's rows need the tiles below `visible` only (at least one tile is
    // visited: fully masked rows then end with a zero denominator and produce zeros).
    int visible = p.n_tiles;
    if (kCausal) {
        const long long last_row = min(static_cast<long long>(m_block + 1) * (2 * kTile), p.Sq) - 1;
        const long long limit = last_row + 1 + p.Sk - p.Sq;  // columns < limit
        visible = static_cast<int>(max(1LL, min(static_cast<long long>(p.n_tiles), (limit + kTile - 1) / kTile)));
    }
    const int n_tiles = visible;  // tiles this CTA visits (all of them unless causal)
    const int n_iters = n_tiles;
    const int j0 = p.mid_window < 0 ? n_tiles - 1
                                    : min(2 * m_block + p.first_tile + p.mid_window, n_tiles - 1);

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&sm.q_full[i]), 1);
            mbar_init(smem_addr(&sm.s_full[i]), 1);
            mbar_init(smem_addr(&sm.pv_done[i]), 1);
            mbar_init(smem_addr(&sm.o_full[i]), 1);
        }
        for (int i = 0; i < kKStages; ++i) {
            mbar_init(smem_addr(&sm.k_full[i]), 1);
            mbar_init(smem_addr(&sm.k_empty[i]), 1);
        }
        for (int i = 0; i < kVStages; ++i) {
            mbar_init(smem_addr(&sm.v_full[i]), 1);
            mbar_init(smem_addr(&sm.v_empty[i]), 1);
        }
        mbar_init(smem_addr(&sm.gate[0]), 128);    // the stage's conversion threads
        mbar_init(smem_addr(&sm.gate[1]), 129);    // + the relay: K(n+1) has landed
        mbar_init(smem_addr(&sm.p_full[0]), 129);  // + the relay: V(n) has landed
        mbar_init(smem_addr(&sm.p_full[1]), 128);
        mbar_init(smem_addr(&sm.drain[0]), 1);
        mbar_init(smem_addr(&sm.drain[1]), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&sm.m_full[i]), 1);
            mbar_init(smem_addr(&sm.m_free[i]), 1);
        }
        sm.abort_flag = 0;
        mbar_init_fence();
    }
    // Rows 128.. of every V slot: E4M3 1.0, so PV also accumulates the row sums of P.
    // (V-Smooth: all zero; the relay sets the row of the tile that has landed.)
    for (int i = threadIdx.x; i < kVStages * ext_rows(kVS) * 128 / 4; i += kThreads) {
        const int slot = i / (ext_rows(kVS) * 128 / 4), w = i % (ext_rows(kVS) * 128 / 4);
        reinterpret_cast<uint32_t*>(&sm.v[slot][kTileBytes])[w] = kVS ? 0u : 0x38383838u;
    }
    if (kVNat) {
        for (int i = threadIdx.x; i < kTileBytes / 4; i += kThreads) reinterpret_cast<uint32_t*>(sm.ones)[i] = 0x38383838u;
    }
    fence_proxy_async_smem();
    if (warp == 9) {
        tmem_alloc(smem_addr(&sm.tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 8) {
            // ---------------- TMA producer ----------------
            if (lane == 0) {
                tma_prefetch_desc(&tmap_q);
                tma_prefetch_desc(&tmap_k);
                tma_prefetch_desc(&tmap_v);
                const uint64_t keep = policy_evict_last(), stream = policy_evict_first();
                for (int s = 0; s < 2; ++s) {
                    mbar_expect_tx(smem_addr(&sm.q_full[s]), kTileBytes);
                    tma_load_4d(smem_addr(sm.q[s]), &tmap_q, smem_addr(&sm.q_full[s]), 0, head,
                                (2 * m_block + s) * kTile, batch, stream);
                }
                int issued_k = 0, issued_v = 0, issued_m = 0, j_before = 0;
                for (int it = 0; it < n_iters; ++it) {
                    const int j = tile_at(it, j0, p.first_tile, n_tiles);
                    const int ks = it % kKStages, vs = it % kVStages;
                    // K(it - kKStages) was last read by stage 1's QK of that step; stage 1 releases the slot
                    // when it sees those scores.
                    if (it >= kKStages &&
                        !wait_bar(sm, &sm.k_empty[ks], (it / kKStages - 1) & 1, p.status))
                        break;
                    mbar_expect_tx(smem_addr(&sm.k_full[ks]), kTileBytes);
                    tma_load_4d(smem_addr(sm.k[ks]), &tmap_k, smem_addr(&sm.k_full[ks]), 0, head, j * kTile, batch, keep);
                    issued_k = it + 1;
                    // V(it - kVStages) was last read by stage 1's PV of that step; stage 1 releases the slot
                    // when it sees that PV done.
                    if (it >= kVStages &&
                        !wait_bar(sm, &sm.v_empty[vs], (it / kVStages - 1) & 1, p.status))
                        break;
                    mbar_expect_tx(smem_addr(&sm.v_full[vs]), kTileBytes);
                    if (kVNat)  // [keys, head, 128 channels] like a K tile
                        tma_load_4d(smem_addr(sm.v[vs]), &tmap_v, smem_addr(&sm.v_full[vs]), 0, head, j * kTile, batch, keep);
                    else
                        tma_load_4d(smem_addr(sm.v[vs]), &tmap_v, smem_addr(&sm.v_full[vs]), j * kTile, 0, head, batch, keep);
                    issued_v = it + 1;
                    if (kVS && (it == 0 || j / kMeanGroup != j_before / kMeanGroup)) {
                        // The scan enters another group of 32 key blocks: fetch its means.  The buffer's previous
                        // group was left two groups ago; the PV issuer commits m_free when it leaves a group, at
                        // the step that enters the group before this one.  That step needs K of its successor
                        // (the relay hands "K(n+1) landed" over before "V(n) landed"), which may be this very
                        // iteration's tile: so the wait comes after this iteration's K and V loads, never before.
                        const int b = issued_m & 1;
                        if (issued_m >= 2 && !wait_bar(sm, &sm.m_free[b], ((issued_m >> 1) - 1) & 1, p.status)) break;
                        mbar_expect_tx(smem_addr(&sm.m_full[b]), kTileBytes);
                        if constexpr (kVS)
                            tma_load_4d(smem_addr(sm.means[b]), &means_map.map, smem_addr(&sm.m_full[b]), (j / kMeanGroup) * 128, 0, head, 0, keep);
                        ++issued_m;
                    }
                    j_before = j;
                }
                if (kVS) {
                    // A group whose blocks never complete a slice has no reader: its copy must still have landed
                    // before the CTA exits.
                    for (int c = max(0, issued_m - 2); c < issued_m; ++c) {
                        const long long t0 = clock64();
                        while (!mbar_try_wait(smem_addr(&sm.m_full[c & 1]), (c >> 1) & 1) && clock64() - t0 < kWaitCycles) {}
                    }
                }
                if (sm.abort_flag) {
                    // Give the copies already issued a bounded time to land before the CTA exits.
                    for (int s = 0; s < kKStages; ++s) {
                        int last = issued_k - 1;
                        while (last >= 0 && last % kKStages != s) --last;
                        const long long t0 = clock64();
                        while (last >= 0 && !mbar_try_wait(smem_addr(&sm.k_full[s]), (last / kKStages) & 1) &&
                               clock64() - t0 < kWaitCycles) {}
                    }
                    for (int s = 0; s < kVStages; ++s) {
                        int last = issued_v - 1;
                        while (last >= 0 && last % kVStages != s) --last;
                        const long long t0 = clock64();
                        while (last >= 0 && !mbar_try_wait(smem_addr(&sm.v_full[s]), (last / kVStages) & 1) &&
                               clock64() - t0 < kWaitCycles) {}
                    }
                    const long long t0 = clock64();
                    while (!(mbar_try_wait(smem_addr(&sm.q_full[0]), 0) && mbar_try_wait(smem_addr(&sm.q_full[1]), 0)) &&
                           clock64() - t0 < kWaitCycles) {}
                }
            }
        } else if (warp == 9) {
            // ---------------- MMA issuer ----------------
            constexpr uint32_t idesc_qk = idesc_e4m3_f32(kTile);
            bool ok = wait_bar(sm, &sm.q_full[0], 0, p.status) && wait_bar(sm, &sm.q_full[1], 0, p.status) &&
                      wait_bar(sm, &sm.k_full[0], 0, p.status);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (ok) {
                mma4_f8_ss(tmem + kColS, smem_desc_lo(smem_addr(sm.q[0])), smem_desc_lo(smem_addr(sm.k[0])), idesc_qk);
                mma_commit_elect(smem_addr(&sm.s_full[0]));
            }
            // gate[s] completion n: stage s has copied S_s(n) out, so the score buffer is free for the other
            // stage's next step (stage 1: step n, stage 0: step n + 1).
            for (int n = 0; ok && n < n_iters; ++n) {
                for (int s = 0; s < 2; ++s) {
                    const int qk_step = n + s;
                    if (qk_step >= n_iters) break;
                    const uint32_t a_lo = smem_desc_lo(smem_addr(sm.q[1 - s]));
                    const uint32_t b_lo = smem_desc_lo(smem_addr(sm.k[qk_step % kKStages]));
                    const uint64_t da[4] = {desc64(a_lo), desc64(a_lo + 2), desc64(a_lo + 4), desc64(a_lo + 6)};
                    const uint64_t db[4] = {desc64(b_lo), desc64(b_lo + 2), desc64(b_lo + 4), desc64(b_lo + 6)};
                    const uint32_t score_bar = smem_addr(&sm.s_full[1 - s]);
                    ok = __all_sync(0xFFFFFFFFu, wait_bar(sm, &sm.gate[s], n & 1, p.status));
                    if (!ok) break;
                    qk_issue(tmem + kColS, da, db, idesc_qk, score_bar);
                }
            }
            if (!ok) drain_mmas(sm, 0);
        } else if (warp == 11) {
            // ---------------- PV issuer ----------------
            // p_full[s] completion n: stage s has stored P_s(n) and V(n) has landed.
            // (The MN-major operand comes in units of 16 columns: N = 144, all sixteen extra columns sum P.)
            constexpr uint32_t idesc_pv = kVNat ? idesc_e4m3_f32_bmn(pv_n(true)) : idesc_e4m3_f32(pv_n(kVS));
            constexpr uint32_t kColOStride = pv_n(kVS || kVNat);
            constexpr uint32_t idesc_mean = idesc_bf16_f32(kDim);
            bool ok = true;
            int groups_left = 0;  // V-Smooth: groups of block means the scan has left (buffer groups_left & 1 is current)
            for (int n = 0; ok && n < n_iters; ++n) {
                // V-Smooth: when the previous step closed a slice of sixteen key blocks, the stages have stored the
                // slice's masses with this step's probabilities; O += W_hi M_hi + W_lo M_hi + W_hi M_lo goes first.
                bool restore = false, leave_group = false;
                uint32_t mean_lo = 0;
                if (kVS && n > 0) {
                    const int j_done = tile_at(n - 1, j0, p.first_tile, n_tiles);
                    restore = (j_done % kMeanSlice) == 0;
                    leave_group = tile_at(n, j0, p.first_tile, n_tiles) / kMeanGroup != j_done / kMeanGroup;
                    if (restore) {
                        ok = __all_sync(0xFFFFFFFFu, wait_bar(sm, &sm.m_full[groups_left & 1], (groups_left >> 1) & 1, p.status));
                        if (!ok) break;
                        mean_lo = smem_desc_lo(smem_addr(sm.means[groups_left & 1])) + 2 * ((j_done % kMeanGroup) / kMeanSlice);
                    }
                }
                for (int s = 0; s < 2; ++s) {
                    ok = __all_sync(0xFFFFFFFFu, wait_bar(sm, &sm.p_full[s], n & 1, p.status));
                    if (!ok) break;
                    tc_fence_after();
                    if (kVS && restore) {
                        const uint32_t w_hi = tmem + kColW + 16 * s, w_lo = w_hi + 8;
                        mma_bf16_ts(tmem + kColO + s * kColOStride, w_hi, mean_lo, idesc_mean);
                        mma_bf16_ts(tmem + kColO + s * kColOStride, w_lo, mean_lo, idesc_mean);
                        mma_bf16_ts(tmem + kColO + s * kColOStride, w_hi, mean_lo + 4, idesc_mean);
                    }
                    if (kVNat) {
                        const uint32_t slot = smem_addr(sm.v[n % kVStages]);
                        mma4_f8_ts_bmn(tmem + kColO + s * kColOStride, tmem + kColP + 32 * s,
                                       smem_desc_lo_bmn(slot, smem_addr(sm.ones) - slot), idesc_pv, n > 0 ? 1u : 0u);
                    } else {
                        mma4_f8_ts(tmem + kColO + s * kColOStride, tmem + kColP + 32 * s,
                                   smem_desc_lo(smem_addr(sm.v[n % kVStages])), idesc_pv, n > 0 ? 1u : 0u);
                    }
                    if (kVS && leave_group && s == 1) mma_commit_elect(smem_addr(&sm.m_free[groups_left & 1]));
                    mma_commit_elect(smem_addr(n + 1 < n_iters ? &sm.pv_done[s] : &sm.o_full[s]));
                }
                if (leave_group) ++groups_left;
            }
            if (!ok) drain_mmas(sm, 1);
        } else if (warp == 10) {
            // ---------------- relay: TMA arrivals -> MMA barriers ----------------
            // gate[1] completion n precedes the first product with K(n+1); p_full[0] completion n the first
            // with V(n).  One arrival per phase: the previous phase must have completed first.
            if (lane == 0) {
                for (int n = 0; n < n_iters; ++n) {
                    if (n > 0 && !wait_bar(sm, &sm.gate[1], (n - 1) & 1, p.status)) break;
                    if (n + 1 < n_iters &&
                        !wait_bar(sm, &sm.k_full[(n + 1) % kKStages], ((n + 1) / kKStages) & 1, p.status))
                        break;
                    mbar_arrive(smem_addr(&sm.gate[1]));
                    if (n > 0 && !wait_bar(sm, &sm.p_full[0], (n - 1) & 1, p.status)) break;
                    if (!wait_bar(sm, &sm.v_full[n % kVStages], (n / kVStages) & 1, p.status)) break;
                    if (kVS) {
                        // Row (key block mod 16) of the slot's extension holds ones, the others zeros: clear the row
                        // of the tile that used the slot before (its products are long done), set this tile's, and
                        // publish to the async proxy before the arrival that lets the first PV with this tile start.
                        uint4* ext = reinterpret_cast<uint4*>(&sm.v[n % kVStages][kTileBytes]);
                        if (n >= kVStages) {
                            const int old_row = tile_at(n - kVStages, j0, p.first_tile, n_tiles) % kMeanSlice;
#pragma unroll
                            for (int i = 0; i < 8; ++i) ext[old_row * 8 + i] = make_uint4(0u, 0u, 0u, 0u);
                        }
                        const int row = tile_at(n, j0, p.first_tile, n_tiles) % kMeanSlice;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            ext[row * 8 + i] = make_uint4(0x38383838u, 0x38383838u, 0x38383838u, 0x38383838u);
                        fence_proxy_async_smem();
                    }
                    mbar_arrive(smem_addr(&sm.p_full[0]));
                }
            }
        }
    } else {
        // ---------------- score conversion: one query row per thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int stage = warp >> 2;
        const int row_in_tile = (warp & 3) * 32 + lane;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t t_s = lane_base + kColS, t_p = lane_base + kColP + 32 * stage;
        const uint32_t t_o = lane_base + kColO + stage * pv_n(kVS || kVNat);
        const int q_tile = 2 * m_block + stage;
        const long long bh_l = static_cast<long long>(batch) * p.H + head;
        const float qd = q_tile < p.q_blocks ? __ldg(p.q_descale + bh_l * p.q_blocks + q_tile) : 1.0f;
        const float sigma = p.scale_log2 * qd;
        const float code_scale0 = sigma * 4.76837158203125e-07f;  // sigma * 8 * 2^-24
        const float* kd_row = p.k_descale + bh_l * p.n_tiles;
        const int tail_valid = static_cast<int>(p.Sk - static_cast<long long>(p.n_tiles - 1) * kTile);
        const uint32_t my_gate = smem_addr(&sm.gate[stage]);  // "scores copied out"

        float row_max = 0.0f, bias = 0.0f, saved_denominator = 0.0f;
        float l_closed = 0.0f;  // V-Smooth: denominator of the slices already closed, in the accumulator's scale
        int j_prev = 0;         // V-Smooth: key tile of the previous step
        const uint32_t t_w = lane_base + kColW + 16 * stage;
        bool ok = true;
        for (int it = 0; it < n_iters; ++it) {
            const int j = tile_at(it, j0, p.first_tile, n_tiles);
            const float kd = __ldg(kd_row + j);
            ok = __all_sync(0xFFFFFFFFu, wait_bar(sm, &sm.s_full[stage], it & 1, p.status));
            if (!ok) break;
            tc_fence_after();
            if (warp == 4 && lane == 0) mbar_arrive(smem_addr(&sm.k_empty[it % kKStages]));  // K(it) has been read
            uint32_t s[128];
            tmem_ld32(t_s, s);
            tmem_ld32(t_s + 32, s + 32);
            tmem_ld32(t_s + 64, s + 64);
            tmem_ld32(t_s + 96, s + 96);
            tmem_wait_ld();
            tc_fence_before();
            mbar_arrive(my_gate);

            if (j == p.n_tiles - 1 && tail_valid < kTile) {
#pragma unroll
                for (int c = 0; c < 128; ++c)
                    if (c >= tail_valid) s[c] = 0xFF800000u;  // -inf
            }
            if (kCausal) {
                // Columns of this tile that row `row` may see: c < row + 1 + Sk - Sq - 128 j.
                const long long first_row = static_cast<long long>(q_tile) * kTile;
                if (static_cast<long long>(j) * kTile + kTile - 1 > first_row + p.Sk - p.Sq) {  // some row of the tile is cut
                    const long long limit = first_row + row_in_tile + 1 + p.Sk - p.Sq - static_cast<long long>(j) * kTile;
                    const int visible_columns = static_cast<int>(max(0LL, min(static_cast<long long>(kTile), limit)));
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c >= visible_columns) s[c] = 0xFF800000u;  // -inf
                }
            }
            if (kRepair && j < p.first_tile) {
                // Repair keys come from different K blocks: each column carries its own K descale.
                const float4* kd4 = reinterpret_cast<const float4*>(p.repair_kd + static_cast<long long>(head) * p.first_tile * kTile + j * kTile);
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    const float4 f = __ldg(kd4 + c);
                    s[4 * c] = __float_as_uint(__uint_as_float(s[4 * c]) * f.x);
                    s[4 * c + 1] = __float_as_uint(__uint_as_float(s[4 * c + 1]) * f.y);
                    s[4 * c + 2] = __float_as_uint(__uint_as_float(s[4 * c + 2]) * f.z);
                    s[4 * c + 3] = __float_as_uint(__uint_as_float(s[4 * c + 3]) * f.w);
                }
            }
            // Row max first, then one encoding pass against the (possibly raised) max: a single copy of the
            // encoder in the loop body measured faster than encoding speculatively while the max is reduced.
            const float code_scale = code_scale0 * kd;
            const uint64_t scale2 = pack2(code_scale, code_scale);
            const float tile_max = max128(s) * kd;
            float alpha = 1.0f;
            if (it == 0 || tile_max > row_max) {
                float new_max = tile_max;
                alpha = 0.0f;
                if (it > 0) {
                    new_max = fmaxf(row_max, tile_max);
                    const float safe = new_max == -INFINITY ? 0.0f : new_max;
                    alpha = ex2((row_max - safe) * sigma);
                }
                row_max = new_max;
                bias = expcast_bias(new_max == -INFINITY ? 0.0f : new_max, code_scale0);
            }
            uint32_t codes[32];
            encode128(s, scale2, pack2(bias, bias), codes);
            if (it > 0) {
                // The stage's previous PV (step it-1) reads P_s and accumulates into O_s: wait for it before
                // P is overwritten or O is rescaled.
                ok = __all_sync(0xFFFFFFFFu, wait_bar(sm, &sm.pv_done[stage], (it - 1) & 1, p.status));
                if (!ok) break;
                tc_fence_after();
                if (warp == 4 && lane == 0) mbar_arrive(smem_addr(&sm.v_empty[(it - 1) % kVStages]));  // V(it-1) has been read
            }
            tmem_st32(t_p, codes);

            if (kVS) {
                const bool rescale = it > 0 && __any_sync(0xFFFFFFFFu, alpha < 1.0f);
                if (it > 0) {
                    // The sixteen mass columns hold the probability sums of the current slice's key blocks (the tensor
                    // core wrote them, one block per column).  When the previous step closed the slice, its masses
                    // go to the W columns as BF16 high and low parts - the PV issuer adds masses x block means to the
                    // accumulator before this step's PV - and the columns start again from zero.
                    const bool slice_closed = j_prev % kMeanSlice == 0;
                    l_closed *= alpha;
                    if (slice_closed || rescale) {
                        uint32_t m[kMeanSlice];
                        tmem_ld16(t_o + kDim, m);
                        tmem_wait_ld();
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < kMeanSlice; ++i) {
                            m[i] = __float_as_uint(__uint_as_float(m[i]) * alpha);
                            sum += __uint_as_float(m[i]);
                        }
                        if (slice_closed) {
                            l_closed += sum;
                            uint32_t hi[8], lo[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float a = __uint_as_float(m[2 * i]), b = __uint_as_float(m[2 * i + 1]);
                                hi[i] = bf16x2(a, b);
                                lo[i] = bf16x2(a - __uint_as_float(hi[i] << 16), b - __uint_as_float(hi[i] & 0xFFFF0000u));
                                m[2 * i] = 0u, m[2 * i + 1] = 0u;
                            }
                            tmem_st8(t_w, hi);
                            tmem_st8(t_w + 8, lo);
                        }
                        tmem_st16(t_o + kDim, m);
                    }
                    if (rescale) {
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
                j_prev = j;
            } else {
                const bool first_repair = kRepair && j == p.first_tile - 1;
                const bool rescale = it > 0 && __any_sync(0xFFFFFFFFu, alpha < 1.0f);
                if (first_repair) {
                    // First repair tile: the denominator holds the original tokens' total only.
                    saved_denominator = __uint_as_float(tmem_ld1(t_o + kDim));
                    tmem_wait_ld();
                }
                if (rescale) {
                    // The running max moved: rescale the accumulator and the denominator in place.
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        tmem_ld32(t_o + 32 * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st32(t_o + 32 * c, o);
                    }
                    const float l = __uint_as_float(tmem_ld1(t_o + kDim));
                    tmem_wait_ld();
                    tmem_st1(t_o + kDim, __float_as_uint(l * alpha));
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_addr(&sm.p_full[stage]));  // P_s(it) stored, O_s rescaled
        }
        if (ok) ok = __all_sync(0xFFFFFFFFu, wait_bar(sm, &sm.o_full[stage], 0, p.status));
        if (ok) {
            tc_fence_after();
            float l;
            float mass[kVS ? kMeanSlice : 1];  // V-Smooth: masses of the last slice (block = slice_first + column)
            if (kVS) {
                uint32_t m[kMeanSlice];
                tmem_ld16(t_o + kDim, m);
                tmem_wait_ld();
                l = l_closed;
#pragma unroll
                for (int i = 0; i < kMeanSlice; ++i) {
                    mass[i] = __uint_as_float(m[i]);
                    l += mass[i];
                }
            } else {
                l = __uint_as_float(tmem_ld1(t_o + kDim));
                tmem_wait_ld();
            }
            if (kRepair) l = saved_denominator;
            const bool bad = l == 0.0f || l != l;
            float inv;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(bad ? 1.0f : l));
            const float factor = inv * __ldg(p.v_descale + bh_l);
            if (p.lse != nullptr && static_cast<long long>(q_tile) * kTile + row_in_tile < p.Sq) {
                // (m*sigma + log2(l) - 8) ln 2: the codes put the row maximum at 2^8 (cute/flash_fwd_sm100.py:4455-4466).
                float lg;
                asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"(l));
                p.lse[bh_l * p.Sq + static_cast<long long>(q_tile) * kTile + row_in_tile] =
                    bad ? -INFINITY : (fmaf(row_max, sigma, lg) - 8.0f) * 0.6931471805599453f;
            }
            // V-Smooth: the masses still pending belong to the slice of the last tile visited; their means are
            // added here on the CUDA cores (once per CTA).
            const int slice_first = j_prev / kMeanSlice * kMeanSlice;
            const float* slice_means = kVS ? p.vs_means + (static_cast<long long>(slice_first) * p.H + head) * kDim : nullptr;
            const float* channel_scale = kVS ? p.vs_scale + static_cast<long long>(head) * kDim : nullptr;
            const long long row = static_cast<long long>(q_tile) * kTile + row_in_tile;
            uint4* dst = reinterpret_cast<uint4*>(p.out + ((static_cast<long long>(batch) * p.Sq + row) * p.H + head) * kDim);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                tmem_ld32(t_o + 32 * c, o);
                tmem_wait_ld();
                if (kVS) {
#pragma unroll
                    for (int i = 0; i < kMeanSlice; ++i) {
                        if (slice_first + i < p.n_tiles) {
                            const float4* mean4 = reinterpret_cast<const float4*>(
                                slice_means + static_cast<long long>(i) * p.H * kDim + 32 * c);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float4 m = __ldg(mean4 + e);
                                o[4 * e] = __float_as_uint(fmaf(mass[i], m.x, __uint_as_float(o[4 * e])));
                                o[4 * e + 1] = __float_as_uint(fmaf(mass[i], m.y, __uint_as_float(o[4 * e + 1])));
                                o[4 * e + 2] = __float_as_uint(fmaf(mass[i], m.z, __uint_as_float(o[4 * e + 2])));
                                o[4 * e + 3] = __float_as_uint(fmaf(mass[i], m.w, __uint_as_float(o[4 * e + 3])));
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        o[e] = __float_as_uint(__uint_as_float(o[e]) * __ldg(channel_scale + 32 * c + e));
                }
                if (row < p.Sq) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint4 w;
                        w.x = bf16x2(__uint_as_float(o[8 * e]) * factor, __uint_as_float(o[8 * e + 1]) * factor);
                        w.y = bf16x2(__uint_as_float(o[8 * e + 2]) * factor, __uint_as_float(o[8 * e + 3]) * factor);
                        w.z = bf16x2(__uint_as_float(o[8 * e + 4]) * factor, __uint_as_float(o[8 * e + 5]) * factor);
                        w.w = bf16x2(__uint_as_float(o[8 * e + 6]) * factor, __uint_as_float(o[8 * e + 7]) * factor);
                        dst[4 * c + e] = w;
                    }
                }
            }
        } else {
            poison_row(p, batch, head, static_cast<long long>(q_tile) * kTile + row_in_tile);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// V-Smooth: block means [n_tiles, H, 128] float32 -> the layout the attention kernel loads by TMA and multiplies as
// the B operand of a BF16 product: for every head and channel a row of n_groups x 128 bytes, each 128 bytes holding
// the BF16 high parts of the 32 key blocks of a group and then their BF16 low parts (mean = high + low to 16 bits;
// blocks past the end are zero).  One CTA per (group, head), one thread per channel.
__global__ void __launch_bounds__(kDim) means_split_kernel(const float* __restrict__ means, uint4* __restrict__ out,
                                                           int n_tiles, int H, int n_groups) {
    const int g = blockIdx.x, head = blockIdx.y, c = threadIdx.x;
    uint32_t hi[kMeanGroup / 2], lo[kMeanGroup / 2];
#pragma unroll
    for (int t = 0; t < kMeanGroup / 2; ++t) {
        float m[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = g * kMeanGroup + 2 * t + e;
            m[e] = j < n_tiles ? __ldg(means + (static_cast<long long>(j) * H + head) * kDim + c) : 0.0f;
        }
        hi[t] = bf16x2(m[0], m[1]);
        lo[t] = bf16x2(m[0] - __uint_as_float(hi[t] << 16), m[1] - __uint_as_float(hi[t] & 0xFFFF0000u));
    }
    uint4* row = out + ((static_cast<long long>(head) * kDim + c) * n_groups + g) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        row[i] = make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
        row[4 + i] = make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
    }
}

// The bounded wait on its own: one small CTA waits, with a caller-given limit, on a barrier that is one
// arrival short of its count and so can never complete.  Nothing else is in flight (no TMA, no MMA, no tensor
// memory), so giving up is the whole story: the status bit is set, the wait returns false and the CTA exits.
__global__ void __launch_bounds__(64, 1) wait_selftest_kernel(uint32_t* status, long long limit, uint32_t* gave_up) {
    __shared__ alignas(8) uint64_t barrier;
    __shared__ volatile uint32_t abort_flag;
    if (threadIdx.x == 0) {
        mbar_init(smem_addr(&barrier), 2);
        abort_flag = 0;
        mbar_init_fence();
    }
    __syncthreads();
    if (threadIdx.x == 0) mbar_arrive(smem_addr(&barrier));  // one of the two arrivals; the other never comes
    const bool completed = wait_bar(&abort_flag, &barrier, 0, status, limit);
    if (!completed) atomicAdd(gave_up, 1u);
}

// The score conversion on its own, for the MUFU-free ExpCast roofline: every SM runs the eight conversion warps
// of the attention kernel on scores that sit in tensor memory - tcgen05.ld of 128 columns, three-input max tree,
// bias, 128 ExpCast codes, tcgen05.st of the 32 code columns - with no barrier, no tensor-core product and no
// rescale in the loop.  What it sustains is the rate the CUDA cores alone allow the attention kernel.
__global__ void __launch_bounds__(256, 1) conversion_bench_kernel(uint32_t* sink, int tiles) {
    __shared__ uint32_t tmem_slot;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        tmem_alloc(smem_addr(&tmem_slot), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int stage = warp >> 2;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = lane_base + kColS, t_p = lane_base + kColP + 32 * stage;
    // scores: a ramp per row, so that no value is special
    if (stage == 0) {
        uint32_t init[32];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int e = 0; e < 32; ++e) init[e] = __float_as_uint(-0.25f * static_cast<float>((lane + 32 * c + e) & 127));
            tmem_st32(t_s + 32 * c, init);
        }
        tmem_wait_st();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    float row_max = -1e30f;
    uint32_t mix = 0;
    const float code_scale0 = 0.088388347648f * 1.4426950408889634f * 4.76837158203125e-07f;
    for (int it = 0; it < tiles; ++it) {
        uint32_t s[128];
        tmem_ld32(t_s, s);
        tmem_ld32(t_s + 32, s + 32);
        tmem_ld32(t_s + 64, s + 64);
        tmem_ld32(t_s + 96, s + 96);
        tmem_wait_ld();
        const float kd = 1.0f + 1e-3f * static_cast<float>(it & 7);
        const float tile_max = max128(s) * kd;
        row_max = fmaxf(row_max, tile_max);
        const float bias = expcast_bias(row_max, code_scale0);
        const float code_scale = code_scale0 * kd;
        uint32_t codes[32];
        encode128(s, pack2(code_scale, code_scale), pack2(bias, bias), codes);
        tmem_st32(t_p, codes);
        tmem_wait_st();
        mix ^= codes[it & 31];
    }
    if (mix == 0x9E3779B9u) sink[0] = mix;  // keeps the loop alive
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// ---- host side -------------------------------------------------------------------------------

// 4-D byte tensor (innermost first) with a 128-byte-swizzled box of box0 x box1 x 1 x 1.
int make_map(CUtensorMap* map, const void* base, const cuuint64_t (&dims)[4], const cuuint64_t (&strides)[3],
             cuuint32_t box0, cuuint32_t box1_dim, int box1_axis) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return OVC_ERR_DRIVER;
    cuuint32_t box[4] = {box0, 1, 1, 1};
    box[box1_axis] = box1_dim;
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_last_cuda_error(static_cast<int>(r));
        return OVC_ERR_DRIVER;
    }
    return OVC_OK;
}

}  // namespace
}  // namespace ovc

using namespace ovc;

namespace {

int launch_attention(const void* q8, const void* k8, const void* v_packed, const float* q_descale, int64_t q_blocks,
                     const float* k_descale, const float* v_descale, const float* repair_kd, int64_t repair_rows,
                     const float* vs_means, const float* vs_scale, void* vs_workspace, void* out, float* lse, int flags, int64_t B,
                     int64_t Sq, int64_t Sk, int64_t H, float softmax_scale, int mid_window_blocks, uint32_t* status,
                     void* stream) {
    if ((flags & ~(OVC_ATTN_CAUSAL | OVC_ATTN_V_UNPACKED)) != 0) return OVC_ERR_ARGUMENT;
    const bool causal = (flags & OVC_ATTN_CAUSAL) != 0, v_natural = (flags & OVC_ATTN_V_UNPACKED) != 0;
    if (causal && (mid_window_blocks != -1 || repair_rows != 0 || vs_means != nullptr)) return OVC_ERR_ARGUMENT;
    if (v_natural && (repair_rows != 0 || vs_means != nullptr)) return OVC_ERR_ARGUMENT;
    if (!q8 || !k8 || !v_packed || !q_descale || !k_descale || !v_descale || !out || B < 1 || Sq < 1 || Sk < 1 ||
        H < 1 || Sq > (1LL << 30) || Sk > (1LL << 30) || q_blocks < ceil_div(Sq, kTile) || !(softmax_scale > 0.0f) ||
        !isfinite(softmax_scale) || mid_window_blocks < -1 || repair_rows < 0 || repair_rows % kTile != 0 ||
        (repair_rows > 0 && (repair_kd == nullptr || repair_rows >= Sk || B != 1)) || !aligned16(q8) ||
        !aligned16(k8) || !aligned16(v_packed) || !aligned16(out) || (repair_kd && !aligned16(repair_kd)) ||
        (vs_means && (!vs_workspace || !aligned16(vs_workspace) || B != 1)))
        return OVC_ERR_ARGUMENT;
    const int64_t n_tiles = ceil_div(Sk, kTile), Sk_pad = n_tiles * kTile;
    const int64_t m_blocks = ceil_div(Sq, 2 * kTile);
    if (m_blocks * H * B > 0x7FFFFFFFLL) return OVC_ERR_ARGUMENT;

    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    int major = 0, minor = 0;
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device);
    if (err != cudaSuccess) { set_last_cuda_error(err); return OVC_ERR_CUDA; }
    if (major != 10 || minor != 0) return OVC_ERR_UNSUPPORTED;  // the library holds sm_100a code only

    CUtensorMap map_q, map_k, map_v;
    MeansMap<true> map_m{};
    {
        const cuuint64_t dq[4] = {128, static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(Sq), static_cast<cuuint64_t>(B)};
        const cuuint64_t sq[3] = {128, static_cast<cuuint64_t>(H) * 128, static_cast<cuuint64_t>(Sq) * H * 128};
        int rc = make_map(&map_q, q8, dq, sq, 128, 128, 2);
        if (rc != OVC_OK) return rc;
        const cuuint64_t dk[4] = {128, static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(Sk), static_cast<cuuint64_t>(B)};
        const cuuint64_t sk[3] = {128, static_cast<cuuint64_t>(H) * 128, static_cast<cuuint64_t>(Sk) * H * 128};
        rc = make_map(&map_k, k8, dk, sk, 128, 128, 2);
        if (rc != OVC_OK) return rc;
        // Extent Sk (not Sk_pad) along the keys: the padded tail reads as zero whatever it holds.
        const cuuint64_t dv[4] = {static_cast<cuuint64_t>(Sk), 128, static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(B)};
        const cuuint64_t sv[3] = {static_cast<cuuint64_t>(Sk_pad), static_cast<cuuint64_t>(Sk_pad) * 128,
                                  static_cast<cuuint64_t>(Sk_pad) * 128 * H};
        // V in [B,Sk,H,128] is loaded like K: a box of 128 channels x 128 keys, keys past Sk read as zero.
        rc = v_natural ? make_map(&map_v, v_packed, dk, sk, 128, 128, 2) : make_map(&map_v, v_packed, dv, sv, 128, 128, 1);
        if (rc != OVC_OK) return rc;
        if (vs_means != nullptr) {
            // Rows of n_groups x 128 bytes per (head, channel): see means_split_kernel.
            const cuuint64_t row_bytes = static_cast<cuuint64_t>(ceil_div(n_tiles, kMeanGroup)) * 128;
            const cuuint64_t dm[4] = {row_bytes, 128, static_cast<cuuint64_t>(H), 1};
            const cuuint64_t sm_[3] = {row_bytes, row_bytes * 128, row_bytes * 128 * H};
            rc = make_map(&map_m.map, vs_workspace, dm, sm_, 128, 128, 1);
            if (rc != OVC_OK) return rc;
        }
    }

    AttnParams p{};
    p.q_descale = q_descale, p.k_descale = k_descale, p.v_descale = v_descale, p.repair_kd = repair_kd;
    p.vs_means = vs_means, p.vs_scale = vs_scale;
    p.out = static_cast<__nv_bfloat16*>(out), p.lse = lse, p.status = status;
    p.Sq = Sq, p.Sk = Sk, p.H = static_cast<int>(H), p.B = static_cast<int>(B);
    p.q_blocks = static_cast<int>(q_blocks), p.n_tiles = static_cast<int>(n_tiles);
    p.first_tile = static_cast<int>(repair_rows / kTile), p.m_blocks = static_cast<int>(m_blocks);
    p.mid_window = mid_window_blocks;
    p.scale_log2 = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);

    const size_t smem_vs = sizeof(SmemLayout<true, false>) + 1024, smem_plain = sizeof(SmemLayout<false, false>) + 1024;
    const size_t smem_nat = sizeof(SmemLayout<false, true>) + 1024;
    const size_t smem_bytes = vs_means != nullptr ? smem_vs : (v_natural ? smem_nat : smem_plain);
    static std::atomic<bool> configured[64];
    if (device < 64 && !configured[device].load(std::memory_order_acquire)) {
        const auto grow = [&err](const void* kernel, size_t bytes) {
            if (err == cudaSuccess)
                err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
        };
        grow(reinterpret_cast<const void*>(attention_kernel<false, false, false, false>), smem_plain);
        grow(reinterpret_cast<const void*>(attention_kernel<false, false, true, false>), smem_plain);
        grow(reinterpret_cast<const void*>(attention_kernel<false, true, false, false>), smem_plain);
        grow(reinterpret_cast<const void*>(attention_kernel<true, false, false, false>), smem_vs);
        grow(reinterpret_cast<const void*>(attention_kernel<false, false, false, true>), smem_nat);
        grow(reinterpret_cast<const void*>(attention_kernel<false, true, false, true>), smem_nat);
        if (err != cudaSuccess) { set_last_cuda_error(err); return OVC_ERR_CUDA; }
        configured[device].store(true, std::memory_order_release);
    }
    const unsigned grid = static_cast<unsigned>(m_blocks * H * B);
    auto s = static_cast<cudaStream_t>(stream);
    if (status != nullptr) {
        // status[0] belongs to this launch alone: an expiry in an earlier call must not stop this one.
        err = cudaMemsetAsync(status, 0, sizeof(uint32_t), s);
        if (err != cudaSuccess) { set_last_cuda_error(err); return OVC_ERR_CUDA; }
    }
    if (vs_means != nullptr) {
        const int n_groups = static_cast<int>(ceil_div(n_tiles, kMeanGroup));
        means_split_kernel<<<dim3(n_groups, static_cast<unsigned>(H)), kDim, 0, s>>>(
            vs_means, static_cast<uint4*>(vs_workspace), static_cast<int>(n_tiles), static_cast<int>(H), n_groups);
        attention_kernel<true, false, false, false><<<grid, kThreads, smem_bytes, s>>>(map_q, map_k, map_v, map_m, p);
    } else {
        const MeansMap<false> none{};
        if (causal && v_natural) attention_kernel<false, true, false, true><<<grid, kThreads, smem_bytes, s>>>(map_q, map_k, map_v, none, p);
        else if (causal) attention_kernel<false, true, false, false><<<grid, kThreads, smem_bytes, s>>>(map_q, map_k, map_v, none, p);
        else if (v_natural) attention_kernel<false, false, false, true><<<grid, kThreads, smem_bytes, s>>>(map_q, map_k, map_v, none, p);
        else if (repair_rows > 0) attention_kernel<false, false, true, false><<<grid, kThreads, smem_bytes, s>>>(map_q, map_k, map_v, none, p);
        else attention_kernel<false, false, false, false><<<grid, kThreads, smem_bytes, s>>>(map_q, map_k, map_v, none, p);
    }
    return check_launch();
}

}  // namespace

extern "C" int ovc_bench_conversion(uint32_t* sink, int64_t ctas, int64_t tiles, void* stream) {
    if (!sink || ctas < 1 || ctas > 65535 || tiles < 1 || tiles > (1 << 24)) return OVC_ERR_ARGUMENT;
    conversion_bench_kernel<<<static_cast<unsigned>(ctas), 256, 0, static_cast<cudaStream_t>(stream)>>>(sink, static_cast<int>(tiles));
    return check_launch();
}

extern "C" int ovc_selftest_wait(uint32_t* status, int64_t limit_cycles, uint32_t* gave_up, void* stream) {
    if (!status || !gave_up || limit_cycles < 1 || limit_cycles > (1LL << 32)) return OVC_ERR_ARGUMENT;
    wait_selftest_kernel<<<1, 64, 0, static_cast<cudaStream_t>(stream)>>>(status, limit_cycles, gave_up);
    return check_launch();
}

extern "C" int ovc_attention(const void* q8, const void* k8, const void* v_packed, const float* q_descale,
                             int64_t q_blocks, const float* k_descale, const float* v_descale, const float* repair_kd,
                             int64_t repair_rows, void* out, int64_t B, int64_t Sq, int64_t Sk, int64_t H,
                             float softmax_scale, int mid_window_blocks, uint32_t* status, void* stream) {
    return launch_attention(q8, k8, v_packed, q_descale, q_blocks, k_descale, v_descale, repair_kd, repair_rows, nullptr,
                            nullptr, nullptr, out, nullptr, 0, B, Sq, Sk, H, softmax_scale, mid_window_blocks, status, stream);
}

extern "C" int ovc_attention_ex(const void* q8, const void* k8, const void* v_packed, const float* q_descale,
                                int64_t q_blocks, const float* k_descale, const float* v_descale, const float* repair_kd,
                                int64_t repair_rows, void* out, float* lse, int flags, int64_t B, int64_t Sq, int64_t Sk,
                                int64_t H, float softmax_scale, int mid_window_blocks, uint32_t* status, void* stream) {
    return launch_attention(q8, k8, v_packed, q_descale, q_blocks, k_descale, v_descale, repair_kd, repair_rows, nullptr,
                            nullptr, nullptr, out, lse, flags, B, Sq, Sk, H, softmax_scale, mid_window_blocks, status, stream);
}

extern "C" int64_t ovc_attention_vsmooth_workspace(int64_t Sk, int64_t H) {
    if (Sk < 1 || H < 1) return 0;
    return ceil_div(ceil_div(Sk, kTile), kMeanGroup) * 128 * kDim * H;
}

extern "C" int ovc_attention_vsmooth(const void* q8, const void* k8, const void* v_packed, const float* unit_descale,
                                     const float* means, const float* channel_scale, void* workspace, void* out,
                                     int64_t Sq, int64_t Sk, int64_t H, float softmax_scale, int mid_window_blocks,
                                     uint32_t* status, void* stream) {
    if (!means || !channel_scale || !unit_descale || !aligned16(means) || !aligned16(channel_scale) || H > 65535)
        return OVC_ERR_ARGUMENT;  // (the means are split by a grid with one row of CTAs per head)
    const int64_t blocks = ceil_div(Sq > Sk ? Sq : Sk, kTile);
    // unit_descale: at least H * ceil(max(Sq,Sk)/128) floats equal to 1.0 (no Q/K/V descales on this path).
    return launch_attention(q8, k8, v_packed, unit_descale, blocks, unit_descale, unit_descale, nullptr, 0, means,
                            channel_scale, workspace, out, nullptr, 0, 1, Sq, Sk, H, softmax_scale, mid_window_blocks, status, stream);
}
