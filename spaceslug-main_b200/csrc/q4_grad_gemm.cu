// The two large products of training through frozen int4 weights, on CTA
// pairs (tcgen05, cta_group::2):
//
//   TR = false, logits:  z[m][n]  = sum_k x[m][k] w(k, n)    (softmax cross entropy)
//   TR = true:           dx[m][k] = sum_n d[m][n] w(k, n)    (input gradient)
//
// w(k, n) = float(v) * scale (vulkan-runtime/shaders/q4gemm.comp:104-122).
// Both read the packed weights as they lie, [n][k/2] bytes, and dequantise
// them straight into the MMA's shared-memory operand: one packed word becomes
// 16 bytes (8 f16 of consecutive k) of the 128-byte row of its n, 128-byte
// swizzled.  That one image is the K-major operand of the logits (rows n,
// contraction k) and the MN-major operand of the transposed product (64 k
// contiguous, contraction n): only the descriptors differ.
//
// Precision.  The rows of x (or d) enter as f16 planes scaled by a power of
// two per row, the weights as f16 planes scaled by one power of two per
// handle.  PA, PB planes each: 1 = the value rounded once to 11 bits, 2 = hi
// and lo, 22 bits.  (1, 1): bf16 in and out, whose 8 bits are exact in f16,
// so only w is rounded (2^-12) below the output's own 2^-9.  (1, 2): logits
// of bf16 x, products to 2^-22, because the loss is fp32 (with the lo product
// in fp8 the logits' product took a quarter less, but logits were right to 7e-6
// of their norm only, where a plain 32-bit product has 3e-7).  (2, 2): fp32 (hi
// hi + hi lo + lo hi).  One scale for the whole handle loses nothing that
// shows: columns 2^-28 below the largest still have 11 bits.  The target's own
// logit comes from an fp32 product and its term is kept out of the sums, so
// that a loss near zero keeps its digits.
//
// The tensor core adds each MMA into its fp32 accumulator with truncation, so
// the accumulator is restarted after every chunk of `chunk` 64-wide stages
// and the chunks are added in registers, rounded to nearest.  The same place
// rescales: the cross entropy's second product takes p~ = exp(z - max of its
// 256-column tile) as operand and multiplies each 256-column chunk by
// exp(tile max - row max), so that no pass over the probabilities is needed
// between the two products.
//
// Roles (20 warps, 5 warpgroups): warp 0 loads the f16 planes of 128 rows per
// CTA (TMA, 128-byte swizzled boxes of 64), warp 1 of the leader issues the
// MMAs (M = 256, N = 256, K = 16); warp 3 loads packed words and scales (TMA:
// as cp.async copies, 16 or 4 bytes from a different row per lane, they took
// 512 of a stage's shared-memory cycles); warps 4-11 dequantise; warps 12-19 hold 128 fp32
// sums per thread (thread = row, two warps per tensor-memory lane quarter)
// and run the epilogue while the MMAs fill the other accumulator buffer.
// Every wait is bounded (status word + abort flag).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "q4_dequant.cuh"
#include "q4_grad.cuh"
#include "q4_kernels.h"

namespace q4 {

namespace {

constexpr int kGgRows = 256;   // rows of the pair's tile (128 per CTA, one accumulator lane each)
constexpr int kGgCols = 256;   // columns of the pair's tile
constexpr int kGgBK = 64;      // contraction per stage
constexpr int kGgHalf = 128;
constexpr int kGgTile = kGgHalf * kGgBK * 2;  // 16 KB: 128 rows of 64 f16
constexpr int kGgOutBytes = 4096;  // one block of 32 rows x 128 bytes per epilogue warp
constexpr int kGgRaw = 3;  // raw blocks in flight
constexpr int kGgDeqWarp0 = 4, kGgDeqWarps = 8;  // two warpgroups, one per stage of a raw block
constexpr int kGgEpiWarps = 8;
// Registers per thread after the split: the launch's 640 x 96 cover 128 x 32 + 256 x 56 + 256 x 168.
constexpr int kGgRegsLaunch = 96, kGgRegsCtl = 32, kGgRegsDeq = 56, kGgRegsEpi = 168;
static_assert(128 * kGgRegsCtl + 256 * kGgRegsDeq + 256 * kGgRegsEpi <= 640 * kGgRegsLaunch, "register split");

// WT: the weights come dequantised from planes in memory (TMA), without dequant
// warps and without a register split (384 threads of up to 168 registers).
template <int PA, int PB, bool WT>
struct GgCfg {
    static constexpr int kThreads = WT ? 384 : 640;
    static constexpr int kEpiWarp0 = WT ? 4 : 12;
    static constexpr int kRegsLaunch = WT ? 0 : kGgRegsLaunch;  // least the launch must have
    static constexpr int kB = PA * kGgTile;  // w hi, then w lo
    static constexpr int kStageBytes = (PA + PB) * kGgTile;
    static constexpr int kStages = PA + PB == 2 ? (WT ? 6 : 5) : PA + PB == 3 ? (WT ? 4 : 3) : 2;
    static constexpr int kOutOff = kStages * kStageBytes;
    static constexpr int kRawOff = kOutOff + kGgEpiWarps * kGgOutBytes;
    static constexpr int kXchOff = kRawOff + (WT ? 0 : kGgRaw * kGgRawBytes);  // [2 buffers][2 halves][128 rows] floats
    static constexpr int kBarOff = kXchOff + 2 * 2 * 128 * 4;
    // full_x[S], full_w[S] (leader), empty[S] (both), acc_full[2] (both), acc_empty[2] (leader), done (leader),
    // xch[4], full_r[R], empty_r[R] (own)
    static constexpr int kNumBars = 3 * kStages + 9 + 2 * kGgRaw;
    static constexpr int kMiscOff = kBarOff + kNumBars * 8;
    static constexpr int kBytes = kMiscOff + 16;
    // Dynamic shared memory starts 1024-aligned; with no room for slack a
    // window that does not is reported and nothing is loaded.
    static constexpr int kSlack = WT ? 0 : 1024;
    static constexpr int kSmem = kBytes + kSlack;
    static_assert(kSmem <= 232448, "shared memory budget");
};

template <int R>
__device__ __forceinline__ void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}

struct GgUnit {
    int mt, ct, z, c0, c1;  // row tile, column tile, split, chunks [c0, c1)
};
__device__ __forceinline__ GgUnit gg_unit(const GradGemmArgs& P, int u) {
    GgUnit w;
    const int tiles = P.row_tiles * P.col_tiles;
    const int t = u % tiles;
    w.z = u / tiles;
    w.mt = t % P.row_tiles;
    w.ct = t / P.row_tiles;
    w.c0 = static_cast<int>(static_cast<long long>(w.z) * P.chunks / P.splits);
    w.c1 = static_cast<int>(static_cast<long long>(w.z + 1) * P.chunks / P.splits);
    return w;
}

// Stores 16-byte piece `piece` of lane's 128-byte row of a warp's 32-row
// block, 128-byte swizzled as its tensor map expects.
__device__ __forceinline__ void gg_stage_row(uint8_t* buf, int lane, int piece, uint4 v) {
    *reinterpret_cast<uint4*>(buf + lane * 128 + ((piece ^ (lane & 7)) << 4)) = v;
}

template <bool TR, int PA, int PB, int EPI, bool WT>
__global__ void __launch_bounds__(WT ? 384 : 640, 1) grad_gemm_kernel(const __grid_constant__ GradGemmArgs P) {
    using C = GgCfg<PA, PB, WT>;
    constexpr int ST = C::kStages;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw_base = smem_u32(smem_raw);
    const uint32_t base = (raw_base + 1023u) & ~1023u;
    if (base - raw_base > static_cast<uint32_t>(C::kSlack)) {  // the same in every CTA
        if (threadIdx.x == 0 && P.status) atomicCAS(P.status, 0, kStatusBadLaunch);
        return;
    }
    uint8_t* smem = smem_raw + (base - raw_base);
    const uint32_t bar = base + C::kBarOff;
    auto full_x = [&](int s) { return bar + 8u * s; };
    auto full_w = [&](int s) { return bar + 8u * (ST + s); };
    auto empty = [&](int s) { return bar + 8u * (2 * ST + s); };
    auto acc_full = [&](int b) { return bar + 8u * (3 * ST + b); };
    auto acc_empty = [&](int b) { return bar + 8u * (3 * ST + 2 + b); };
    const uint32_t done_bar = bar + 8u * (3 * ST + 4);
    auto xch_bar = [&](int q) { return bar + 8u * (3 * ST + 5 + q); };
    auto full_r = [&](int r) { return bar + 8u * (3 * ST + 9 + r); };
    auto empty_r = [&](int r) { return bar + 8u * (3 * ST + 9 + kGgRaw + r); };
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kMiscOff);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kMiscOff + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t crank = cluster_ctarank();
    const bool leader = crank == 0;
    const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);
    const int units = P.row_tiles * P.col_tiles * P.splits;
    int* status = P.status;
    auto leader_addr = [&](uint32_t a) { return mapa_shared(a, 0); };

    if (tid == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(full_x(s), 1);                  // leader's expect_tx (both CTAs' bytes)
            mbar_init(full_w(s), kGgDeqWarps);        // one dequant warpgroup of each CTA
            mbar_init(empty(s), 1);                   // the leader's commit to both
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 2 * kGgEpiWarps);
        }
        for (int r = 0; r < kGgRaw; ++r) {
            mbar_init(full_r(r), 1);
            mbar_init(empty_r(r), kGgDeqWarps);
        }
        mbar_init(done_bar, 1);
        for (int q = 0; q < 4; ++q) mbar_init(xch_bar(q), 2);  // the two warps of a lane quarter
        *abort_flag = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&P.tm_a);
        tma_prefetch_desc(&P.tm_w);
        tma_prefetch_desc(&P.tm_s);
        tma_prefetch_desc(&P.tm_out);
    }
    if (warp == 2) {
        tmem_alloc_pair(smem_u32(tmem_holder), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_holder;

    if (warp < 4) {
        if constexpr (!WT) regs_dec<kGgRegsCtl>();
        if (warp == 0 && lane == 0) {
            // ------------------------------------------------ row planes --
            pdl_wait();
            int it = 0;
            bool ok = true;
            for (int u = pair; u < units && ok; u += npairs) {
                const GgUnit w = gg_unit(P, u);
                const int m0 = w.mt * kGgRows + static_cast<int>(crank) * kGgHalf;
                const int s1 = min(w.c1 * P.chunk, P.stages);
                for (int st = w.c0 * P.chunk; st < s1; ++st, ++it) {
                    const int s = it % ST;
                    if (!gg_wait(empty(s), ((it / ST) & 1u) ^ 1u, abort_flag, status, kStatusTimeoutProducer)) {
                        ok = false;
                        break;
                    }
                    if (leader) mbar_arrive_expect_tx(full_x(s), 2u * static_cast<uint32_t>(WT ? C::kStageBytes : C::kB));
                    const uint32_t fx = leader_addr(full_x(s));
                    if constexpr (WT) {
                        const uint32_t b = base + s * C::kStageBytes + C::kB;
                        const int tile0 = w.ct * kGgCols + static_cast<int>(crank) * kGgHalf;
                        if constexpr (TR) {  // 64 n x 128 k as two boxes of 64 k; the adapter's stage from A^T's planes
                            const bool at = st == P.lora_stage;
#pragma unroll
                            for (int p = 0; p < PB; ++p)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    tma_load_2d_pair(b + p * kGgTile + h * (kGgTile / 2),
                                                     at ? &P.tm_at : p == 0 ? &P.tm_w : &P.tm_s, fx, tile0 + 64 * h,
                                                     at ? 64 * p : st * kGgBK);
                        } else {
                            tma_load_2d_pair(b, &P.tm_w, fx, st * kGgBK, tile0);
                            if constexpr (PB == 2) tma_load_2d_pair(b + kGgTile, &P.tm_s, fx, st * kGgBK, tile0);
                        }
                    }
#pragma unroll
                    for (int p = 0; p < PA; ++p)
                        tma_load_2d_pair(base + s * C::kStageBytes + p * kGgTile, &P.tm_a, fx, st * kGgBK,
                                         p * P.plane_rows + m0);
                }
            }
            if (*abort_flag && leader)
                for (int j = (it > ST ? it - ST : 0); j < it; ++j) mbar_drain(full_x(j % ST), (j / ST) & 1u);
        } else if (!WT && warp == 3 && lane == 0) {
            // ---------------------------------------------- raw weights --
            int it = 0;
            bool ok = true;
            for (int u = pair; u < units && ok; u += npairs) {
                const GgUnit w = gg_unit(P, u);
                const int tile0 = w.ct * kGgCols + static_cast<int>(crank) * kGgHalf;
                const int s1 = min(w.c1 * P.chunk, P.stages);
                for (int st = w.c0 * P.chunk; st < s1; st += 2, ++it) {
                    const int r = it % kGgRaw;
                    if (!gg_wait(empty_r(r), ((it / kGgRaw) & 1u) ^ 1u, abort_flag, status, kStatusTimeoutProducer)) {
                        ok = false;
                        break;
                    }
                    const int k0 = TR ? tile0 : st * kGgBK, n0 = TR ? st * kGgBK : tile0;
                    const uint32_t dst = base + C::kRawOff + r * kGgRawBytes;
                    mbar_arrive_expect_tx(full_r(r), kGgRawBytes);
                    tma_load_2d(dst, &P.tm_w, full_r(r), k0 / 8, n0);
                    tma_load_2d(dst + kGgRawWords, &P.tm_s, full_r(r), k0 / 32, n0);
                }
            }
            if (*abort_flag)
                for (int j = (it > kGgRaw ? it - kGgRaw : 0); j < it; ++j)
                    mbar_drain(full_r(j % kGgRaw), (j / kGgRaw) & 1u);
        } else if (warp == 1 && leader && elect_one()) {
            // ------------------------------------------------------- MMA --
            constexpr uint32_t idesc = umma_idesc_f16(0u, kGgRows, kGgCols) | (TR ? (1u << 16) : 0u);
            int it = 0, cq = 0;
            bool ok = true;
            for (int u = pair; u < units && ok; u += npairs) {
                const GgUnit w = gg_unit(P, u);
                for (int c = w.c0; c < w.c1 && ok; ++c, ++cq) {
                    const int b = cq & 1;
                    if (!gg_wait(acc_empty(b), ((cq >> 1) & 1u) ^ 1u, abort_flag, status, kStatusTimeoutMma)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t dacc = tmem + static_cast<uint32_t>(b * kGgCols);
                    const int s1 = min((c + 1) * P.chunk, P.stages);
                    uint32_t acc = 0;
                    for (int st = c * P.chunk; st < s1; ++st, ++it) {
                        const int s = it % ST;
                        const uint32_t ph = (it / ST) & 1u;
                        if (!gg_wait(full_x(s), ph, abort_flag, status, kStatusTimeoutMma) ||
                            (!WT && !gg_wait(full_w(s), ph, abort_flag, status, kStatusTimeoutMma))) {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
                        const uint32_t at = base + s * C::kStageBytes, bt = at + C::kB;
                        auto mma = [&](int pa, int pb, int kk) {
                            const uint64_t ad = umma_desc_k_sw128(at + pa * kGgTile + kk * 32);
                            const uint64_t bd = TR ? gg_desc_mn_sw128(bt + pb * kGgTile + kk * 2048, kGgTile / 2)
                                                   : umma_desc_k_sw128(bt + pb * kGgTile + kk * 32);
                            umma_f16_ss_pair(dacc, ad, bd, idesc, acc);
                            acc = 1;
                        };
#pragma unroll
                        for (int kk = 0; kk < kGgBK / 16; ++kk) {
                            if constexpr (PA == 2) mma(1, 0, kk);
                            if constexpr (PB == 2) mma(0, 1, kk);
                            mma(0, 0, kk);
                        }
                        umma_commit_pair_both(empty(s), 0x3);
                    }
                    if (ok) umma_commit_pair_both(acc_full(b), 0x3);
                }
            }
            umma_commit_pair(mapa_shared(done_bar, 0));  // tracks every MMA issued above
            mbar_drain(done_bar, 0u);
        }
        __syncwarp();
    } else if (!WT && warp < C::kEpiWarp0) {
        // ------------------------------------------------------- dequant --
        // A raw block holds two stages: the k halves (logits) or the n halves
        // (transposed).  The two warpgroups take the stages of the whole
        // sequence in turn, so each waits for every second stage's slot, at most
        // kStages after the one before: a parity then cannot mistake the phase
        // before the last for the one waited for (as it could if a warpgroup
        // always took the same half and skipped the odd stage at a unit's end).
        // Thread t of a warpgroup: logits, column n = t of this CTA's 128 and
        // the stage's 64 k; transposed, n = t % 64 of the stage's 64 and the 64
        // k t / 64 of this CTA's 128: either way two scale groups of one n.
        if constexpr (!WT) regs_dec<kGgRegsDeq>();
        const int wg = (warp - kGgDeqWarp0) >> 2, t = (tid - kGgDeqWarp0 * 32) & 127;
        const float cs = exp2i(*P.w_exp);
        const int row = TR ? (t & 63) : t;  // row of the operand image, and of the block's first half
        const uint32_t out_row = static_cast<uint32_t>((TR ? (t >> 6) * (kGgTile / 2) : 0) + row * 128);
        const int rh = TR ? t >> 6 : 0, rkey = (row >> 1) & 3;  // 64-k half of the block's first half
        const uint32_t at0 = static_cast<uint32_t>(row * 64 + (((2 * rh) ^ rkey) << 4));
        const uint32_t at1 = static_cast<uint32_t>(row * 64 + (((2 * rh + 1) ^ rkey) << 4));
        const uint32_t ats = static_cast<uint32_t>(kGgRawWords + row * 16 + rh * 8);
        int it = 0, sq = 0;  // raw block and stage counters
        bool ok = true;
        for (int u = pair; u < units && ok; u += npairs) {
            const GgUnit w = gg_unit(P, u);
            const int s1 = min(w.c1 * P.chunk, P.stages);
            for (int st0 = w.c0 * P.chunk; st0 < s1; st0 += 2, ++it) {
                const int r = it % kGgRaw, n = min(2, s1 - st0);
                if (!gg_wait_warp(full_r(r), (it / kGgRaw) & 1u, abort_flag, status, kStatusTimeoutDequant)) {
                    ok = false;
                    break;
                }
                const uint8_t* raw = smem + C::kRawOff + r * kGgRawBytes;
                const int j = (sq ^ wg) & 1;  // this warpgroup's half
                // second half: 64 rows on (transposed), or the other 32 bytes of the row
                const uint32_t add = TR ? j * 64 * 64 : 0, flip = TR ? 0 : j * 32;
                const uint4 q[2] = {*reinterpret_cast<const uint4*>(raw + (at0 ^ flip) + add),
                                    *reinterpret_cast<const uint4*>(raw + (at1 ^ flip) + add)};
                const float2 sc = *reinterpret_cast<const float2*>(raw + ats + (TR ? j * 64 * 16 : j * 8));
                __syncwarp();
                if (lane == 0) mbar_arrive(empty_r(r));
                if (j < n) {
                    const int s = (sq + j) % ST;
                    if (!gg_wait_warp(empty(s), (((sq + j) / ST) & 1u) ^ 1u, abort_flag, status, kStatusTimeoutDequant)) {
                        ok = false;
                        break;
                    }
                    uint8_t* dst = smem + s * C::kStageBytes + C::kB + out_row;
                    if (TR && st0 + j == P.lora_stage) {  // A^T: row = rank, 64 k of this half, planes as prepared
                        pdl_wait();
                        const __half* lora_at = after_wait(static_cast<const __half*>(P.lora_at));
                        const int k0 = w.ct * kGgCols + static_cast<int>(crank) * kGgHalf + (t >> 6) * 64;
#pragma unroll
                        for (int p = 0; p < PB; ++p) {
                            const uint4* src = reinterpret_cast<const uint4*>(
                                lora_at + static_cast<size_t>(p * 64 + row) * P.ld_at + k0);
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                *reinterpret_cast<uint4*>(dst + p * kGgTile + ((i ^ (row & 7)) << 4)) = __ldg(src + i);
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            __half2 s_hi, s_lo;
                            split_scale_f16((h == 0 ? sc.x : sc.y) * cs, s_hi, s_lo);
                            const uint32_t words[4] = {q[h].x, q[h].y, q[h].z, q[h].w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint4 hi, lo;
                                gg_dequant<PB>(words[i], s_hi, s_lo, hi, lo);
                                const int o = ((4 * h + i) ^ (row & 7)) << 4;
                                *reinterpret_cast<uint4*>(dst + o) = hi;
                                if constexpr (PB == 2) *reinterpret_cast<uint4*>(dst + kGgTile + o) = lo;
                            }
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_remote(leader_addr(full_w(s)));
                }
                sq += n;
            }
        }
    } else {
        // ------------------------------------------------------ epilogue --
        if constexpr (!WT) regs_inc<kGgRegsEpi>();
        const int ew = warp - C::kEpiWarp0, quarter = warp & 3, half = ew >> 2;
        const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(half * 128);
        uint8_t* buf = smem + C::kOutOff + ew * kGgOutBytes;
        const uint32_t buf_s = base + C::kOutOff + ew * kGgOutBytes;
        const int row_in = quarter * 32 + lane;  // row of this CTA's 128
        const int wexp = *P.w_exp;
        pdl_wait();
        int cq = 0, xq = 0;
        bool ok = true;
        for (int u = pair; u < units && ok; u += npairs) {
            const GgUnit w = gg_unit(P, u);
            const int row0 = w.mt * kGgRows + static_cast<int>(crank) * kGgHalf + quarter * 32;
            const int row = row0 + lane;
            float acc[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[i][j] = 0.0f;
            for (int c = w.c0; c < w.c1; ++c, ++cq) {
                const int b = cq & 1;
                const float f = P.coef != nullptr ? after_wait(P.coef)[static_cast<size_t>(c) * P.ld_stat + row] : 1.0f;
                if (!gg_wait_warp(acc_full(b), (cq >> 1) & 1u, abort_flag, status, kStatusTimeoutEpilogue)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t v[16];
                    tmem_ld16(t_lane + static_cast<uint32_t>(b * kGgCols + i * 16), v);
                    gg_ld_wait(v);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        acc[i / 2][(i % 2) * 16 + j] = fmaf(f, __uint_as_float(v[j]), acc[i / 2][(i % 2) * 16 + j]);
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(leader_addr(acc_empty(b)));
            }
            if (!ok) break;
            const int rexp = P.row_exp != nullptr ? (row < P.M ? after_wait(P.row_exp)[row] : 0) : P.fixed_exp;
            const float scale = exp2i(-(rexp + wexp) / 2) * exp2i(-(rexp + wexp) - (-(rexp + wexp) / 2));
            const int col0 = w.ct * kGgCols + half * 128;
            if constexpr (EPI == kGgLoss || EPI == kGgProb) {
                // In units of log2: z2 = z log2(e); this tile's row maximum over the
                // columns that exist other than the target's (whose logit the
                // cast has from an fp32 product), and the sum of 2^(z2 - max).
                const float s2 = scale * 1.4426950408889634f;
                const long long tgt = row < P.M ? after_wait(P.targets)[row] : -1;
                const int tcol = tgt >= col0 && tgt < col0 + 128 ? static_cast<int>(tgt) - col0 : -1;
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const int c = i * 32 + j;
                        acc[i][j] = col0 + c < P.N && c != tcol ? acc[i][j] * s2 : -INFINITY;
                        top = fmaxf(top, acc[i][j]);
                    }
                // the two warps of these rows, through a buffer that alternates: a warp
                // writes one again only after its partner has arrived for the other
                float* xch = reinterpret_cast<float*>(smem + C::kXchOff) + (xq & 1) * 256;
                xch[half * 128 + row_in] = top;
                __syncwarp();
                if (lane == 0) mbar_arrive(xch_bar(quarter));
                if (!gg_wait_warp(xch_bar(quarter), xq & 1u, abort_flag, status, kStatusTimeoutEpilogue)) {
                    ok = false;
                    break;
                }
                ++xq;
                top = fmaxf(top, xch[(half ^ 1) * 128 + row_in]);
                const float ref = top == -INFINITY ? 0.0f : top;  // a tile of the target alone: all terms 0
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        acc[i][j] = ex2(acc[i][j] - ref);  // 2^-inf = 0 where there is no term
                        sum += acc[i][j];
                    }
                if (half == 0) P.smax[static_cast<size_t>(w.ct) * P.ld_stat + row] = top;
                P.ssum[(static_cast<size_t>(w.ct) * 2 + half) * P.ld_stat + row] = sum;
                if constexpr (EPI == kGgProb) {
                    constexpr int PP = PA;  // planes of p~: as many as the rows' own
#pragma unroll
                    for (int p = 0; p < PP; ++p)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {  // 64 columns = 128 bytes at a time
                            if (lane == 0) bulk_wait_group_read<0>();
                            __syncwarp();
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                uint32_t o[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    float& a0 = acc[2 * h + e / 4][(e % 4) * 8 + 2 * j];
                                    float& a1 = acc[2 * h + e / 4][(e % 4) * 8 + 2 * j + 1];
                                    const float f0 = p == 0 ? a0 * 16384.0f : a0, f1 = p == 0 ? a1 * 16384.0f : a1;
                                    const __half2 hv = __floats2half2_rn(f0, f1);
                                    if (PP == 2 && p == 0) {
                                        a0 = f0 - __low2float(hv);  // exact: what lo keeps
                                        a1 = f1 - __high2float(hv);
                                    }
                                    o[j] = *reinterpret_cast<const uint32_t*>(&hv);
                                }
                                gg_stage_row(buf, lane, e, make_uint4(o[0], o[1], o[2], o[3]));
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0 && row0 < P.M) {
                                tma_store_2d(&P.tm_out, buf_s, col0 + h * 64, p * P.out_rows + row0);
                                bulk_commit_group();
                            }
                        }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[i][j] *= scale;
                constexpr int kOutCols = EPI == kGgBf16 ? 64 : 32;  // columns of a 128-byte block row
                const int orow = w.z * P.out_rows + row0;
#pragma unroll
                for (int h = 0; h < 128 / kOutCols; ++h) {
                    if (lane == 0) bulk_wait_group_read<0>();
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint4 o;
                        if constexpr (EPI == kGgBf16) {
                            const int c8 = h * kOutCols + e * 8;
                            uint32_t q[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const __nv_bfloat162 hv =
                                    __floats2bfloat162_rn(acc[c8 / 32][c8 % 32 + gg_place(2 * j)],
                                                          acc[c8 / 32][c8 % 32 + gg_place(2 * j + 1)]);
                                q[j] = *reinterpret_cast<const uint32_t*>(&hv);
                            }
                            o = make_uint4(q[0], q[1], q[2], q[3]);
                        } else {
                            const int c4 = h * kOutCols + e * 4, c8 = c4 & ~7, k4 = c4 & 4;
                            o = make_uint4(__float_as_uint(acc[c8 / 32][c8 % 32 + gg_place(k4)]),
                                           __float_as_uint(acc[c8 / 32][c8 % 32 + gg_place(k4 + 1)]),
                                           __float_as_uint(acc[c8 / 32][c8 % 32 + gg_place(k4 + 2)]),
                                           __float_as_uint(acc[c8 / 32][c8 % 32 + gg_place(k4 + 3)]));
                        }
                        gg_stage_row(buf, lane, e, o);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    const int oc = col0 + h * kOutCols;
                    if (lane == 0 && row0 < P.M && oc < P.K) {
                        tma_store_2d(&P.tm_out, buf_s, oc, orow);
                        bulk_commit_group();
                    }
                }
            }
        }
        if (lane == 0) bulk_wait_group_all();
    }

    pdl_launch_dependents();  // here: blocks of the next launch that wait beside this one's cost it 3%
    tc_fence_before_sync();
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while its peer may still use its shared memory or tensor memory
    if (warp == 2) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem, 512);
    }
}

template <bool TR, int PA, int PB, int EPI, bool WT>
int gg_pairs() {
    using C = GgCfg<PA, PB, WT>;
    static std::atomic<int> cache[64];  // pairs + 1; 0: not asked yet
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (const int known = cache[dev].load(std::memory_order_acquire)) return known - 1;
    auto kern = grad_gemm_kernel<TR, PA, PB, EPI, WT>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess) return 0;
    cudaFuncAttributes fa{};
    // the register split draws on the launch's registers: refuse a build that was given fewer
    if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess || fa.numRegs < C::kRegsLaunch) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2, 1, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) return 0;
    cache[dev].store(n + 1, std::memory_order_release);
    return n;
}

template <bool TR, int PA, int PB, int EPI, bool WT>
int gg_launch(const GradGemmArgs& a, cudaStream_t stream) {
    using C = GgCfg<PA, PB, WT>;
    auto kern = grad_gemm_kernel<TR, PA, PB, EPI, WT>;
    int cap = gg_pairs<TR, PA, PB, EPI, WT>();
    if (a.max_pairs > 0 && cap > a.max_pairs) cap = a.max_pairs;
    const long long units = static_cast<long long>(a.row_tiles) * a.col_tiles * a.splits;
    if (cap < 1 || units < 1 || units > (1ll << 30)) return static_cast<int>(cudaErrorInvalidConfiguration);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (units < cap ? units : cap)), 1, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, a));
}

// ------------------------------------------------------------------ helpers --
// Every kernel of this file starts under the tail of the one before
// (programmatic dependent launch) and waits for it before it touches memory
// that a call writes.
template <typename... Params, typename... Args>
int gg_launch_pdl(void (*kern)(Params...), unsigned grid, unsigned threads, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...));
}
__device__ __forceinline__ float gg_in(const float* p) { return *p; }
__device__ __forceinline__ float gg_in(const __nv_bfloat16* p) { return __bfloat162float(*p); }
// Threads per row of the cast: 2048 x 11008 bf16 takes 19 us with 128, 23 with
// 256 and 30 with 512 (block-wide steps); up to kCastFew rows, a block per SM or
// less, 512 (fp32, 32 x 11008: 6.8 us against 9.2; 128 x 11008: 5.6 against 8.1).
constexpr int kCastThreads = 128, kCastThreadsFew = 512, kCastFew = 128;
// Eight columns as loaded: a batch of them is in flight before the first is used.
template <typename T>
struct GgRaw8;
template <>
struct GgRaw8<float> {
    static constexpr int kBatch = 2;
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <>
struct GgRaw8<__nv_bfloat16> {
    static constexpr int kBatch = 4;
    uint4 q;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { q = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
// f(p, v) for this thread's pieces of 8 columns p = thread, thread + THREADS, ... of a row of whole 16-byte pieces.
template <int THREADS, typename T, typename F>
__device__ __forceinline__ void gg_row(const T* row, int cols, F&& f) {
    const int pieces = cols / 8;
    using R = GgRaw8<T>;
    for (int p0 = threadIdx.x; p0 < pieces; p0 += THREADS * R::kBatch) {
        R q[R::kBatch];
#pragma unroll
        for (int u = 0; u < R::kBatch; ++u)
            if (p0 + THREADS * u < pieces) q[u].load(row + (p0 + THREADS * u) * 8);
#pragma unroll
        for (int u = 0; u < R::kBatch; ++u)
            if (p0 + THREADS * u < pieces) {
                float v[8];
                q[u].values(v);
                f(p0 + THREADS * u, v);
            }
    }
}
// f(c, v) for this thread's columns c = thread, thread + THREADS, ..., zero from cols to `end`: a row that starts
// anywhere, whole lines per warp and eight loads in flight (515 x 4099 and 2048 x 11007: fp32 8.7 and 41 us, bf16 8.2
// and 36; as pieces of 8 columns per thread 10.6 and 54, 7.1 and 37).
template <int THREADS, typename T, typename F>
__device__ __forceinline__ void gg_row_each(const T* row, int cols, int end, F&& f) {
    for (int c0 = threadIdx.x; c0 < end; c0 += THREADS * 8) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = c0 + THREADS * u < cols ? gg_in(row + c0 + THREADS * u) : 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (c0 + THREADS * u < end) f(c0 + THREADS * u, v[u]);
    }
}

// One block per row: f16 planes [planes][M][ld] of row * 2^e, e such that the
// largest magnitude lies in [2^13, 2^14); lo = the f16 rounding of what hi
// leaves.  Columns past the row are zero.  With an adapter the last 64 columns
// are the row's G = s dY B^T (the sum of its partial products) times 2^gexp[j],
// the exponents that A^T's planes were scaled down by, so that G A^T is 64
// more terms of the same contraction; the row's exponent covers them too.
// For the loss it also forms the target's logit in fp32.
// The row is read twice, the second time from L1 / L2: keeping it in registers
// (48 floats a thread) halves the blocks per SM and measured slower (24 against
// 16 us at 4096 x 4096 bf16).
template <typename T, int PA, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS) cast_planes_kernel(const CastArgs A) {
    __shared__ float red[THREADS / 32];
    __shared__ float gs[64];
    pdl_launch_dependents();
    pdl_wait();
    const long long m = blockIdx.x;
    const T* row = after_wait(static_cast<const T*>(A.x)) + m * A.cols;
    const long long* targets = after_wait(A.targets);
    const float* gpart = after_wait(A.gpart);
    const int* gexp = after_wait(A.gexp);
    const int pieces = (A.cols + 7) / 8;
    float top = 0.0f, dot = 0.0f;
    const long long tgt = targets != nullptr ? targets[m] : -1;
    const bool want_dot = tgt >= 0 && tgt < A.N;
    if constexpr (VEC) {
        gg_row<THREADS>(row, A.cols, [&](int p, const float (&v)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
            if (want_dot) {  // the target's logit, w = v s in fp32
                const uint32_t q = __ldg(A.packed + tgt * (A.cols / 8) + p);
                float part = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    part = fmaf(v[i], static_cast<float>((static_cast<int>((q >> (4 * i)) & 15u) ^ 8) - 8), part);
                dot = fmaf(part, __ldg(A.scales + tgt * (A.cols / 32) + (p >> 2)), dot);
            }
        });
    } else {
        gg_row_each<THREADS>(row, A.cols, A.cols, [&](int, float v) { top = fmaxf(top, fabsf(v)); });
    }
    if (A.rank > 0 && threadIdx.x < 64) {
        float g = 0.0f;
        if (threadIdx.x < A.rank) {
            for (int z = 0; z < A.gsplits; ++z)
                g += gpart[(static_cast<long long>(z) * A.M + m) * A.gpitch + threadIdx.x];
            g = ldexpf(g * A.gscale, gexp[threadIdx.x]);
        }
        gs[threadIdx.x] = g;
        top = fmaxf(top, fabsf(g));
    }
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int i = 0; i < THREADS / 32; ++i) top = fmaxf(top, red[i]);
    int e = 0;
    if (top > 0.0f && isfinite(top)) {
        int e2;
        frexpf(top, &e2);
        e = min(max(14 - e2, -120), 120);
    }
    if (threadIdx.x == 0) A.row_exp[m] = e;
    const float s = exp2i(e);
    if (targets != nullptr) {
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        __syncthreads();  // red has been read
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = dot;
        __syncthreads();
        if (threadIdx.x == 0) {
            float z = 0.0f;
            for (int i = 0; i < THREADS / 32; ++i) z += red[i];
            A.zt[m] = z;
        }
    }
    __half* hi = static_cast<__half*>(A.out) + m * A.ld;
    auto put = [&](int p, const float (&v)[8]) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // in order, or as (0, 4), (1, 5), (2, 6), (3, 7): the order of the dequantised words
            const float a = (A.by_word ? v[i] : v[2 * i]) * s, b = (A.by_word ? v[i + 4] : v[2 * i + 1]) * s;
            const __half2 hv = __floats2half2_rn(a, b);
            h[i] = *reinterpret_cast<const uint32_t*>(&hv);
            if constexpr (PA == 2) {
                const __half2 lv = __floats2half2_rn(a - __low2float(hv), b - __high2float(hv));
                l[i] = *reinterpret_cast<const uint32_t*>(&lv);
            }
        }
        *reinterpret_cast<uint4*>(hi + p * 8) = make_uint4(h[0], h[1], h[2], h[3]);
        if constexpr (PA == 2)
            *reinterpret_cast<uint4*>(hi + static_cast<long long>(A.M) * A.ld + p * 8) = make_uint4(l[0], l[1], l[2], l[3]);
    };
    if constexpr (VEC) {
        gg_row<THREADS>(row, A.cols, put);
    } else {  // no targets, nothing by word: rows of dY
        gg_row_each<THREADS>(row, A.cols, 8 * pieces, [&](int c, float v) {
            const __half h = __float2half_rn(v * s);
            hi[c] = h;
            if constexpr (PA == 2)
                hi[static_cast<long long>(A.M) * A.ld + c] = __float2half_rn(v * s - __half2float(h));
        });
    }
    const int end = static_cast<int>(A.ld / 8), gp = A.rank > 0 ? end - 8 : end;
    for (int p = pieces + threadIdx.x; p < end; p += THREADS) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p >= gp ? gs[(p - gp) * 8 + i] : 0.0f;
        put(p, v);
    }
}

// The dequantised planes [N][K] of a handle's weights, in the dequantised
// words' order: what the products' dequant warps write to shared memory, once
// for all row tiles.  Four words per thread, a block apart.
template <bool LO>
__global__ void __launch_bounds__(256) weight_planes_kernel(const uint32_t* __restrict__ packed,
                                                            const float* __restrict__ scales,
                                                            const int* __restrict__ w_exp, __half* __restrict__ hi,
                                                            __half* __restrict__ lo, long long words) {
    pdl_launch_dependents();
    const float cs = exp2i(*w_exp);
    const long long i0 = static_cast<long long>(blockIdx.x) * 1024 + threadIdx.x;
    uint32_t q[4];
    float s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const long long i = i0 + u * 256;
        q[u] = i < words ? __ldcs(packed + i) : 0u;
        s[u] = i < words ? __ldg(scales + (i >> 2)) : 0.0f;  // a row has K / 8 words and K / 32 scales
    }
    pdl_wait();  // the scratch may still be read by the launch before
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const long long i = i0 + u * 256;
        if (i >= words) break;
        __half2 s_hi, s_lo;
        split_scale_f16(s[u] * cs, s_hi, s_lo);
        uint4 h, l;
        gg_dequant<LO ? 2 : 1>(q[u], s_hi, s_lo, h, l);
        reinterpret_cast<uint4*>(hi)[i] = h;
        if constexpr (LO) reinterpret_cast<uint4*>(lo)[i] = l;
    }
}

// The least of the handle's column exponents, the one for its largest scale.
__global__ void __launch_bounds__(1024) min_exp_kernel(const int* __restrict__ col_exp, const float* __restrict__ scales,
                                                       int* __restrict__ out, int N, int groups) {
    __shared__ int red[32];
    int e = 1 << 20;
    for (int n = threadIdx.x; n < N; n += 1024) {
        bool zero = true;  // an all-zero column has no say (its exponent is 0)
        const float* s = scales + static_cast<size_t>(n) * groups;
        for (int g = 0; g < groups && zero; ++g) zero = s[g] == 0.0f;
        if (!zero) e = min(e, col_exp[n]);
    }
    for (int o = 16; o > 0; o >>= 1) e = min(e, __shfl_xor_sync(0xffffffffu, e, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = e;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 32; ++i) e = min(e, red[i]);
        *out = e == (1 << 20) ? 0 : e;
    }
}

// Row statistics of the tiles' (log2 units, target excluded) and the target's
// logit: row max M2 with the target, S = sum over tiles of sums * 2^(tile max -
// M2) + 2^(target - M2), the factor 2^(tile max - M2) of every tile in place of
// its max, lse and loss.  The loss of a likely target is log1p(others /
// target), which does not cancel.  ROWS rows x 1024 / ROWS threads per block: 4
// rows of few, whose tiles a few blocks would walk in turn, 32 of many, for
// whole lines (32 rows of 391 tiles of 128 columns: 8.5 us with 4, 21 with 32;
// 50000 columns in tiles of 256: 1024 rows 7.7 and 12.5 us, 2048 rows 12.6 and
// 12.7, 4096 rows 19.8 and 12.7).
constexpr int kLossRowsFew = 1024;
template <int ROWS>
__global__ void __launch_bounds__(1024) loss_rows_kernel(float* smax, const float* ssum, const float* zt,
                                                         const long long* targets,
                                                         float* __restrict__ total, float* __restrict__ loss,
                                                         float* __restrict__ lse, int M, int N, int tiles, int parts,
                                                         long long ld) {
    constexpr int kParts = 1024 / ROWS;
    __shared__ float red[32][ROWS];
    pdl_launch_dependents();
    pdl_wait();
    smax = after_wait(smax);
    ssum = after_wait(ssum);
    zt = after_wait(zt);
    targets = after_wait(targets);
    const int r = threadIdx.x % ROWS, p = threadIdx.x / ROWS, warp = threadIdx.x >> 5;
    const int row = blockIdx.x * ROWS + r;
    const bool in = row < M;
    const long long t = in ? targets[row] : -1;
    const float t2 = t >= 0 && t < N ? zt[row] * 1.4426950408889634f : -INFINITY;
    float top = t2;
#pragma unroll 4
    for (int i = p; i < tiles && in; i += kParts) top = fmaxf(top, smax[static_cast<size_t>(i) * ld + row]);
    for (int o = 16; o >= ROWS; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    red[warp][r] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, red[i][r]);
    __syncthreads();
    float sum = 0.0f;
#pragma unroll 4
    for (int i = p; i < tiles && in; i += kParts) {
        float* at = smax + static_cast<size_t>(i) * ld + row;
        const float f = exp2f(*at - top);
        const float* st = ssum + static_cast<size_t>(parts * i) * ld + row;
        float all = st[0] + st[ld];
        if (parts == 4) all += st[2 * ld] + st[3 * ld];
        sum += f * all;
        *at = f;
    }
    for (int o = 16; o >= ROWS; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    red[warp][r] = sum;
    __syncthreads();
    if (p != 0 || !in) return;
    for (int i = 1; i < 32; ++i) sum += red[i][r];
    const float et = exp2f(t2 - top), all = sum + et;
    total[row] = all;
    const float l = 0.69314718055994531f * (top + log2f(all));
    if (lse != nullptr) lse[row] = l;
    loss[row] = t < 0 ? 0.0f : t >= N ? NAN : et > 0.0009765625f ? log1pf(sum / et) : l - zt[row];
}

// dx[row][k] = g (sum_z partial[z][row][k] / S + (p_t - 1) w(k, target)), p_t - 1 =
// expm1(-loss); one block per row.
template <typename T>
__global__ void __launch_bounds__(256) loss_dx_kernel(const float* partial, int splits, long long out_rows,
                                                      const float* total, const float* loss,
                                                      const long long* targets, const float* row_scale,
                                                      const uint32_t* __restrict__ packed,
                                                      const float* __restrict__ scales, T* __restrict__ dx, int N, int K) {
    pdl_launch_dependents();
    pdl_wait();
    partial = after_wait(partial);
    total = after_wait(total);
    loss = after_wait(loss);
    targets = after_wait(targets);
    row_scale = after_wait(row_scale);
    const long long row = blockIdx.x;
    const long long t = targets[row];
    T* out = dx + row * K;
    const float g = row_scale != nullptr ? row_scale[row] : 1.0f;
    const float inv = 1.0f / total[row], hot = expm1f(-loss[row]);
    for (int k = threadIdx.x * 8; k < K; k += 256 * 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        if (t >= 0) {
            const bool in = t < N;  // the target's weights are on their way while the splits are added
            const uint32_t q = in ? __ldg(packed + t * (K / 8) + k / 8) : 0u;
            const float s = in ? __ldg(scales + t * (K / 32) + k / 32) : 0.0f;
#pragma unroll 4
            for (int z = 0; z < splits; ++z) {
                const float4* p = reinterpret_cast<const float4*>(partial + (z * out_rows + row) * K + k);
                const float4 a = p[0], b = p[1];
                v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
                v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
            }
            if (in) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int nib = static_cast<int>((q >> (4 * i)) & 15u);
                    v[i] = g * (v[i] * inv + hot * (static_cast<float>((nib ^ 8) - 8) * s));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = NAN;
            }
        }
        if constexpr (std::is_same<T, float>::value) {
            reinterpret_cast<float4*>(out + k)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(out + k)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                o[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(out + k) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// out[i] = sum in order of the splits' partial[z][i], four floats per thread.
template <typename T>
__global__ void __launch_bounds__(256) sum_splits_kernel(const float* partial, int splits, long long split_floats,
                                                         T* __restrict__ out, long long quads) {
    pdl_launch_dependents();
    pdl_wait();
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= quads) return;
    const float4* p = reinterpret_cast<const float4*>(after_wait(partial)) + i;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int z = 0; z < splits; ++z) {
        const float4 a = p[z * (split_floats / 4)];
        v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
    }
    if constexpr (std::is_same<T, float>::value) {
        reinterpret_cast<float4*>(out)[i] = v;
    } else {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
        reinterpret_cast<uint2*>(out)[i] =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
}

constexpr int kGgNoColumn = -512;  // 2^-512 of any finite fp32 value is 0
// One block per rank j < 64: f16 planes [planes][64][ld] of A^T's row j times
// 2^E_j, E_j such that its largest magnitude lies in [2^13, 2^14) (k in the
// dequantised words' order, zeros past K and past the rank), and the exponent
// w_exp - E_j that G's column j carries in exchange.
__global__ void __launch_bounds__(256) lora_at_kernel(const float* a, __half* __restrict__ at,
                                                      int* __restrict__ gexp, const int* __restrict__ w_exp, int K,
                                                      int rank, int ld, int planes) {
    __shared__ float red[8];
    pdl_launch_dependents();
    pdl_wait();  // A may come from an optimizer step, the planes may still be read
    a = after_wait(a);
    const int j = blockIdx.x;
    float top = 0.0f;
    if (j < rank) {
#pragma unroll 8
        for (int k = threadIdx.x; k < K; k += 256) top = fmaxf(top, fabsf(a[static_cast<size_t>(k) * rank + j]));
    }
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int i = 0; i < 8; ++i) top = fmaxf(top, red[i]);
    int e = 0;
    if (top > 0.0f && isfinite(top)) {
        int e2;
        frexpf(top, &e2);
        e = min(max(14 - e2, -120), 120);
    }
    // a column of zeros: G's column, which meets nothing, shrinks to 0 and has no say in its row's exponent
    if (threadIdx.x == 0) gexp[j] = top > 0.0f ? *w_exp - e : kGgNoColumn;
    const float s = exp2i(e);
#pragma unroll 4
    for (int i = threadIdx.x; i < ld; i += 256) {
        const int k = (i & ~7) + (i & 1) * 4 + ((i & 7) >> 1);  // place i holds k
        const float v = j < rank && k < K ? a[static_cast<size_t>(k) * rank + j] * s : 0.0f;
        const __half h = __float2half_rn(v);
        at[static_cast<size_t>(j) * ld + i] = h;
        if (planes == 2) at[static_cast<size_t>(64 + j) * ld + i] = __float2half_rn(v - __half2float(h));
    }
}

}  // namespace

int grad_gemm_pairs() { return gg_pairs<true, 1, 1, kGgBf16, false>(); }

int launch_grad_gemm(const GradGemmArgs& a, int planes, int epi, bool from_planes, cudaStream_t stream) {
    if (from_planes && planes != 1) return static_cast<int>(cudaErrorInvalidValue);
    switch (epi) {
        case kGgLoss:
            return from_planes   ? gg_launch<false, 1, 2, kGgLoss, true>(a, stream)
                   : planes == 1 ? gg_launch<false, 1, 2, kGgLoss, false>(a, stream)
                                 : gg_launch<false, 2, 2, kGgLoss, false>(a, stream);
        case kGgProb:
            return from_planes   ? gg_launch<false, 1, 2, kGgProb, true>(a, stream)
                   : planes == 1 ? gg_launch<false, 1, 2, kGgProb, false>(a, stream)
                                 : gg_launch<false, 2, 2, kGgProb, false>(a, stream);
        case kGgF32:
            return from_planes   ? gg_launch<true, 1, 1, kGgF32, true>(a, stream)
                   : planes == 1 ? gg_launch<true, 1, 1, kGgF32, false>(a, stream)
                                 : gg_launch<true, 2, 2, kGgF32, false>(a, stream);
        case kGgBf16:
            if (planes != 1) break;
            return from_planes ? gg_launch<true, 1, 1, kGgBf16, true>(a, stream)
                               : gg_launch<true, 1, 1, kGgBf16, false>(a, stream);
    }
    return static_cast<int>(cudaErrorInvalidValue);
}

int launch_weight_planes(const uint32_t* packed, const float* scales, const int* w_exp, void* hi, void* lo, int N, int K,
                         cudaStream_t stream) {
    const long long words = static_cast<long long>(N) * (K / 8);
    const unsigned blocks = static_cast<unsigned>((words + 1023) / 1024);
    auto kern = lo == nullptr ? weight_planes_kernel<false> : weight_planes_kernel<true>;
    return gg_launch_pdl(kern, blocks, 256, stream, packed, scales, w_exp, static_cast<__half*>(hi),
                         static_cast<__half*>(lo), words);
}

int launch_cast_planes(const CastArgs& a, bool bf16, int planes, cudaStream_t stream) {
    if (a.M < 1 || a.ld % 8 != 0 || a.ld < a.cols || a.rank > 64) return static_cast<int>(cudaErrorInvalidValue);
    const bool vec = a.cols % 8 == 0;  // rows of whole 16-byte pieces
    if (!vec && (a.targets != nullptr || a.by_word)) return static_cast<int>(cudaErrorInvalidValue);
    const unsigned grid = static_cast<unsigned>(a.M);
    auto launch = [&](auto few, auto wide, auto one, auto two) {
        return a.M <= kCastFew ? (vec ? gg_launch_pdl(few, grid, kCastThreadsFew, stream, a)
                                      : gg_launch_pdl(wide, grid, kCastThreadsFew, stream, a))
                               : (vec ? gg_launch_pdl(one, grid, kCastThreads, stream, a)
                                      : gg_launch_pdl(two, grid, kCastThreads, stream, a));
    };
    if (bf16)
        return launch(cast_planes_kernel<__nv_bfloat16, 1, true, kCastThreadsFew>,
                      cast_planes_kernel<__nv_bfloat16, 1, false, kCastThreadsFew>,
                      cast_planes_kernel<__nv_bfloat16, 1, true, kCastThreads>,
                      cast_planes_kernel<__nv_bfloat16, 1, false, kCastThreads>);
    if (planes == 2)
        return launch(cast_planes_kernel<float, 2, true, kCastThreadsFew>, cast_planes_kernel<float, 2, false, kCastThreadsFew>,
                      cast_planes_kernel<float, 2, true, kCastThreads>, cast_planes_kernel<float, 2, false, kCastThreads>);
    return static_cast<int>(cudaErrorInvalidValue);
}

int launch_min_exp(const int* col_exp, const float* scales, int* out, int N, int K, cudaStream_t stream) {
    min_exp_kernel<<<1, 1024, 0, stream>>>(col_exp, scales, out, N, K / 32);
    return static_cast<int>(cudaGetLastError());
}

int launch_loss_rows(float* smax, const float* ssum, const float* zt, const long long* targets, float* total,
                     float* loss, float* lse, int M, int N, int tiles, int parts, long long ld, cudaStream_t stream) {
    auto launch = [&](auto kern, int rows) {
        return gg_launch_pdl(kern, static_cast<unsigned>((M + rows - 1) / rows), 1024, stream, smax, ssum, zt, targets, total,
                             loss, lse, M, N, tiles, parts, ld);
    };
    return M <= kLossRowsFew ? launch(loss_rows_kernel<4>, 4) : launch(loss_rows_kernel<32>, 32);
}

int launch_loss_dx(const float* partial, int splits, long long out_rows, const float* total, const float* loss,
                   const long long* targets, const float* row_scale, const uint32_t* packed, const float* scales, void* dx,
                   bool bf16, int M, int N, int K, cudaStream_t stream) {
    if (bf16)
        return gg_launch_pdl(loss_dx_kernel<__nv_bfloat16>, static_cast<unsigned>(M), 256, stream, partial, splits, out_rows,
                             total, loss, targets, row_scale, packed, scales, static_cast<__nv_bfloat16*>(dx), N, K);
    return gg_launch_pdl(loss_dx_kernel<float>, static_cast<unsigned>(M), 256, stream, partial, splits, out_rows, total, loss,
                         targets, row_scale, packed, scales, static_cast<float*>(dx), N, K);
}

int launch_sum_splits(const float* partial, int splits, long long split_floats, void* out, bool bf16, long long count,
                      cudaStream_t stream) {
    const long long quads = count / 4, blocks = (quads + 255) / 256;
    if (count % 4 != 0 || split_floats % 4 != 0 || blocks > (1ll << 30)) return static_cast<int>(cudaErrorInvalidValue);
    if (bf16)
        return gg_launch_pdl(sum_splits_kernel<__nv_bfloat16>, static_cast<unsigned>(blocks), 256, stream, partial, splits,
                             split_floats, static_cast<__nv_bfloat16*>(out), quads);
    return gg_launch_pdl(sum_splits_kernel<float>, static_cast<unsigned>(blocks), 256, stream, partial, splits, split_floats,
                         static_cast<float*>(out), quads);
}

int launch_lora_at(const float* a, void* at, int* gexp, const int* w_exp, int K, int rank, int ld, int planes,
                   cudaStream_t stream) {
    return gg_launch_pdl(lora_at_kernel, 64, 256, stream, a, static_cast<__half*>(at), gexp, w_exp, K, rank, ld, planes);
}

}  // namespace q4
