// The two products of training through frozen int4 weights for a few rows (up
// to 64), one CTA per SM:
//
//   TR = false, logits:  z[m][n]  = sum_k x[m][k] w(k, n)    (softmax cross entropy)
//   TR = true:           dx[m][k] = sum_n d[m][n] w(k, n)    (input gradient)
//
// The same f16 planes, dequantisation and epilogues as the CTA-pair kernel of
// q4_grad_gemm.cu, but with the operands' roles exchanged: the 128 lanes of the
// accumulator are weights (128 n of the logits, 128 k of the transposed
// product) and the rows are the MMA's N, so that a few rows cost a few columns
// instead of a 256-row tile of zeros.  The rows' planes are stacked in N, [hi
// rows; lo rows], so that both meet the weights' hi plane in one MMA.
//
// The weights are then the MMA's A operand.  For the logits a thread's weights
// are one lane's (its n) and go from registers to tensor memory; the transposed
// product contracts over n and takes them from shared memory, MN-major (128 n x
// 128 k as two images of 128 rows of 128 bytes, 128-byte swizzled).  With the
// logits' operand in shared memory too, the fp32 loss of 32 x 2048 x 50000 (its
// cast and statistics included, calls in a loop) took 72 us instead of 62.
//
// What bounds it is the dequantisation beside everything else an SM issues: a
// block of 128 n x 128 k takes about 1600 cycles (logits) or 1900 (transposed,
// fp32), with 60% and 57% of the issue slots, a fifth of the tensor pipe and a
// quarter of HBM's bandwidth in use (32 x 2048 x 50000: 48 and 53 us by ncu, one launch).  Tried and slower: stages of half a block,
// a second MMA warp with an accumulator per block, one lane per warp polling.
//
// Roles (28 warps): warp 0 loads the rows' planes, warp 2 packed words and
// scales (TMA), warp 1 issues the MMAs (M = 128, K = 16), warps 4-11 hold the
// sums (thread = lane of the accumulator, half of the rows each) and run the
// epilogue, warps 12-27 dequantise: two groups of eight take the blocks of 128 x
// 128 in turn.  The numbers of slots are even, so a slot belongs to one group,
// which sees every phase of its barriers.  Every wait is bounded (status word +
// abort flag).
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "q4_dequant.cuh"
#include "q4_grad.cuh"
#include "q4_kernels.h"

namespace q4 {

namespace {

constexpr int kFrPlane = 128 * 128 * 2;  // one f16 plane of a block in shared memory: [2 halves of k][128 n][64 k]
constexpr int kFrEpiWarp0 = 4, kFrEpiWarps = 8, kFrDeqWarp0 = 12, kFrGroupWarps = 8;
constexpr int kFrThreads = 32 * (kFrDeqWarp0 + 2 * kFrGroupWarps);

// RP: padded rows; PA, PB: planes of the rows and of the weights.
template <bool TR, int RP, int PA, int PB>
struct FrCfg {
    static constexpr int kHalf = PA * RP * 128;  // PA * RP rows of 64 of the contraction
    static constexpr int kXBytes = 2 * kHalf;
    static constexpr int kAcc = 2 * PA * RP;       // tensor memory columns of the two accumulators
    // Slots of the weights' blocks: 128 KB of shared memory, or two of PB * 64 columns of tensor memory.
    static constexpr int kWBytes = TR ? PB * kFrPlane : 0;
    static constexpr int kW = TR ? 131072 / kWBytes : 2;
    static constexpr int kRaw = !TR ? 8 : kXBytes > 16384 ? 2 : 4;
    // The rows get what 223 KB leave: their loads have the latency of L2 to hide.
    static constexpr int kX0 = (228352 - kW * kWBytes - kRaw * kGgRawBytes) / kXBytes, kX = kX0 < 8 ? kX0 : 8;
    static_assert(kW % 2 == 0 && kRaw % 2 == 0 && kX >= 2, "a slot of weights belongs to one dequant group");
    static constexpr int kXOff = kW * kWBytes;
    static constexpr int kRawOff = kXOff + kX * kXBytes;
    static constexpr int kRedOff = kRawOff + kRaw * kGgRawBytes;  // [2 buffers][4 quarters][RP] floats
    static constexpr int kBarOff = kRedOff + 2 * 4 * RP * 4;
    // full_x[X], empty_x[X], full_w[W], empty_w[W], full_r[R], empty_r[R], acc_full[2], acc_empty[2], xch[2], done
    static constexpr int kNumBars = 2 * (kX + kW + kRaw) + 7;
    static constexpr int kMiscOff = kBarOff + kNumBars * 8;
    static constexpr int kSmem = kMiscOff + 16 + 1024;
    static_assert(kSmem <= 232448, "shared memory budget");
    static constexpr int kTmemUsed = kAcc + (TR ? 0 : kW * PB * 64);
    static constexpr uint32_t kTmemCols = kTmemUsed <= 64 ? 64 : kTmemUsed <= 128 ? 128 : kTmemUsed <= 256 ? 256 : 512;
    static_assert(kTmemUsed <= 512, "tensor memory");
};

struct FrUnit {
    int tile, z, c0, c1;  // 128 lanes, split, chunks [c0, c1)
};
__device__ __forceinline__ FrUnit fr_unit(const FewRowsArgs& P, int u) {
    FrUnit w;
    w.tile = u % P.tiles;
    w.z = u / P.tiles;
    w.c0 = static_cast<int>(static_cast<long long>(w.z) * P.chunks / P.splits);
    w.c1 = static_cast<int>(static_cast<long long>(w.z + 1) * P.chunks / P.splits);
    return w;
}

// Over the warp's lanes, each of V values' maximum or sum: lane l ends with
// value value_index<V>(l).  The first step reads `v` and leaves it.
template <int V, bool MAX>
__device__ __forceinline__ float fr_reduce(const float (&v)[V], int lane) {
    auto both = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
    float t[V / 2];
    const bool up = (lane & 16) != 0;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const float send = up ? v[i] : v[i + V / 2], keep = up ? v[i + V / 2] : v[i];
        t[i] = both(keep, __shfl_xor_sync(0xffffffffu, send, 16));
    }
    int bit = 8;
#pragma unroll
    for (int half = V / 4; half >= 1; half >>= 1, bit >>= 1) {
        const bool hi = (lane & bit) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float send = hi ? t[i] : t[i + half], keep = hi ? t[i + half] : t[i];
            t[i] = both(keep, __shfl_xor_sync(0xffffffffu, send, bit));
        }
    }
    for (; bit >= 1; bit >>= 1) t[0] = both(t[0], __shfl_xor_sync(0xffffffffu, t[0], bit));
    return t[0];
}

template <bool TR, int RP, int PA, int PB, int EPI>
__global__ void __launch_bounds__(kFrThreads, 1) few_rows_kernel(const __grid_constant__ FewRowsArgs P) {
    using C = FrCfg<TR, RP, PA, PB>;
    constexpr int SX = C::kX, SW = C::kW, R = C::kRaw, NC = PA * RP;
    static_assert(TR || PB == 2, "the logits take hi and lo of the weights");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_base = smem_u32(smem_raw), base = (raw_base + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_base);
    const uint32_t bar = base + C::kBarOff;
    auto full_x = [&](int s) { return bar + 8u * s; };
    auto empty_x = [&](int s) { return bar + 8u * (SX + s); };
    auto full_w = [&](int s) { return bar + 8u * (2 * SX + s); };
    auto empty_w = [&](int s) { return bar + 8u * (2 * SX + SW + s); };
    auto full_r = [&](int r) { return bar + 8u * (2 * SX + 2 * SW + r); };
    auto empty_r = [&](int r) { return bar + 8u * (2 * SX + 2 * SW + R + r); };
    const uint32_t bar2 = bar + 8u * (2 * (SX + SW + R));
    auto acc_full = [&](int b) { return bar2 + 8u * b; };
    auto acc_empty = [&](int b) { return bar2 + 8u * (2 + b); };
    auto xch_bar = [&](int h) { return bar2 + 8u * (4 + h); };
    const uint32_t done_bar = bar2 + 8u * 6;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kMiscOff);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kMiscOff + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int units = P.tiles * P.splits;
    int* status = P.status;
    if (tid == 0) {
        for (int s = 0; s < SX; ++s) {
            mbar_init(full_x(s), 1);
            mbar_init(empty_x(s), 1);
        }
        for (int s = 0; s < SW; ++s) {
            mbar_init(full_w(s), kFrGroupWarps);
            mbar_init(empty_w(s), 1);
        }
        for (int r = 0; r < R; ++r) {
            mbar_init(full_r(r), 1);
            mbar_init(empty_r(r), kFrGroupWarps);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), kFrEpiWarps);
            mbar_init(xch_bar(b), 4);  // the four warps of one half of the rows
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&P.tm_a);
        tma_prefetch_desc(&P.tm_w);
        tma_prefetch_desc(&P.tm_s);
    }
    if (warp == 3) {
        tmem_alloc(smem_u32(tmem_holder), C::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_holder;
    pdl_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            // ------------------------------------------------ row planes --
            pdl_wait();
            int q = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
                const FrUnit w = fr_unit(P, u);
                const int b1 = min(w.c1 * P.chunk, P.blocks);
                for (int b = w.c0 * P.chunk; b < b1; ++b, ++q) {
                    const int s = q % SX;
                    if (!gg_wait(empty_x(s), ((q / SX) & 1u) ^ 1u, abort_flag, status, kStatusTimeoutProducer)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = base + C::kXOff + s * C::kXBytes;
                    mbar_arrive_expect_tx(full_x(s), C::kXBytes);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int p = 0; p < PA; ++p)  // past the row, or the plane: zeros, or columns that nothing reads
                            tma_load_2d(dst + h * C::kHalf + p * RP * 128, &P.tm_a, full_x(s), b * 128 + h * 64, p * P.M);
                }
            }
            if (*abort_flag)
                for (int j = q > SX ? q - SX : 0; j < q; ++j) mbar_drain(full_x(j % SX), (j / SX) & 1u);
        }
        __syncwarp();
    } else if (warp == 2) {
        if (lane == 0) {
            // ---------------------------------------------- raw weights --
            int q = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
                const FrUnit w = fr_unit(P, u);
                const int b1 = min(w.c1 * P.chunk, P.blocks);
                for (int b = w.c0 * P.chunk; b < b1; ++b, ++q) {
                    const int r = q % R;
                    if (!gg_wait(empty_r(r), ((q / R) & 1u) ^ 1u, abort_flag, status, kStatusTimeoutProducer)) {
                        ok = false;
                        break;
                    }
                    const int k0 = (TR ? w.tile : b) * 128, n0 = (TR ? b : w.tile) * 128;
                    const uint32_t dst = base + C::kRawOff + r * kGgRawBytes;
                    mbar_arrive_expect_tx(full_r(r), kGgRawBytes);
                    tma_load_2d(dst, &P.tm_w, full_r(r), k0 / 8, n0);
                    tma_load_2d(dst + kGgRawWords, &P.tm_s, full_r(r), k0 / 32, n0);
                }
            }
            if (*abort_flag)
                for (int j = q > R ? q - R : 0; j < q; ++j) mbar_drain(full_r(j % R), (j / R) & 1u);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            // ------------------------------------------------------- MMA --
            constexpr uint32_t major = TR ? (1u << 15) : 0u;  // A: MN-major
            constexpr uint32_t idesc = umma_idesc_f16(0u, 128, NC) | major, idesc_lo = umma_idesc_f16(0u, 128, RP) | major;
            int x = 0, s = 0, b = 0;           // slots, and the parities to wait for: counted along, not divided out
            uint32_t xp = 0, sp = 0, ap = 1;
            bool ok = true;
            for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
                const FrUnit w = fr_unit(P, u);
                int i = w.c0 * P.chunk;
                const int end = min(w.c1 * P.chunk, P.blocks);
                while (i < end && ok) {
                    if (!gg_wait(acc_empty(b), ap, abort_flag, status, kStatusTimeoutMma)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t dacc = tmem + static_cast<uint32_t>(b * NC);
                    uint32_t acc = 0;
                    for (const int stop = min(i + P.chunk, end); i < stop; ++i) {
                        if (!gg_wait(full_w(s), sp, abort_flag, status, kStatusTimeoutMma) ||
                            !gg_wait(full_x(x), xp, abort_flag, status, kStatusTimeoutMma)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
                        [[maybe_unused]] const uint32_t at = base + s * C::kWBytes;
                        const uint32_t bt = base + C::kXOff + x * C::kXBytes;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint64_t bd = umma_desc_k_sw128(bt + (j >> 2) * C::kHalf + (j & 3) * 32);
                            if constexpr (TR) {
                                umma_f16_ss(dacc, gg_desc_mn_sw128(at + j * 2048, kFrPlane / 2), bd, idesc, j > 0 ? 1u : acc);
                                if constexpr (PB == 2)
                                    umma_f16_ss(dacc, gg_desc_mn_sw128(at + kFrPlane + j * 2048, kFrPlane / 2), bd, idesc_lo,
                                                1u);
                            } else {
                                // a scale group (32 k) is 16 columns of hi, then 16 of lo
                                const uint32_t a = tmem + static_cast<uint32_t>(C::kAcc + s * 128 + (j >> 1) * 32 + (j & 1) * 8);
                                umma_f16_ts(dacc, a, bd, idesc, j > 0 ? 1u : acc);
                                umma_f16_ts(dacc, a + 16, bd, idesc_lo, 1u);
                            }
                        }
                        umma_commit(empty_w(s));
                        umma_commit(empty_x(x));
                        acc = 1;
                        if (++x == SX) x = 0, xp ^= 1u;
                        if (++s == SW) s = 0, sp ^= 1u;
                    }
                    if (ok) umma_commit(acc_full(b));
                    b ^= 1;
                    if (b == 0) ap ^= 1u;
                }
            }
            umma_commit(done_bar);  // tracks every MMA issued above
            mbar_drain(done_bar, 0u);
        }
        __syncwarp();
    } else if (warp >= kFrDeqWarp0) {
        // ------------------------------------------------------- dequant --
        // Thread t of a group: n = t % 128 of the block, 64 k t / 128: two scale groups (32 k) of one n.
        const int group = (warp - kFrDeqWarp0) / kFrGroupWarps;
        const int t = tid - (kFrDeqWarp0 + group * kFrGroupWarps) * 32, row = t & 127, kh = t >> 7;
        const float cs = exp2i(*P.w_exp);
        const int rkey = (row >> 1) & 3;
        const uint32_t at0 = static_cast<uint32_t>(row * 64 + (((2 * kh) ^ rkey) << 4));
        const uint32_t at1 = static_cast<uint32_t>(row * 64 + (((2 * kh + 1) ^ rkey) << 4));
        const uint32_t ats = static_cast<uint32_t>(kGgRawWords + row * 16 + kh * 8);
        int q = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
            const FrUnit w = fr_unit(P, u);
            const int b1 = min(w.c1 * P.chunk, P.blocks);
            for (int b = w.c0 * P.chunk; b < b1; ++b, ++q) {
                if ((q & 1) != group) continue;
                const int r = q % R, s = q % SW;
                if (!gg_wait_warp(full_r(r), (q / R) & 1u, abort_flag, status, kStatusTimeoutDequant)) {
                    ok = false;
                    break;
                }
                const uint8_t* raw = smem + C::kRawOff + r * kGgRawBytes;
                const uint4 words[2] = {*reinterpret_cast<const uint4*>(raw + at0),
                                        *reinterpret_cast<const uint4*>(raw + at1)};
                const float2 sc = *reinterpret_cast<const float2*>(raw + ats);
                __syncwarp();
                if (lane == 0) mbar_arrive(empty_r(r));
                if (!gg_wait_warp(empty_w(s), ((q / SW) & 1u) ^ 1u, abort_flag, status, kStatusTimeoutDequant)) {
                    ok = false;
                    break;
                }
                if constexpr (!TR) tc_fence_after_sync();  // the MMAs that last read this slot have completed
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    __half2 s_hi, s_lo;
                    split_scale_f16((h == 0 ? sc.x : sc.y) * cs, s_hi, s_lo);
                    const uint32_t ww[4] = {words[h].x, words[h].y, words[h].z, words[h].w};
                    if constexpr (TR) {
                        uint8_t* dst = smem + s * C::kWBytes + kh * (kFrPlane / 2) + row * 128;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 hi, lo;
                            gg_dequant<PB>(ww[i], s_hi, s_lo, hi, lo);
                            const int o = ((4 * h + i) ^ (row & 7)) << 4;
                            *reinterpret_cast<uint4*>(dst + o) = hi;
                            if constexpr (PB == 2) *reinterpret_cast<uint4*>(dst + kFrPlane + o) = lo;
                        }
                    } else {
                        uint32_t v[32];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 hi, lo;
                            gg_dequant<2>(ww[i], s_hi, s_lo, hi, lo);
                            v[4 * i] = hi.x; v[4 * i + 1] = hi.y; v[4 * i + 2] = hi.z; v[4 * i + 3] = hi.w;
                            v[16 + 4 * i] = lo.x; v[17 + 4 * i] = lo.y; v[18 + 4 * i] = lo.z; v[19 + 4 * i] = lo.w;
                        }
                        tmem_st32(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) +
                                      static_cast<uint32_t>(C::kAcc + s * 128 + (2 * kh + h) * 32), v);
                    }
                }
                if constexpr (TR) {
                    fence_proxy_async_smem();
                } else {
                    tmem_st_wait();
                    tc_fence_before_sync();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(full_w(s));
            }
        }
    } else if (warp >= kFrEpiWarp0) {
        // ------------------------------------------------------ epilogue --
        constexpr int RH = RP / 2;  // rows of this thread: r0 .. r0 + RH - 1; lane l % RH also keeps row r0 + l's constants
        const int quarter = warp & 3, half = (warp - kFrEpiWarp0) >> 2, r0 = half * RH, mine = r0 + lane % RH;
        const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(r0);
        const int wexp = *P.w_exp;
        pdl_wait();
        const int rexp = P.row_exp != nullptr ? (mine < P.M ? after_wait(P.row_exp)[mine] : 0) : P.fixed_exp;
        const int e = -(rexp + wexp);
        const float scale = exp2i(e / 2) * exp2i(e - e / 2);
        int cq = 0, xq = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
            const FrUnit w = fr_unit(P, u);
            float acc[RH];
#pragma unroll
            for (int i = 0; i < RH; ++i) acc[i] = 0.0f;
            for (int c = w.c0; c < w.c1; ++c, ++cq) {
                const int b = cq & 1;
                float f = 1.0f;
                if (TR && P.coef != nullptr) f = after_wait(P.coef)[static_cast<size_t>(c) * P.ld_stat + mine];
                if (!gg_wait_warp(acc_full(b), (cq >> 1) & 1u, abort_flag, status, kStatusTimeoutEpilogue)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
#pragma unroll
                for (int i = 0; i < RH; i += 16) {
                    uint32_t v[16];
                    tmem_ld16(t_lane + static_cast<uint32_t>(b * NC + i), v);
                    gg_ld_wait(v);
                    if constexpr (PA == 2) {  // rows' lo against the weights' hi
                        uint32_t l[16];
                        tmem_ld16(t_lane + static_cast<uint32_t>(b * NC + RP + i), l);
                        gg_ld_wait(l);
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(l[j]));
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float fj = TR ? __shfl_sync(0xffffffffu, f, i + j) : 1.0f;
                        acc[i + j] = fmaf(fj, __uint_as_float(v[j]), acc[i + j]);
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(b));
            }
            if (!ok) break;
            const int col = w.tile * 128 + quarter * 32 + lane;
            if constexpr (TR) {
                // the accumulator's lanes hold each 8 k in the order 0 4 1 5 2 6 3 7
                const int k = (col & ~7) | ((col & 1) << 2) | ((col & 7) >> 1);
                float* out = static_cast<float*>(P.out) + static_cast<long long>(w.z) * P.M * P.K + k;
#pragma unroll
                for (int i = 0; i < RH; ++i) {
                    const float v = acc[i] * __shfl_sync(0xffffffffu, scale, i);
                    if (r0 + i < P.M && k < P.K) out[static_cast<long long>(r0 + i) * P.K] = v;
                }
            } else {
                // In units of log2, without the columns that do not exist and the target's
                // (whose logit the cast has from an fp32 product): the maximum over
                // the tile's 128 columns, terms 2^(z2 - max) and their sums.
                const long long tgt = mine < P.M ? after_wait(P.targets)[mine] : -1;
                const int tcol = tgt >= w.tile * 128ll && tgt < w.tile * 128ll + 128 ? static_cast<int>(tgt) : -1;
                const float s2 = scale * 1.4426950408889634f;
#pragma unroll
                for (int i = 0; i < RH; ++i) {
                    const float si = __shfl_sync(0xffffffffu, s2, i);
                    const int ti = __shfl_sync(0xffffffffu, tcol, i);
                    acc[i] = col < P.N && col != ti ? acc[i] * si : -INFINITY;
                }
                // a buffer that alternates: a warp writes one again only after its partners have arrived for the other
                float* red = reinterpret_cast<float*>(smem + C::kRedOff) + (xq & 1) * 4 * RP;
                red[quarter * RP + r0 + value_index<RH>(lane)] = fr_reduce<RH, true>(acc, lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(xch_bar(half));
                if (!gg_wait_warp(xch_bar(half), xq & 1u, abort_flag, status, kStatusTimeoutEpilogue)) {
                    ok = false;
                    break;
                }
                ++xq;
                const float top = fmaxf(fmaxf(red[mine], red[RP + mine]), fmaxf(red[2 * RP + mine], red[3 * RP + mine]));
                const float ref = top == -INFINITY ? 0.0f : top;  // a tile of the target alone: all terms 0
#pragma unroll
                for (int i = 0; i < RH; ++i) {
                    acc[i] = ex2(acc[i] - __shfl_sync(0xffffffffu, ref, i));  // 2^-inf = 0 where there is no term
                    if constexpr (EPI == kGgProb) {
                        __half* out = static_cast<__half*>(P.out) + static_cast<long long>(r0 + i) * P.ld_out + col;
                        if (r0 + i < P.M) {
                            const float v = acc[i] * 16384.0f;
                            const __half h = __float2half_rn(v);
                            *out = h;
                            if constexpr (PA == 2)
                                out[static_cast<long long>(P.M) * P.ld_out] = __float2half_rn(v - __half2float(h));
                        }
                    }
                }
                const float sum = fr_reduce<RH, false>(acc, lane);
                if (quarter == 0 && lane < RH) P.smax[static_cast<size_t>(w.tile) * P.ld_stat + mine] = top;
                P.ssum[(static_cast<size_t>(w.tile) * 4 + quarter) * P.ld_stat + r0 + value_index<RH>(lane)] = sum;
            }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, C::kTmemCols);
    }
}

template <bool TR, int RP, int PA, int PB, int EPI>
int fr_launch(const FewRowsArgs& a, cudaStream_t stream) {
    using C = FrCfg<TR, RP, PA, PB>;
    auto kern = few_rows_kernel<TR, RP, PA, PB, EPI>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    const long long units = static_cast<long long>(a.tiles) * a.splits;
    if (a.sm_count < 1 || a.M < 1 || a.M > RP || units < 1 || units > (1ll << 30))
        return static_cast<int>(cudaErrorInvalidConfiguration);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(units < a.sm_count ? units : a.sm_count));
    cfg.blockDim = dim3(kFrThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, a));
}

template <int RP>
int fr_dispatch(const FewRowsArgs& a, int planes, bool logits, int epi, cudaStream_t stream) {
    if (!logits)
        return planes == 1 ? fr_launch<true, RP, 1, 1, kGgF32>(a, stream) : fr_launch<true, RP, 2, 2, kGgF32>(a, stream);
    if (epi == kGgProb)
        return planes == 1 ? fr_launch<false, RP, 1, 2, kGgProb>(a, stream) : fr_launch<false, RP, 2, 2, kGgProb>(a, stream);
    return planes == 1 ? fr_launch<false, RP, 1, 2, kGgLoss>(a, stream) : fr_launch<false, RP, 2, 2, kGgLoss>(a, stream);
}

}  // namespace

int few_rows_padded(int M) { return M <= 32 ? 32 : 64; }

int launch_few_rows(const FewRowsArgs& a, int planes, int epi, cudaStream_t stream) {
    const bool logits = epi == kGgLoss || epi == kGgProb;
    return few_rows_padded(a.M) == 32 ? fr_dispatch<32>(a, planes, logits, epi, stream)
                                      : fr_dispatch<64>(a, planes, logits, epi, stream);
}

}  // namespace q4
