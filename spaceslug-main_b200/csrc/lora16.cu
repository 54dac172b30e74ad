// LoRA adapter gradients whose wide operands are exact in bf16: X kept in 8
// bits (act8.cu: code * 2^e, 7 significant bits) and bf16 dY.  The same four
// contractions as lora_tc.cu,
//
//   T  = X A        [M x r]        G  = dY B^T      [M x r]
//   dB = s T^T dY   [r x N]        dA = s X^T G     [K x r]
//
// each D[R x r] = sum over l < L of Aop[row][l] * Bop[j][l], in two launches
// (T and G; dB and dA) of work units (128 rows of D, a range of l), with the
// partial sums added in a fixed order afterwards (deterministic).
//
// Against the fp32 form: the wide operand needs no hi / lo split, so a stage
// of 64 l is four MMAs (kind::f16 on bf16, M = 128, K = 16) instead of the
// sixteen of the TF32 passes, and X crosses HBM in a byte per value.  The narrow operand enters
// as three stacked bf16 planes (hi, mid, lo: 24 bits, exact), N = 3 RP, whose
// sums the epilogue adds.  So every product is exact and the sums are fp32:
// restarted every 64 l and added in registers, rounded to nearest.
//
// For ranks up to 16 an fp32 dY comes the same way (F32): its values as three
// bf16 planes in tensor memory, 32 + 6 KB and twelve MMAs per stage, so that T
// and G, dA and dB stay one launch each.  Higher ranks leave tensor memory no
// room for that; their dY goes through lora_tc.cu.  (M x K x N, rank, the whole
// backward in a CUDA graph this way and with lora_tc.cu: 128 x 64 x 256, 4: 12.9
// and 18.2 us; 7 x 4096 x 4096, 16: 21.0 and 27.2; 512 x 4096 x 4096: 23.6 and 32.1;
// 2048 x 4096 x 4096: 39.4 and 47.9; 4096 x 4096 x 11008: 109 and 115.)
//
//  - T and G read the wide operand with its rows as rows of D: TMA boxes of
//    128 rows x 64 l (bf16 128-byte swizzled, codes 64-byte swizzled).
//  - dB and dA read it transposed: boxes of 64 l x 128 contiguous rows of D.
//  - Eight split warps (two per tensor-memory lane quarter, alternate stages)
//    give each row of D to one thread, turn its 64 values into bf16 pairs in
//    registers (codes: the byte under 2^23's exponent, minus 2^23 + 128, times
//    the step; all exact) and store them as the MMA's A operand in tensor
//    memory, so the transposed form costs nothing extra.
// Every wait is bounded (status word + abort flag).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "common.cuh"
#include "q4_kernels.h"

namespace q4 {

namespace {

constexpr int kL16Rows = 128;     // rows of D per unit (the MMA's M)
constexpr int kL16L = 64;         // contraction elements per stage
constexpr int kL16Threads = 512;  // warps: 0 TMA, 1-2 MMA, 4-7 epilogue, 8-15 split
constexpr int kL16ATile = kL16Rows * kL16L * 2;

template <int RP, bool F32>
struct L16Cfg {
    static constexpr int kN = 3 * RP;
    static constexpr int kATile = F32 ? 2 * kL16ATile : kL16ATile;
    static constexpr int kBTile = kN * kL16L * 2;  // 128-byte rows: 6, 12 or 24 KB
    static constexpr int kStageBytes = kATile + kBTile;
    // tensor memory: two accumulator buffers of 3 RP columns, then per stage 32 columns (64 bf16) for each plane of Aop
    static constexpr int kACol = 2 * kN;
    static constexpr int kACols = F32 ? 96 : 32;
    static constexpr int kTmemStages = (512 - kACol) / kACols;
    static constexpr int kSmemStages = 200 * 1024 / kStageBytes;
    static constexpr int kStages0 = kSmemStages < kTmemStages ? kSmemStages : kTmemStages;
    // even: a slot then belongs to one group of split warps and one MMA warp,
    // which see each of its phases (a parity only tells two successive ones apart)
    static constexpr int kStages = (kStages0 > 8 ? 8 : kStages0) / 2 * 2;
    static_assert(kStages > 2, "the epilogue waits on the stages' commits: it must not fall a phase behind");
    static constexpr int kStepOff = kStages * kStageBytes;      // 8 split warps x 64 steps
    static constexpr int kBarOff = kStepOff + 8 * 64 * 4;
    static constexpr int kNumBars = 3 * kStages + 2;            // full, split, empty; chunk_empty[2]
    static constexpr int kSmem = kBarOff + kNumBars * 8 + 16;
    static constexpr int kSmemAlloc = kSmem + 1024;
    static_assert(kSmemAlloc <= 232448, "shared memory budget");
};

struct L16Unit {
    int pi, tile, z, s0, s1;
};
__device__ __forceinline__ int l16_units(const Lora16Problem& q) { return (q.R + kL16Rows - 1) / kL16Rows * q.splits; }
__device__ __forceinline__ L16Unit l16_unit(const Lora16Pass& P, int u) {
    L16Unit w;
    const int u0 = l16_units(P.prob[0]);
    w.pi = (P.count > 1 && u >= u0) ? 1 : 0;
    const Lora16Problem& q = P.prob[w.pi];
    const int lu = w.pi ? u - u0 : u;
    const int tiles = (q.R + kL16Rows - 1) / kL16Rows, ns = (q.L + kL16L - 1) / kL16L;
    w.tile = lu % tiles;
    w.z = lu / tiles;
    w.s0 = static_cast<int>(static_cast<long long>(w.z) * ns / q.splits);
    w.s1 = static_cast<int>(static_cast<long long>(w.z + 1) * ns / q.splits);
    return w;
}

__device__ __forceinline__ float step_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Two codes (bytes with the sign bit flipped, i.e. code + 128) times their steps as a bf16 pair; exact.
__device__ __forceinline__ uint32_t code_pair(uint32_t u0, uint32_t u1, float2 step) {
    const float2 f = __fadd2_rn(make_float2(__uint_as_float(u0), __uint_as_float(u1)),
                                make_float2(-8388736.0f, -8388736.0f));  // -(2^23 + 128)
    const float2 v = __fmul2_rn(f, step);
    return __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632);
}

template <int RP, bool MN, bool F32>
__global__ void __launch_bounds__(kL16Threads, 1) lora16_kernel(const __grid_constant__ Lora16Pass P) {
    using C = L16Cfg<RP, F32>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int units = l16_units(P.prob[0]) + (P.count > 1 ? l16_units(P.prob[1]) : 0);
    int* status = P.status;

    const uint32_t bar = base + C::kBarOff;
    auto full = [&](int s) { return bar + 8u * s; };
    auto split = [&](int s) { return bar + 8u * (C::kStages + s); };
    auto empty = [&](int s) { return bar + 8u * (2 * C::kStages + s); };
    auto chunk_empty = [&](int b) { return bar + 8u * (3 * C::kStages + b); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kBarOff + C::kNumBars * 8);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBarOff + C::kNumBars * 8 + 8);

    if (tid == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(split(s), 4);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) mbar_init(chunk_empty(b), 4);
        *abort_flag = 0;
        fence_mbarrier_init();
    }
    if (warp == 3) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    pdl_launch_dependents();
    pdl_wait();  // the planes (and the activations) may come from the launch before

    if (warp == 0) {
        if (lane == 0) {
            // --------------------------------------------------- producer --
            for (int i = 0; i < P.count; ++i) {
                tma_prefetch_desc(&P.prob[i].tm_a);
                tma_prefetch_desc(&P.prob[i].tm_b);
            }
            int q = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
                const L16Unit w = l16_unit(P, u);
                const Lora16Problem& pb = P.prob[w.pi];
                const bool wide = F32 && pb.kind == kL16F32;
                const uint32_t bytes = (pb.kind == kL16Act8 ? kL16ATile / 2 : wide ? 2 * kL16ATile : kL16ATile) + C::kBTile;
                const int row0 = w.tile * kL16Rows;
                for (int st = w.s0; st < w.s1; ++st, ++q) {
                    const int s = q % C::kStages;
                    if (q >= C::kStages &&
                        !mbar_wait(empty(s), ((q / C::kStages) - 1) & 1u, abort_flag, status, kStatusTimeoutProducer)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a = base + s * C::kStageBytes;
                    const int l0 = st * kL16L;
                    mbar_arrive_expect_tx(full(s), bytes);
                    if constexpr (MN) {
                        tma_load_2d(a, &pb.tm_a, full(s), row0, l0);
                    } else {
                        tma_load_2d(a, &pb.tm_a, full(s), l0, row0);
                        if (wide) tma_load_2d(a + kL16ATile, &pb.tm_a, full(s), l0 + 32, row0);  // 32 fp32 per box row
                    }
                    tma_load_2d(a + C::kATile, &pb.tm_b, full(s), l0, 0);
                }
            }
            if (*abort_flag)
                for (int j = q > C::kStages ? q - C::kStages : 0; j < q; ++j)
                    mbar_drain(full(j % C::kStages), (j / C::kStages) & 1u);
        }
        __syncwarp();
    } else if (warp == 1 || warp == 2) {
        if (lane == 0) {
            // -------------------------------- MMA: even and odd stages --
            const int par = warp - 1;
            constexpr uint32_t idesc = umma_idesc_f16(1u, kL16Rows, C::kN);
            const uint32_t dacc = tmem + static_cast<uint32_t>(par * C::kN);
            int last = -1, q = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
                const L16Unit w = l16_unit(P, u);
                const bool wide = F32 && P.prob[w.pi].kind == kL16F32;
                for (int st = w.s0; st < w.s1; ++st, ++q) {
                    if ((q & 1) != par) continue;
                    const int s = q % C::kStages;
                    if ((q >= 2 &&
                         !mbar_wait(chunk_empty(par), ((q >> 1) - 1) & 1u, abort_flag, status, kStatusTimeoutMma)) ||
                        !mbar_wait(split(s), (q / C::kStages) & 1u, abort_flag, status, kStatusTimeoutMma)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t bt = base + s * C::kStageBytes + C::kATile;
                    const uint32_t at = tmem + static_cast<uint32_t>(C::kACol + C::kACols * s);
#pragma unroll
                    for (int kk = 0; kk < kL16L / 16; ++kk) {
                        const uint64_t bd = umma_desc_k_sw128(bt + kk * 32);
                        umma_f16_ts(dacc, at + 8 * kk, bd, idesc, kk > 0 ? 1u : 0u);
                        if (wide) {  // the mid and lo planes
                            umma_f16_ts(dacc, at + 32 + 8 * kk, bd, idesc, 1u);
                            umma_f16_ts(dacc, at + 64 + 8 * kk, bd, idesc, 1u);
                        }
                    }
                    umma_commit(empty(s));
                    last = q;
                }
            }
            if (*abort_flag && last >= 0) mbar_drain(empty(last % C::kStages), (last / C::kStages) & 1u);
        }
        __syncwarp();
    } else if (warp >= 4 && warp < 8) {
        // -------------------------------------------------------- epilogue --
        const int quarter = warp & 3;
        const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        int q = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
            const L16Unit w = l16_unit(P, u);
            const Lora16Problem& pb = P.prob[w.pi];
            float total[RP];
#pragma unroll
            for (int j = 0; j < RP; ++j) total[j] = 0.0f;
            for (int st = w.s0; st < w.s1; ++st, ++q) {
                const int b = q & 1;
                if (!mbar_wait_warp(empty(q % C::kStages), (q / C::kStages) & 1u, abort_flag, status,
                                    kStatusTimeoutEpilogue)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const uint32_t col = t_lane + static_cast<uint32_t>(b * C::kN);
#pragma unroll
                for (int cb = 0; cb < RP; cb += 16) {
                    uint32_t h[16], m[16], l[16];
                    tmem_ld16(col + cb, h);
                    tmem_ld16(col + RP + cb, m);
                    tmem_ld16(col + 2 * RP + cb, l);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        total[cb + j] += __uint_as_float(h[j]) + (__uint_as_float(m[j]) + __uint_as_float(l[j]));
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(chunk_empty(b));
            }
            if (!ok) break;
            const int row = w.tile * kL16Rows + quarter * 32 + lane;
            if (row < pb.R) {
                float4* dst = reinterpret_cast<float4*>(pb.partial + (static_cast<size_t>(w.z) * pb.R + row) * RP);
#pragma unroll
                for (int j = 0; j < RP; j += 4)
                    dst[j / 4] = make_float4(total[j], total[j + 1], total[j + 2], total[j + 3]);
            }
        }
    } else if (warp >= 8) {
        // ----------------------------------------------------------- split --
        const int quarter = warp & 3, par = (warp - 8) >> 2, row = quarter * 32 + lane;
        const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        float* steps = reinterpret_cast<float*>(smem + C::kStepOff) + (warp - 8) * 64;
        int q = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
            const L16Unit w = l16_unit(P, u);
            const Lora16Problem& pb = P.prob[w.pi];
            const int drow = w.tile * kL16Rows + row;
            for (int st = w.s0; st < w.s1; ++st, ++q) {
                if ((q & 1) != par) continue;
                const int s = q % C::kStages, l0 = st * kL16L;
                float step0 = 0.0f, step1 = 0.0f;  // this thread's two step factors of the stage
                if (pb.kind == kL16Act8) {
                    if constexpr (MN) {
                        // group of this warp's 32 rows of D, at l = l0 + lane and l0 + 32 + lane
                        const long long g = w.tile * (kL16Rows / 32) + quarter;
                        const uint8_t* e = pb.exps + static_cast<long long>(l0 + lane) * pb.groups + g;
                        if (g < pb.groups) {
                            if (l0 + lane < pb.L) step0 = step_of(__ldg(e));
                            if (l0 + 32 + lane < pb.L) step1 = step_of(__ldg(e + 32ll * pb.groups));
                        }
                    } else {
                        const uint8_t* e = pb.exps + static_cast<long long>(drow) * pb.groups + l0 / 32;
                        if (drow < pb.R) {
                            step0 = step_of(__ldg(e));
                            if (l0 / 32 + 1 < pb.groups) step1 = step_of(__ldg(e + 1));
                        }
                    }
                }
                if (!mbar_wait_warp(full(s), (q / C::kStages) & 1u, abort_flag, status, kStatusTimeoutDequant)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();  // the MMAs that last read this stage's tensor memory have completed
                const uint8_t* stage = smem + s * C::kStageBytes;
                const uint32_t acol = t_lane + static_cast<uint32_t>(C::kACol + C::kACols * s);
                uint32_t v[32];
                if (F32 && pb.kind == kL16F32) {
                    if constexpr (F32) {
                        // 64 fp32 of this row, cut into bf16 hi, mid and lo parts of 8 bits each
                        // (exact, and no value near the largest rounds up to infinity)
                        float f[64];
                        if constexpr (MN) {
                            const float* col = reinterpret_cast<const float*>(stage) + row;  // l at 512 l
#pragma unroll
                            for (int l = 0; l < 64; ++l) f[l] = col[128 * l];
                        } else {
#pragma unroll
                            for (int c = 0; c < 16; ++c) {  // two boxes of 32 l, 128-byte rows
                                const float4 x = *reinterpret_cast<const float4*>(stage + (c >> 3) * kL16ATile + 128 * row +
                                                                                  (((c & 7) ^ (row & 7)) << 4));
                                f[4 * c] = x.x; f[4 * c + 1] = x.y; f[4 * c + 2] = x.z; f[4 * c + 3] = x.w;
                            }
                        }
#pragma unroll
                        for (int p = 0; p < 3; ++p) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                v[i] = __byte_perm(__float_as_uint(f[2 * i]), __float_as_uint(f[2 * i + 1]), 0x7632);
                                f[2 * i] -= __uint_as_float(v[i] << 16);
                                f[2 * i + 1] -= __uint_as_float(v[i] & 0xFFFF0000u);
                            }
                            if (p < 2) tmem_st32(acol + 32 * p, v);
                        }
                    }
                } else if (pb.kind == kL16Act8) {
                    if constexpr (MN) {
                        steps[lane] = step0;
                        steps[32 + lane] = step1;
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 32; ++i) {  // code of l at 128 l + row
                            const uint32_t u0 = stage[256 * i + row], u1 = stage[256 * i + 128 + row];
                            v[i] = code_pair((u0 ^ 0x80u) | 0x4B000000u, (u1 ^ 0x80u) | 0x4B000000u,
                                             *reinterpret_cast<const float2*>(steps + 2 * i));
                        }
                        __syncwarp();  // every lane has read the steps
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {  // 64-byte row, 16-byte piece c at c ^ (row / 2 % 4)
                            const uint4 x = *reinterpret_cast<const uint4*>(stage + 64 * row + ((c ^ ((row >> 1) & 3)) << 4));
                            const uint32_t wd[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
                            const float2 st2 = c < 2 ? make_float2(step0, step0) : make_float2(step1, step1);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    v[c * 8 + i * 2 + h] = code_pair(__byte_perm(wd[i], 0x4B000000u, 0x7440u | (2 * h)),
                                                                     __byte_perm(wd[i], 0x4B000000u, 0x7440u | (2 * h + 1)), st2);
                        }
                    }
                } else if constexpr (MN) {
                    const uint16_t* col = reinterpret_cast<const uint16_t*>(stage) + row;  // l at 256 l
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        v[i] = static_cast<uint32_t>(col[256 * i]) | (static_cast<uint32_t>(col[256 * i + 128]) << 16);
                } else {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint4 x = *reinterpret_cast<const uint4*>(stage + 128 * row + ((c ^ (row & 7)) << 4));
                        v[4 * c] = x.x;
                        v[4 * c + 1] = x.y;
                        v[4 * c + 2] = x.z;
                        v[4 * c + 3] = x.w;
                    }
                }
                tmem_st32(acol + (F32 && pb.kind == kL16F32 ? 64 : 0), v);
                tmem_st_wait();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(split(s));
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

struct L16FinishLaunch {
    Lora16Finish f[2];
    int count, blocks0;
};

// v[row][j] = sum over z of src[z][row][j] in order (or src[j][row] of a
// row-major [r][R] source), written as the planes of a narrow operand or as a
// gradient.  One block per ROWS rows, transposed through shared memory: 32 (whole
// 128-byte lines of fp32 rows), or 16 where few rows have many splits (a thread
// then has two sums at most, eight loads of each in flight).
constexpr int kL16FinThreads = 512;
template <int ROWS>
__global__ void __launch_bounds__(kL16FinThreads) lora16_finish_kernel(const L16FinishLaunch F) {
    __shared__ float tile[ROWS][65];
    pdl_launch_dependents();
    pdl_wait();
    const bool second = F.count > 1 && static_cast<int>(blockIdx.x) >= F.blocks0;
    const Lora16Finish& f = F.f[second ? 1 : 0];
    const int rp = f.rp, R = f.R, r = f.r;
    const long long ld = f.ld;
    const float* src = after_wait(f.src);
    const int r0 = (static_cast<int>(blockIdx.x) - (second ? F.blocks0 : 0)) * ROWS;
    if (f.from_rows) {
        for (int i = threadIdx.x; i < rp * ROWS; i += kL16FinThreads) {
            const int j = i / ROWS, rr = i % ROWS, row = r0 + rr;
            tile[rr][j] = row < R && j < r ? src[static_cast<size_t>(j) * f.pitch + row] : 0.0f;
        }
    } else {
        for (int i = threadIdx.x; i < ROWS * rp; i += kL16FinThreads) {
            const int rr = i / rp, j = i % rp, row = r0 + rr;
            float v = 0.0f;
            if (row < R && j < r) {
                const float* p = src + static_cast<size_t>(row) * f.pitch + j;
                const size_t step = static_cast<size_t>(R) * f.pitch;
#pragma unroll 8
                for (int z = 0; z < f.splits; ++z) v += p[z * step];
            }
            tile[rr][j] = v;
        }
    }
    __syncthreads();
    if (f.mode == kL16Planes16) {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(f.out);
        for (int i = threadIdx.x; i < rp * ROWS; i += kL16FinThreads) {
            const int j = i / ROWS, rr = i % ROWS, row = r0 + rr;
            if (row >= R) continue;
            const float v = tile[rr][j];
            const __nv_bfloat16 hi = __float2bfloat16_rn(v);
            const float e = v - __bfloat162float(hi);
            const __nv_bfloat16 mid = __float2bfloat16_rn(e);
            out[static_cast<size_t>(j) * ld + row] = hi;
            out[static_cast<size_t>(rp + j) * ld + row] = mid;
            out[static_cast<size_t>(2 * rp + j) * ld + row] = __float2bfloat16_rn(e - __bfloat162float(mid));
        }
    } else if (f.mode == kL16PlanesTf32) {
        float* out = static_cast<float*>(f.out);
        for (int i = threadIdx.x; i < rp * ROWS; i += kL16FinThreads) {
            const int j = i / ROWS, rr = i % ROWS, row = r0 + rr;
            if (row >= R) continue;
            const float v = tile[rr][j], h = to_tf32(v);
            out[static_cast<size_t>(j) * ld + row] = h;
            out[static_cast<size_t>(rp + j) * ld + row] = v - h;
        }
    } else if (f.mode == kL16Transposed) {
        for (int i = threadIdx.x; i < r * ROWS; i += kL16FinThreads) {
            const int j = i / ROWS, rr = i % ROWS, row = r0 + rr;
            if (row >= R) continue;
            const float v = f.s * tile[rr][j];
            static_cast<float*>(f.out)[static_cast<size_t>(j) * ld + row] = v;
            if (f.out2) f.out2[static_cast<size_t>(j) * ld + row] = v;
        }
    } else {
        for (int i = threadIdx.x; i < ROWS * r; i += kL16FinThreads) {
            const int rr = i / r, j = i % r, row = r0 + rr;
            if (row >= R) continue;
            const float v = f.s * tile[rr][j];
            static_cast<float*>(f.out)[static_cast<size_t>(row) * ld + j] = v;
            if (f.out2) f.out2[static_cast<size_t>(row) * ld + j] = v;
        }
    }
}

template <typename Kern, typename Arg>
int l16_launch(Kern kern, unsigned grid, int threads, int smem, cudaStream_t stream, const Arg& arg) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, arg));
}

template <int RP, bool MN, bool F32 = false>
int l16_pass(const Lora16Pass& p, cudaStream_t stream) {
    using C = L16Cfg<RP, F32>;
    auto kern = lora16_kernel<RP, MN, F32>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemAlloc);
    if (e != cudaSuccess) return static_cast<int>(e);
    long long units = 0;
    for (int i = 0; i < p.count; ++i)
        units += static_cast<long long>((p.prob[i].R + kL16Rows - 1) / kL16Rows) * p.prob[i].splits;
    if (units > INT_MAX) return static_cast<int>(cudaErrorInvalidValue);
    return l16_launch(kern, static_cast<unsigned>(units < p.sm_count ? units : p.sm_count), kL16Threads, C::kSmemAlloc,
                      stream, p);
}

}  // namespace

int lora16_rp(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }
int lora16_stage() { return kL16L; }

int launch_lora16_pass(const Lora16Pass& p, cudaStream_t stream) {
    if (p.count < 1 || p.count > 2 || p.sm_count < 1) return static_cast<int>(cudaErrorInvalidValue);
    bool f32 = false;
    for (int i = 0; i < p.count; ++i) {
        const Lora16Problem& q = p.prob[i];
        if (q.R < 1 || q.L < 1 || q.splits < 1 || q.splits > (q.L + kL16L - 1) / kL16L || !q.partial ||
            (q.kind == kL16Act8 && (!q.exps || q.groups < 1)) || (q.kind == kL16F32 && p.rp != 16))
            return static_cast<int>(cudaErrorInvalidValue);
        f32 |= q.kind == kL16F32;
    }
    switch (p.rp) {
        case 16:
            if (f32) return p.mn_major ? l16_pass<16, true, true>(p, stream) : l16_pass<16, false, true>(p, stream);
            return p.mn_major ? l16_pass<16, true>(p, stream) : l16_pass<16, false>(p, stream);
        case 32: return p.mn_major ? l16_pass<32, true>(p, stream) : l16_pass<32, false>(p, stream);
        case 64: return p.mn_major ? l16_pass<64, true>(p, stream) : l16_pass<64, false>(p, stream);
        default: return static_cast<int>(cudaErrorInvalidValue);
    }
}

int launch_lora16_finish(const Lora16Finish* f, int count, cudaStream_t stream) {
    if (count < 1 || count > 2) return static_cast<int>(cudaErrorInvalidValue);
    L16FinishLaunch F{};
    F.count = count;
    int most = 0;
    for (int i = 0; i < count; ++i) {
        const Lora16Finish& q = f[i];
        if (q.R < 1 || q.splits < 1 || q.r < 1 || q.rp < q.r || q.rp > 64 || !q.src || !q.out)
            return static_cast<int>(cudaErrorInvalidValue);
        F.f[i] = q;
        most = q.R > most ? q.R : most;
    }
    // 4096 x 4096 x 11008, rank 16: dA / dB in 6.5 us with 32 rows, 9.1 with 16;
    // 32 x 1536 x 2328, rank 64: the whole backward 45 us with 16 rows (77 with
    // 32 rows on 256 threads, one load in flight).
    const int rows = most >= 2048 ? 32 : 16;
    int blocks = 0;
    for (int i = 0; i < count; ++i) {
        blocks += (f[i].R + rows - 1) / rows;
        if (i == 0) F.blocks0 = blocks;
    }
    return rows == 32
               ? l16_launch(lora16_finish_kernel<32>, static_cast<unsigned>(blocks), kL16FinThreads, 0, stream, F)
               : l16_launch(lora16_finish_kernel<16>, static_cast<unsigned>(blocks), kL16FinThreads, 0, stream, F);
}

}  // namespace q4
