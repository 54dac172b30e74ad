// What the training products of q4_grad_gemm.cu and q4_few_rows.cu share: the
// packed weights' blocks in shared memory, their dequantisation into f16 hi and
// lo operands, the transposed operand's descriptor, waits.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "common.cuh"

namespace q4 {

// Raw weights: blocks of 128 n x 128 k (two stages of either product), 64
// bytes of words per n (64-byte swizzled) and 4 scales.
constexpr int kGgRawWords = 128 * 64, kGgRawBytes = kGgRawWords + 128 * 16;

// K-major: see umma_desc_k_sw128.  MN-major, 128-byte swizzle: 64 elements of
// the non-contracted dimension per 128-byte row, 8 rows (contraction) per
// 1024-byte atom; stride-byte-offset 1024 to the next 8 rows, leading-byte-
// offset to the next 64 elements.
__device__ __forceinline__ uint64_t gg_desc_mn_sw128(uint32_t addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// mbar_wait / mbar_wait_warp with the bounded spin in line: a kernel whose
// warpgroups change their register counts makes no calls, and the epilogue
// waits with 128 sums in registers.
__device__ __forceinline__ bool gg_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    const unsigned long long limit = *static_cast<volatile unsigned long long*>(&g_wait_limit_ns);
#pragma unroll 1
    while (true) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > limit) {
            *abort_flag = 1;
            if (status) atomicCAS(status, 0, code);
            return false;
        }
    }
}
__device__ __forceinline__ bool gg_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                             int code) {
    return __all_sync(0xffffffffu, gg_wait(bar, parity, abort_flag, status, code));
}
// tcgen05.wait::ld that takes the loaded registers along, so that they are not read before it.
__device__ __forceinline__ void gg_ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// Eight weights of one word as four f16 pairs of hi (and, with PB = 2, lo)
// parts.  With every nibble's sign bit flipped (v + 8), one LOP3 puts nibbles
// i and i + 4 under f16's 1024 in the two halves of a register, so a pair
// holds k = (0, 4), (1, 5), (2, 6), (3, 7): the operands' order within each 8
// is 0 4 1 5 2 6 3 7 (18 instructions per word; keeping k in order takes a
// byte permute and a second LOP3 per pair, 24).  The logits' rows are stored
// in that order by the cast; of the transposed product it is the order of the
// accumulator's columns, undone by the epilogue's choice of registers.
// hi = RN16(v s_hi + RN16(v s_lo)) as in dequant_word_f16x2, lo = (v s_hi -
// hi) + RN16(v s_lo), whose bracket is exact, so hi + lo is v s to 2^-22.
template <int PB>
__device__ __forceinline__ void gg_dequant(uint32_t q, __half2 s_hi, __half2 s_lo, uint4& hi, uint4& lo) {
    const __half2 sixteenth = __half2half2(__ushort_as_half(0x2C00u));  // 1/16
    const __half2 bias0 = __half2half2(__ushort_as_half(0xE408u));      // -1032: 1024 + (v + 8)
    const __half2 bias1 = __half2half2(__ushort_as_half(0xD480u));      // -72: (1024 + 16 (v + 8)) / 16
    const uint32_t x = q ^ 0x88888888u, y = x >> 8;
    uint32_t t[4] = {(x & 0x000F000Fu) | 0x64006400u, (x & 0x00F000F0u) | 0x64006400u,
                     (y & 0x000F000Fu) | 0x64006400u, (y & 0x00F000F0u) | 0x64006400u};
    uint32_t h[4], l[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const __half2 u = *reinterpret_cast<const __half2*>(&t[b]);
        const __half2 v = (b & 1) ? __hfma2(u, sixteenth, bias1) : __hadd2(u, bias0);
        const __half2 c = __hmul2(v, s_lo);
        const __half2 w = __hfma2(v, s_hi, c);
        h[b] = *reinterpret_cast<const uint32_t*>(&w);
        if constexpr (PB == 2) {
            const __half2 r = __hadd2(__hfma2(v, s_hi, __hneg2(w)), c);
            l[b] = *reinterpret_cast<const uint32_t*>(&r);
        }
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]);
    if constexpr (PB == 2) lo = make_uint4(l[0], l[1], l[2], l[3]);
}
// Place of k (0..7) in that order.
__host__ __device__ constexpr int gg_place(int k) { return k < 4 ? 2 * k : 2 * (k - 4) + 1; }

}  // namespace q4
