// Activations kept in 8 bits for a backward pass (no reference counterpart).
//
// Each group of 32 consecutive values of a row has one power-of-two step 2^e:
// e is the smallest integer >= -126 with max|x| <= 127 2^e, kept as the byte
// e + 127, and a value is kept as the int8 code rn(x 2^-e).  The restored
// value code * 2^e is off by at most 2^e / 2.  A power-of-two step costs up to
// one bit against max / 127, and buys two things: x 2^-e is exact, so the
// codes are the same on every machine, and code * 2^e has 7 significant bits,
// so the backward's tensor-core products take it as bf16 without rounding it
// a second time.  From the bits of the largest magnitude, b = 2^(E-127) (1 +
// f), the step byte is E - 6, plus 1 where 64 (1 + f) > 127.  With the
// largest step, 2^122, codes stop at 63, since 64 of it is no fp32 value (the
// largest fp32 values are then up to one step off).  A group that
// holds an infinity or a NaN keeps the byte 255 and zero codes, which every
// reader turns into NaN (0 * inf).
//
// K is a multiple of 32, so a contiguous [m][K] matrix is a flat list of
// groups: both kernels give 8 values to a thread and 4 lanes to a group.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "q4_kernels.h"

namespace q4 {

namespace {

constexpr int kActThreads = 256;
constexpr int kActLargest = 249;  // step byte of magnitudes above 127 * 2^121

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);  // exact for restored values
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__global__ void __launch_bounds__(kActThreads) act8_pack_kernel(const T* __restrict__ x, int8_t* __restrict__ codes,
                                                                uint8_t* __restrict__ exps, long long groups) {
    const long long t = static_cast<long long>(blockIdx.x) * kActThreads + threadIdx.x;
    const long long g = t >> 2;
    const bool in = g < groups;  // a group's four lanes agree
    float v[8];
    if (in) {
        load8(x + t * 8, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
    // magnitudes compared as bits: an infinity or a NaN is above every finite value
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const bool bad = top >= 0x7F800000u;
    const int step = max(1, static_cast<int>(top >> 23) - 6 + ((top & 0x7FFFFFu) > 0x7E0000u ? 1 : 0));
    const float inv = __uint_as_float(static_cast<uint32_t>(254 - step) << 23);  // 2^-e
    if (step == kActLargest && !bad) {  // 64 steps would restore as an infinity
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fminf(fmaxf(v[i], -0x1.f8p+127f), 0x1.f8p+127f);
    }
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t c = bad ? 0u : static_cast<uint32_t>(__float2int_rn(v[i] * inv)) & 0xFFu;
        w[i >> 2] |= c << (8 * (i & 3));
    }
    if (in) {
        *reinterpret_cast<uint2*>(codes + t * 8) = make_uint2(w[0], w[1]);
        if ((t & 3) == 0) exps[g] = static_cast<uint8_t>(bad ? 255 : step);
    }
}

template <typename T>
__global__ void __launch_bounds__(kActThreads) act8_unpack_kernel(const int8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ exps, T* __restrict__ x,
                                                                  long long groups) {
    const long long t = static_cast<long long>(blockIdx.x) * kActThreads + threadIdx.x;
    const long long g = t >> 2;
    if (g >= groups) return;
    const uint2 q = __ldcs(reinterpret_cast<const uint2*>(codes + t * 8));
    const float step = __uint_as_float(static_cast<uint32_t>(exps[g]) << 23);
    const uint32_t w[2] = {q.x, q.y};
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = static_cast<float>(static_cast<int8_t>((w[i >> 2] >> (8 * (i & 3))) & 0xFFu)) * step;
    store8(x + t * 8, v);
}

__global__ void __launch_bounds__(256) bf16_to_f32_kernel(const __nv_bfloat16* __restrict__ x, float* __restrict__ y,
                                                          long long count) {
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i < count) y[i] = __bfloat162float(x[i]);
}

}  // namespace

int launch_bf16_to_f32(const void* x, float* y, long long count, cudaStream_t stream) {
    bf16_to_f32_kernel<<<static_cast<unsigned>((count + 255) / 256), 256, 0, stream>>>(
        static_cast<const __nv_bfloat16*>(x), y, count);
    return static_cast<int>(cudaGetLastError());
}

int launch_act8_pack(const void* x, bool bf16, int8_t* codes, uint8_t* exps, long long groups, cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>((groups * 4 + kActThreads - 1) / kActThreads);
    if (bf16)
        act8_pack_kernel<<<blocks, kActThreads, 0, stream>>>(static_cast<const __nv_bfloat16*>(x), codes, exps, groups);
    else
        act8_pack_kernel<<<blocks, kActThreads, 0, stream>>>(static_cast<const float*>(x), codes, exps, groups);
    return static_cast<int>(cudaGetLastError());
}

int launch_act8_unpack(const int8_t* codes, const uint8_t* exps, void* x, bool bf16, long long groups,
                       cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>((groups * 4 + kActThreads - 1) / kActThreads);
    if (bf16)
        act8_unpack_kernel<<<blocks, kActThreads, 0, stream>>>(codes, exps, static_cast<__nv_bfloat16*>(x), groups);
    else
        act8_unpack_kernel<<<blocks, kActThreads, 0, stream>>>(codes, exps, static_cast<float*>(x), groups);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace q4
