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
// groups.  A thread takes 16 bytes of x at a time (4 fp32 or 8 bf16 values, 8
// or 4 lanes per group), so a warp's loads and stores are whole lines, and four
// such pieces a block apart, all loaded before the first is used: both kernels
// are bound by HBM, and one piece per thread leaves too few bytes in flight.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "q4_kernels.h"

namespace q4 {

namespace {

constexpr int kActThreads = 256, kActPieces = 4;
constexpr int kActLargest = 249;  // step byte of magnitudes above 127 * 2^121

template <typename T>
struct ActIo;  // a 16-byte piece of x as V values
template <>
struct ActIo<float> {
    static constexpr int V = 4;
    using Codes = uint32_t;
    static __device__ __forceinline__ void values(uint4 q, float (&v)[4]) {
        v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y);
        v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ Codes codes(const uint32_t (&w)[2]) { return w[0]; }
    static __device__ __forceinline__ void words(Codes c, uint32_t (&w)[2]) { w[0] = c; }
};
template <>
struct ActIo<__nv_bfloat16> {
    static constexpr int V = 8;
    using Codes = uint2;
    static __device__ __forceinline__ void values(uint4 q, float (&v)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        uint32_t w[4];  // restored values are exact in bf16
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ Codes codes(const uint32_t (&w)[2]) { return make_uint2(w[0], w[1]); }
    static __device__ __forceinline__ void words(Codes c, uint32_t (&w)[2]) { w[0] = c.x; w[1] = c.y; }
};

template <typename T>
__global__ void __launch_bounds__(kActThreads) act8_pack_kernel(const T* __restrict__ x, int8_t* __restrict__ codes,
                                                                uint8_t* __restrict__ exps, long long pieces) {
    using Io = ActIo<T>;
    constexpr int V = Io::V, kLanes = 32 / V;  // lanes per group
    const long long t0 = static_cast<long long>(blockIdx.x) * (kActThreads * kActPieces) + threadIdx.x;
    uint4 q[kActPieces];
#pragma unroll
    for (int i = 0; i < kActPieces; ++i) {
        const long long t = t0 + i * kActThreads;
        q[i] = t < pieces ? __ldcs(reinterpret_cast<const uint4*>(x) + t) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kActPieces; ++i) {
        const long long t = t0 + i * kActThreads;  // a group's lanes agree on t < pieces
        float v[V];
        Io::values(q[i], v);
        // magnitudes compared as bits: an infinity or a NaN is above every finite value
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool bad = top >= 0x7F800000u;
        const int step = max(1, static_cast<int>(top >> 23) - 6 + ((top & 0x7FFFFFu) > 0x7E0000u ? 1 : 0));
        const float inv = __uint_as_float(static_cast<uint32_t>(254 - step) << 23);  // 2^-e
        if (step == kActLargest && !bad) {  // 64 steps would restore as an infinity
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = fminf(fmaxf(v[j], -0x1.f8p+127f), 0x1.f8p+127f);
        }
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t c = bad ? 0u : static_cast<uint32_t>(__float2int_rn(v[j] * inv)) & 0xFFu;
            w[j >> 2] |= c << (8 * (j & 3));
        }
        if (t < pieces) {
            reinterpret_cast<typename Io::Codes*>(codes)[t] = Io::codes(w);
            if (t % kLanes == 0) exps[t / kLanes] = static_cast<uint8_t>(bad ? 255 : step);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kActThreads) act8_unpack_kernel(const int8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ exps, T* __restrict__ x,
                                                                  long long pieces) {
    using Io = ActIo<T>;
    constexpr int V = Io::V, kLanes = 32 / V;
    const long long t0 = static_cast<long long>(blockIdx.x) * (kActThreads * kActPieces) + threadIdx.x;
    typename Io::Codes c[kActPieces] = {};
    uint32_t e[kActPieces] = {};
#pragma unroll
    for (int i = 0; i < kActPieces; ++i) {
        const long long t = t0 + i * kActThreads;
        if (t < pieces) {
            c[i] = __ldcs(reinterpret_cast<const typename Io::Codes*>(codes) + t);
            e[i] = __ldg(exps + t / kLanes);
        }
    }
#pragma unroll
    for (int i = 0; i < kActPieces; ++i) {
        const long long t = t0 + i * kActThreads;
        const float step = __uint_as_float(e[i] << 23);
        uint32_t w[2];
        Io::words(c[i], w);
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
            v[j] = static_cast<float>(static_cast<int8_t>((w[j >> 2] >> (8 * (j & 3))) & 0xFFu)) * step;
        if (t < pieces) reinterpret_cast<uint4*>(x)[t] = Io::pack(v);
    }
}

}  // namespace

namespace {
unsigned act8_blocks(long long pieces) {
    const long long per = static_cast<long long>(kActThreads) * kActPieces;
    return static_cast<unsigned>((pieces + per - 1) / per);
}
}  // namespace

int launch_act8_pack(const void* x, bool bf16, int8_t* codes, uint8_t* exps, long long groups, cudaStream_t stream) {
    const long long pieces = groups * (bf16 ? 4 : 8);
    if (bf16)
        act8_pack_kernel<<<act8_blocks(pieces), kActThreads, 0, stream>>>(static_cast<const __nv_bfloat16*>(x), codes, exps,
                                                                          pieces);
    else
        act8_pack_kernel<<<act8_blocks(pieces), kActThreads, 0, stream>>>(static_cast<const float*>(x), codes, exps, pieces);
    return static_cast<int>(cudaGetLastError());
}

int launch_act8_unpack(const int8_t* codes, const uint8_t* exps, void* x, bool bf16, long long groups,
                       cudaStream_t stream) {
    const long long pieces = groups * (bf16 ? 4 : 8);
    if (bf16)
        act8_unpack_kernel<<<act8_blocks(pieces), kActThreads, 0, stream>>>(codes, exps, static_cast<__nv_bfloat16*>(x),
                                                                            pieces);
    else
        act8_unpack_kernel<<<act8_blocks(pieces), kActThreads, 0, stream>>>(codes, exps, static_cast<float*>(x), pieces);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace q4
