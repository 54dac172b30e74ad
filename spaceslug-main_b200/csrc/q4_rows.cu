// The training operators on the frozen int4 weights for a few rows, on the
// CUDA cores in fp32: products that stream the packed weights once per block
// of at most eight rows.
//
//   rows_logits_kernel   z[m][n]  = sum_k x[m][k] w(k, n)        (logits)
//   rows_wt_kernel       dx[m][k] = sum_n d[m][n] w(k, n)        (the transposed product)
//   rows_softmax_kernel  lse, loss and d = g (softmax(z) - onehot) of logit rows, in place
//   rows_proj_kernel     G[m][j]  = s sum_n dy[m][n] B[j][n]     (the adapter's side)
//   rows_finish_kernel   sums the splits of n in order, adds G A^T, rounds once to the output's type
//
// w(k, n) = float(v) * scale as everywhere (vulkan-runtime/shaders/q4gemm.comp:104-122),
// one rounding.  With one to eight rows these products are bound by the
// weights' bytes (0.625 B per weight) or by their unpacking.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "q4_kernels.h"

namespace q4 {

namespace {

__device__ __forceinline__ void row_load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void row_load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ float row_load(const float* p) { return *p; }
__device__ __forceinline__ float row_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void row_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void row_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Eight weights of one word, k ascending: the nibble under 2^23's exponent
// gives 2^23 + (v + 8) exactly, then v, then v * s with one rounding.
__device__ __forceinline__ void word_weights(uint32_t q, float s, float (&w)[8]) {
    const uint32_t lo = (q ^ 0x88888888u) & 0x0F0F0F0Fu;         // k = 0, 2, 4, 6
    const uint32_t hi = ((q >> 4) ^ 0x08080808u) & 0x0F0F0F0Fu;  // k = 1, 3, 5, 7
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        w[2 * b] = (__uint_as_float(__byte_perm(lo, 0x4B000000u, 0x7440u | b)) - 8388616.0f) * s;
        w[2 * b + 1] = (__uint_as_float(__byte_perm(hi, 0x4B000000u, 0x7440u | b)) - 8388616.0f) * s;
    }
}

// One warp per four columns; lanes take the words of k in turn, MR rows of x
// are held in registers against the four columns' weights.
constexpr int kRowsCols = 4;
template <int MR, typename T>
__global__ void __launch_bounds__(256) rows_logits_kernel(const T* __restrict__ x, const uint32_t* __restrict__ packed,
                                                          const float* __restrict__ scales, float* __restrict__ z,
                                                          long long ld_z, int M, int N, int K) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = (blockIdx.x * 8 + warp) * kRowsCols, m0 = blockIdx.y * MR;
    if (n0 >= N) return;
    const int words = K / 8, groups = K / 32;
    float acc[kRowsCols * MR];
#pragma unroll
    for (int i = 0; i < kRowsCols * MR; ++i) acc[i] = 0.0f;
#pragma unroll 2
    for (int w = lane; w < words; w += 32) {
        uint32_t q[kRowsCols];
        float s[kRowsCols];
#pragma unroll
        for (int c = 0; c < kRowsCols; ++c) {
            const size_t n = static_cast<size_t>(min(n0 + c, N - 1));
            q[c] = __ldg(packed + n * words + w);
            s[c] = __ldg(scales + n * groups + (w >> 2));
        }
        float xv[MR][8];
#pragma unroll
        for (int r = 0; r < MR; ++r) row_load8(x + static_cast<size_t>(min(m0 + r, M - 1)) * K + w * 8, xv[r]);
#pragma unroll
        for (int c = 0; c < kRowsCols; ++c) {
            float wv[8];
            word_weights(q[c], s[c], wv);
#pragma unroll
            for (int r = 0; r < MR; ++r)
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[c * MR + r] = fmaf(xv[r][i], wv[i], acc[c * MR + r]);
        }
    }
    const float total = warp_reduce_scatter<kRowsCols * MR>(acc, lane);
    constexpr int kShare = 32 / (kRowsCols * MR);  // lanes that hold the same value
    const int i = value_index<kRowsCols * MR>(lane), c = i / MR, r = i % MR;
    if (lane % kShare == 0 && n0 + c < N && m0 + r < M) z[static_cast<long long>(m0 + r) * ld_z + n0 + c] = total;
}

// One thread per word of k (8 outputs) and MR rows; n in blockIdx.y's range.
// The rows' d values of 256 n at a time sit in shared memory.
constexpr int kWtThreads = 128, kWtTile = 256;
template <int MR, typename T>
__global__ void __launch_bounds__(kWtThreads) rows_wt_kernel(const T* __restrict__ d, long long ld_d,
                                                             const uint32_t* __restrict__ packed,
                                                             const float* __restrict__ scales,
                                                             float* __restrict__ partial, int M, int N, int K) {
    __shared__ float ds[kWtTile][MR];
    const int kw = blockIdx.x * kWtThreads + threadIdx.x, words = K / 8, groups = K / 32;
    const int m0 = blockIdx.z * MR;
    const int nb = static_cast<int>(static_cast<long long>(N) * blockIdx.y / gridDim.y);
    const int ne = static_cast<int>(static_cast<long long>(N) * (blockIdx.y + 1) / gridDim.y);
    float acc[MR][8];
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r][i] = 0.0f;
    for (int n0 = nb; n0 < ne; n0 += kWtTile) {
        const int cnt = min(kWtTile, ne - n0);
        __syncthreads();
        for (int i = threadIdx.x; i < MR * kWtTile; i += kWtThreads) {
            const int r = i / kWtTile, j = i % kWtTile;
            ds[j][r] = (j < cnt && m0 + r < M) ? row_load(d + static_cast<long long>(m0 + r) * ld_d + n0 + j) : 0.0f;
        }
        __syncthreads();
        if (kw < words) {
            const uint32_t* pw = packed + static_cast<size_t>(n0) * words + kw;
            const float* ps = scales + static_cast<size_t>(n0) * groups + (kw >> 2);
#pragma unroll 8
            for (int j = 0; j < cnt; ++j) {
                float wv[8];
                word_weights(__ldg(pw + static_cast<size_t>(j) * words), __ldg(ps + static_cast<size_t>(j) * groups), wv);
#pragma unroll
                for (int r = 0; r < MR; ++r) {
                    const float dv = ds[j][r];
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[r][i] = fmaf(dv, wv[i], acc[r][i]);
                }
            }
        }
    }
    if (kw >= words) return;
#pragma unroll
    for (int r = 0; r < MR; ++r)
        if (m0 + r < M) {
            float4* out = reinterpret_cast<float4*>(
                partial + (static_cast<size_t>(blockIdx.y) * M + m0 + r) * K + static_cast<size_t>(kw) * 8);
            out[0] = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
            out[1] = make_float4(acc[r][4], acc[r][5], acc[r][6], acc[r][7]);
        }
}

__device__ __forceinline__ float rows_block_sum(float v, float* red) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) t += red[i];  // the same order in every thread
    return t;
}

// One block per row of logits.  A negative target takes the row out of the
// loss (loss 0, gradient 0); one past the columns gives NaN, never a read
// outside the row.
__global__ void __launch_bounds__(512) rows_softmax_kernel(float* __restrict__ z, long long ld_z,
                                                           const long long* __restrict__ targets,
                                                           const float* __restrict__ row_scale,
                                                           float* __restrict__ loss, float* __restrict__ lse, int N,
                                                           int want_grad) {
    __shared__ float red[16];
    float* row = z + static_cast<long long>(blockIdx.x) * ld_z;
    float top = -INFINITY;
    for (int n = threadIdx.x; n < N; n += blockDim.x) top = fmaxf(top, row[n]);
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) top = fmaxf(top, red[i]);
    float sum = 0.0f;
    for (int n = threadIdx.x; n < N; n += blockDim.x) sum += expf(row[n] - top);
    sum = rows_block_sum(sum, red);
    const float l = top + logf(sum);
    const long long t = targets[blockIdx.x];
    const bool used = t >= 0;
    const float zt = t >= 0 && t < N ? row[t] : NAN;
    __syncthreads();
    if (threadIdx.x == 0) {
        if (lse != nullptr) lse[blockIdx.x] = l;
        loss[blockIdx.x] = used ? l - zt : 0.0f;
    }
    if (!want_grad) return;
    const float g = used ? (row_scale != nullptr ? row_scale[blockIdx.x] : 1.0f) : 0.0f;
    const float bad = used && t >= N ? NAN : 0.0f;
    for (int n = threadIdx.x; n < N; n += blockDim.x)
        row[n] = used ? g * (expf(row[n] - top) / sum - (n == t ? 1.0f : 0.0f)) + bad : 0.0f;
}

// Four rows x 16 ranks per block; the threads take n in turn and the 64 sums
// are added over the block in a fixed order.
constexpr int kProjRows = 4, kProjRanks = 16;
template <typename T>
__global__ void __launch_bounds__(256) rows_proj_kernel(const T* __restrict__ dy, const float* __restrict__ b,
                                                        float scale, float* __restrict__ g, int M, int N, int rank) {
    __shared__ float red[8][64];
    const int m0 = blockIdx.x * kProjRows, j0 = blockIdx.y * kProjRanks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float acc[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) acc[i] = 0.0f;
    for (int n = threadIdx.x; n < N; n += 256) {
        float dv[kProjRows];
#pragma unroll
        for (int r = 0; r < kProjRows; ++r) dv[r] = row_load(dy + static_cast<size_t>(min(m0 + r, M - 1)) * N + n);
#pragma unroll
        for (int j = 0; j < kProjRanks; ++j) {
            const float bv = __ldg(b + static_cast<size_t>(min(j0 + j, rank - 1)) * N + n);
#pragma unroll
            for (int r = 0; r < kProjRows; ++r) acc[r * kProjRanks + j] = fmaf(dv[r], bv, acc[r * kProjRanks + j]);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = acc[32 * h + i];
        red[warp][32 * h + value_index<32>(lane)] = warp_reduce_scatter<32>(v, lane);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        float t = 0.0f;
        for (int w = 0; w < 8; ++w) t += red[w][threadIdx.x];
        const int r = threadIdx.x / kProjRanks, j = threadIdx.x % kProjRanks;
        if (m0 + r < M && j0 + j < rank) g[static_cast<size_t>(m0 + r) * rank + j0 + j] = scale * t;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) rows_finish_kernel(const float* __restrict__ partial, int splits,
                                                          long long split_floats, const float* __restrict__ g,
                                                          const float* __restrict__ a, int rank, T* __restrict__ out,
                                                          long long count, int K) {
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= count) return;
    float v = 0.0f;
    for (int z = 0; z < splits; ++z) v += partial[z * split_floats + i];
    if (rank > 0) {
        const long long m = i / K;
        const int k = static_cast<int>(i % K);
        float l = 0.0f;
        for (int j = 0; j < rank; ++j) l = fmaf(g[m * rank + j], __ldg(a + static_cast<size_t>(k) * rank + j), l);
        v += l;
    }
    row_store(out + i, v);
}

template <typename F>
void rows_dispatch(int M, F&& f) {
    if (M >= 5)
        f(std::integral_constant<int, 8>());
    else if (M >= 3)
        f(std::integral_constant<int, 4>());
    else if (M == 2)
        f(std::integral_constant<int, 2>());
    else
        f(std::integral_constant<int, 1>());
}

}  // namespace

int launch_rows_logits(const void* x, bool bf16, const uint32_t* packed, const float* scales, float* z, long long ld_z,
                       int M, int N, int K, cudaStream_t stream) {
    rows_dispatch(M, [&](auto mr) {
        constexpr int MR = decltype(mr)::value;
        const dim3 grid(static_cast<unsigned>((N + 8 * kRowsCols - 1) / (8 * kRowsCols)),
                        static_cast<unsigned>((M + MR - 1) / MR));
        if (bf16)
            rows_logits_kernel<MR><<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(x), packed, scales, z,
                                                             ld_z, M, N, K);
        else
            rows_logits_kernel<MR><<<grid, 256, 0, stream>>>(static_cast<const float*>(x), packed, scales, z, ld_z, M,
                                                             N, K);
    });
    return static_cast<int>(cudaGetLastError());
}

// Splits of n: enough blocks for the SMs, at least 64 n each.
int rows_wt_splits(int M, int N, int K, int sm_count) {
    const long long blocks = static_cast<long long>((K / 8 + kWtThreads - 1) / kWtThreads) * ((M + 7) / 8);
    long long s = (8ll * sm_count + blocks - 1) / blocks;
    if (s > (N + 63) / 64) s = (N + 63) / 64;
    return static_cast<int>(s < 1 ? 1 : s);
}

int launch_rows_wt(const void* d, bool bf16, long long ld_d, const uint32_t* packed, const float* scales,
                   float* partial, int splits, int M, int N, int K, cudaStream_t stream) {
    rows_dispatch(M, [&](auto mr) {
        constexpr int MR = decltype(mr)::value;
        const dim3 grid(static_cast<unsigned>((K / 8 + kWtThreads - 1) / kWtThreads), static_cast<unsigned>(splits),
                        static_cast<unsigned>((M + MR - 1) / MR));
        if (bf16)
            rows_wt_kernel<MR><<<grid, kWtThreads, 0, stream>>>(static_cast<const __nv_bfloat16*>(d), ld_d, packed,
                                                                scales, partial, M, N, K);
        else
            rows_wt_kernel<MR><<<grid, kWtThreads, 0, stream>>>(static_cast<const float*>(d), ld_d, packed, scales,
                                                                partial, M, N, K);
    });
    return static_cast<int>(cudaGetLastError());
}

int launch_rows_softmax(float* z, long long ld_z, const long long* targets, const float* row_scale, float* loss,
                        float* lse, int M, int N, bool want_grad, cudaStream_t stream) {
    rows_softmax_kernel<<<static_cast<unsigned>(M), 512, 0, stream>>>(z, ld_z, targets, row_scale, loss, lse, N,
                                                                       want_grad ? 1 : 0);
    return static_cast<int>(cudaGetLastError());
}

int launch_rows_proj(const void* dy, bool bf16, const float* b, float scale, float* g, int M, int N, int rank,
                     cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>((M + kProjRows - 1) / kProjRows),
                    static_cast<unsigned>((rank + kProjRanks - 1) / kProjRanks));
    if (bf16)
        rows_proj_kernel<<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(dy), b, scale, g, M, N, rank);
    else
        rows_proj_kernel<<<grid, 256, 0, stream>>>(static_cast<const float*>(dy), b, scale, g, M, N, rank);
    return static_cast<int>(cudaGetLastError());
}

int launch_rows_finish(const float* partial, int splits, long long split_floats, const float* g, const float* a,
                       int rank, void* out, bool bf16, int M, int K, cudaStream_t stream) {
    const long long count = static_cast<long long>(M) * K;
    const unsigned blocks = static_cast<unsigned>((count + 255) / 256);
    if (bf16)
        rows_finish_kernel<<<blocks, 256, 0, stream>>>(partial, splits, split_floats, g, a, rank,
                                                       static_cast<__nv_bfloat16*>(out), count, K);
    else
        rows_finish_kernel<<<blocks, 256, 0, stream>>>(partial, splits, split_floats, g, a, rank, static_cast<float*>(out),
                                                       count, K);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace q4
