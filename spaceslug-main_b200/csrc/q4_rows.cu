// The training operators on the frozen int4 weights for one to eight rows (up to
// a size; see rows_pay_dx and rows_pay_loss), on the CUDA cores in fp32: products
// that stream the packed weights once.
//
//   rows_logits_kernel   z[m][n]  = sum_k x[m][k] w(k, n), and each 32 columns' max and sum of exponentials
//   rows_loss_kernel     lse, loss and the rows' coefficients of the gradient
//   rows_wt_kernel       dx[m][k] = sum_n d[m][n] w(k, n), d given or formed from z and the coefficients
//   rows_proj_kernel     G[m][j]  = sum_n dy[m][n] B[j][n] (the adapter's side)
//   rows_finish_kernel   sums the splits of n in order, adds s G A^T, rounds once to the output's type
//
// w(k, n) = float(v) * scale as everywhere (vulkan-runtime/shaders/q4gemm.comp:104-122),
// one rounding.  With a row or two these products are bound by the weights'
// bytes (0.625 B per weight), with eight by their unpacking and fp32 FMAs; so
// the row count is a template constant.
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

// z2 += a * b for two packed k.
__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// 32 columns per block, one per lane; the eight warps share k: each takes four
// of the 32 groups of a 1024-k chunk, whose words (16 bytes per group) and
// scales are all loaded before the chunk's x, which every lane reads from
// shared memory at once (one wavefront per four k of a row).  Keeping x in
// registers against four columns per warp instead took 150 registers, eight
// warps per SM and 39 us at 5 x 1024 x 32003.  The warps' sums meet in shared
// memory, and per row the 32 columns give their maximum and the sum of
// exp(z - max), both without the target's column (log2 units: smax, ssum).
constexpr int kRowsCols = 32, kRowsChunk = 1024, kRowsBatch = kRowsChunk / 32 / 8;
template <int MR, typename T>
__global__ void __launch_bounds__(256, 3) rows_logits_kernel(const T* x, const uint32_t* __restrict__ packed,
                                                             const float* __restrict__ scales, const long long* targets,
                                                             float* __restrict__ z, float* __restrict__ zt,
                                                             float* __restrict__ smax, float* __restrict__ ssum, int N,
                                                             int K) {
    __shared__ __align__(16) float xs[MR * kRowsChunk];
    pdl_launch_dependents();
    pdl_wait();
    x = after_wait(x);
    targets = after_wait(targets);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = blockIdx.x * kRowsCols + lane, groups = K / 32;
    const size_t row_g = static_cast<size_t>(min(n, N - 1)) * groups;
    float2 acc[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) acc[r] = make_float2(0.0f, 0.0f);
    for (int k0 = 0; k0 < K; k0 += kRowsChunk) {
        const int g0 = k0 / 32 + warp * kRowsBatch, kn = min(kRowsChunk, K - k0);
        uint4 q[kRowsBatch];
        float s[kRowsBatch];
#pragma unroll
        for (int b = 0; b < kRowsBatch; ++b) {
            const bool in = g0 + b < groups;
            q[b] = in ? __ldg(reinterpret_cast<const uint4*>(packed) + row_g + g0 + b) : make_uint4(0, 0, 0, 0);
            s[b] = in ? __ldg(scales + row_g + g0 + b) : 0.0f;
        }
        __syncthreads();  // the chunk before has been read
        for (int i = threadIdx.x * 8; i < MR * kRowsChunk; i += 256 * 8) {
            const int r = i / kRowsChunk, k = i % kRowsChunk;
            float v[8];
            if (k < kn) {
                row_load8(x + static_cast<size_t>(r) * K + k0 + k, v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = 0.0f;
            }
            *reinterpret_cast<float4*>(xs + i) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(xs + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < kRowsBatch; ++b) {
            if (g0 + b >= groups) break;  // an infinite x may not meet a group that does not exist
            const uint32_t words[4] = {q[b].x, q[b].y, q[b].z, q[b].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float wv[8];
                word_weights(words[i], s[b], wv);
                const float* xp = xs + (warp * kRowsBatch + b) * 32 + i * 8;
#pragma unroll
                for (int r = 0; r < MR; ++r) {
                    const float4 u = *reinterpret_cast<const float4*>(xp + r * kRowsChunk);
                    const float4 v = *reinterpret_cast<const float4*>(xp + r * kRowsChunk + 4);
                    acc[r] = ffma2(make_float2(u.x, u.y), make_float2(wv[0], wv[1]), acc[r]);
                    acc[r] = ffma2(make_float2(u.z, u.w), make_float2(wv[2], wv[3]), acc[r]);
                    acc[r] = ffma2(make_float2(v.x, v.y), make_float2(wv[4], wv[5]), acc[r]);
                    acc[r] = ffma2(make_float2(v.z, v.w), make_float2(wv[6], wv[7]), acc[r]);
                }
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < MR; ++r) xs[(r * 8 + warp) * 32 + lane] = acc[r].x + acc[r].y;
    __syncthreads();
    for (int r = warp; r < MR; r += 8) {  // one warp per row, one column per lane
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) total += xs[(r * 8 + w) * 32 + lane];
        const bool hot = targets[r] == n;
        if (n < N) z[static_cast<long long>(r) * N + n] = total;
        if (hot && n < N) zt[r] = total;
        const float z2 = n < N && !hot ? total * 1.4426950408889634f : -INFINITY;
        float top = z2;
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float sum = exp2f(z2 - (top == -INFINITY ? 0.0f : top));
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            smax[static_cast<size_t>(r) * gridDim.x + blockIdx.x] = top;
            ssum[static_cast<size_t>(r) * gridDim.x + blockIdx.x] = sum;
        }
    }
}

// One block per row of the blocks' statistics: lse, loss, and for the
// gradient M2, g / S and g (p_target - 1) (coef[3 row ..]).  A negative target
// takes the row out of the loss (loss 0, gradient 0); one past the columns
// gives NaN.
__global__ void __launch_bounds__(512) rows_loss_kernel(const float* smax, const float* ssum, const float* zt,
                                                        const long long* targets, const float* row_scale, float* __restrict__ loss,
                                                        float* __restrict__ lse, float* __restrict__ coef, int N,
                                                        int tiles) {
    __shared__ float red[16];
    pdl_launch_dependents();
    pdl_wait();
    smax = after_wait(smax);
    ssum = after_wait(ssum);
    zt = after_wait(zt);
    targets = after_wait(targets);
    row_scale = after_wait(row_scale);
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* sm = smax + static_cast<size_t>(row) * tiles;
    const float* ss = ssum + static_cast<size_t>(row) * tiles;
    const long long t = targets[row];
    const float t2 = t >= 0 && t < N ? zt[row] * 1.4426950408889634f : -INFINITY;
    float top = t2;
    for (int i = threadIdx.x; i < tiles; i += 512) top = fmaxf(top, sm[i]);
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int i = 0; i < 16; ++i) top = fmaxf(top, red[i]);
    __syncthreads();
    float sum = 0.0f;
    for (int i = threadIdx.x; i < tiles; i += 512) sum += exp2f(sm[i] - top) * ss[i];
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    sum = 0.0f;
    for (int i = 0; i < 16; ++i) sum += red[i];
    const float et = exp2f(t2 - top), all = sum + et;
    const float l = 0.69314718055994531f * (top + log2f(all));
    const float v = t < 0 ? 0.0f : t >= N ? NAN : et > 0.0009765625f ? log1pf(sum / et) : l - zt[row];
    if (lse != nullptr) lse[row] = l;
    loss[row] = v;
    const float g = t < 0 ? 0.0f : row_scale != nullptr ? row_scale[row] : 1.0f;
    coef[3 * row] = top;
    coef[3 * row + 1] = t < N ? g / all : NAN;
    coef[3 * row + 2] = t < 0 ? 0.0f : g * expm1f(-v);
}

// Thread (word of k, part p of 4): 8 outputs of MR rows over a quarter of
// blockIdx.y's range of n; the quarters are added through shared memory.  The
// rows' d values of 256 n at a time sit in shared memory: d itself, or with
// `coef` (the loss) g p = coef[1] exp2(z2 - coef[0]) and coef[2] at the target.
// The words of eight n per thread are in flight while d is staged.
// Registers for two blocks per SM from three rows on: held to a quarter of them,
// four rows of 4096 x 11008 took 58 us instead of 39.
constexpr int kWtWords = 64, kWtParts = 4, kWtThreads = kWtWords * kWtParts, kWtTile = 128, kWtBatch = 8;
template <int MR, typename T>
__global__ void __launch_bounds__(kWtThreads, MR <= 2 ? 4 : 2) rows_wt_kernel(const T* d, const float* coef, const long long* targets,
                                                             const uint32_t* __restrict__ packed,
                                                             const float* __restrict__ scales,
                                                             float* __restrict__ partial, int N, int K) {
    __shared__ __align__(16) float ds[kWtTile][MR];
    __shared__ __align__(16) float sums[kWtParts - 1][kWtWords][8];
    pdl_launch_dependents();
    const int wl = threadIdx.x % kWtWords, part = threadIdx.x / kWtWords;
    const int kw = blockIdx.x * kWtWords + wl, words = K / 8, groups = K / 32;
    const int nb = static_cast<int>(static_cast<long long>(N) * blockIdx.y / gridDim.y);
    const int ne = static_cast<int>(static_cast<long long>(N) * (blockIdx.y + 1) / gridDim.y);
    float2 acc[MR][4];
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][i] = make_float2(0.0f, 0.0f);
    for (int n0 = nb; n0 < ne; n0 += kWtTile) {
        const int cnt = min(kWtTile, ne - n0);
        const uint32_t* pw = packed + static_cast<size_t>(n0) * words + kw;
        const float* ps = scales + static_cast<size_t>(n0) * groups + (kw >> 2);
        uint32_t q[kWtBatch];
        float s[kWtBatch];
        auto load = [&](int j0) {
#pragma unroll
            for (int b = 0; b < kWtBatch; ++b) {
                const int j = j0 + b * kWtParts;
                const bool in = j < cnt && kw < words;
                q[b] = in ? __ldg(pw + static_cast<size_t>(j) * words) : 0u;
                s[b] = in ? __ldg(ps + static_cast<size_t>(j) * groups) : 0.0f;
            }
        };
        load(part);
        if (n0 == nb) {
            pdl_wait();  // d, and the partial sums' memory
            d = after_wait(d);
            coef = after_wait(coef);
            targets = after_wait(targets);
        }
        __syncthreads();  // the tile before has been read
        for (int i = threadIdx.x; i < MR * kWtTile; i += kWtThreads) {
            const int r = i / kWtTile, j = i % kWtTile;
            float v = 0.0f;
            if (j < cnt) {
                v = row_load(d + static_cast<size_t>(r) * N + n0 + j);
                if (coef != nullptr) {
                    const float inv = coef[3 * r + 1];
                    v = targets[r] < 0 ? 0.0f
                                       : targets[r] == n0 + j ? coef[3 * r + 2]
                                                              : inv * exp2f(v * 1.4426950408889634f - coef[3 * r]);
                }
            }
            ds[j][r] = v;
        }
        __syncthreads();
        for (int j0 = part; j0 < cnt; j0 += kWtBatch * kWtParts) {
            if (j0 != part) load(j0);
#pragma unroll
            for (int b = 0; b < kWtBatch; ++b) {
                const int j = j0 + b * kWtParts;
                if (j >= cnt) break;
                float wv[8];
                word_weights(q[b], s[b], wv);
#pragma unroll
                for (int r = 0; r < MR; ++r) {
                    const float2 dv = make_float2(ds[j][r], ds[j][r]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[r][i] = ffma2(dv, make_float2(wv[2 * i], wv[2 * i + 1]), acc[r][i]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < MR; ++r) {
        float4* mine = part > 0 ? reinterpret_cast<float4*>(&sums[part - 1][wl][0]) : nullptr;
        __syncthreads();
        if (part > 0) {
            mine[0] = make_float4(acc[r][0].x, acc[r][0].y, acc[r][1].x, acc[r][1].y);
            mine[1] = make_float4(acc[r][2].x, acc[r][2].y, acc[r][3].x, acc[r][3].y);
        }
        __syncthreads();
        if (part == 0 && kw < words) {
            float4 a = make_float4(acc[r][0].x, acc[r][0].y, acc[r][1].x, acc[r][1].y);
            float4 b = make_float4(acc[r][2].x, acc[r][2].y, acc[r][3].x, acc[r][3].y);
#pragma unroll
            for (int p = 0; p < kWtParts - 1; ++p) {
                const float4 u = *reinterpret_cast<const float4*>(&sums[p][wl][0]);
                const float4 v = *reinterpret_cast<const float4*>(&sums[p][wl][4]);
                a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
                b.x += v.x; b.y += v.y; b.z += v.z; b.w += v.w;
            }
            float4* out = reinterpret_cast<float4*>(partial + (static_cast<size_t>(blockIdx.y) * MR + r) * K +
                                                    static_cast<size_t>(kw) * 8);
            out[0] = a;
            out[1] = b;
        }
    }
}

// Four rows x 16 ranks per block and range of n (blockIdx.z): partial[z][M][rank].
constexpr int kProjRows = 4, kProjRanks = 16;
template <typename T>
__global__ void __launch_bounds__(256) rows_proj_kernel(const T* dy, const float* b,
                                                        float* __restrict__ g, int M, int N, int rank) {
    __shared__ float red[8][64];
    pdl_launch_dependents();
    pdl_wait();
    dy = after_wait(dy);
    b = after_wait(b);
    const int m0 = blockIdx.x * kProjRows, j0 = blockIdx.y * kProjRanks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nb = static_cast<int>(static_cast<long long>(N) * blockIdx.z / gridDim.z);
    const int ne = static_cast<int>(static_cast<long long>(N) * (blockIdx.z + 1) / gridDim.z);
    float acc[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) acc[i] = 0.0f;
    for (int n = nb + threadIdx.x; n < ne; n += 256) {
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
        if (m0 + r < M && j0 + j < rank) g[(static_cast<size_t>(blockIdx.z) * M + m0 + r) * rank + j0 + j] = t;
    }
}

__device__ __forceinline__ void prefetch_l1(const float* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// One row's 128 k per block (blockIdx.y: row): the splits' sum, half of them
// per thread of a pair of warps, each in order; and with an adapter
// scale * (sum of G's ranges) A^T.
template <typename T>
__global__ void __launch_bounds__(256) rows_finish_kernel(const float* partial, int splits, long long split_floats,
                                                          const float* g, int gsplits, const float* a, int rank,
                                                          float scale, T* __restrict__ out, int M, int K) {
    __shared__ float gp[4][64], gs[64];
    __shared__ float half[128];
    pdl_launch_dependents();
    pdl_wait();
    partial = after_wait(partial);
    g = after_wait(g);
    a = after_wait(a);
    const long long row = blockIdx.y;
    const int c = threadIdx.x & 127, h = threadIdx.x >> 7, k = blockIdx.x * 128 + c;
    if (rank > 0) {
        // every fourth range of G per thread, and this thread's row of A on its way before either is needed
        const int j = threadIdx.x & 63, q = threadIdx.x >> 6;
        if (h == 0 && k < K) prefetch_l1(a + static_cast<size_t>(k) * rank);
        float t = 0.0f;
        if (j < rank) {
#pragma unroll 8
            for (int z = q; z < gsplits; z += 4) t += g[(static_cast<size_t>(z) * M + row) * rank + j];
        }
        gp[q][j] = t;
    }
    float v = 0.0f;
    if (k < K) {
        const float* p = partial + row * K + k;
        const int z1 = h == 0 ? (splits + 1) / 2 : splits;
#pragma unroll 8
        for (int z = h == 0 ? 0 : (splits + 1) / 2; z < z1; ++z) v += p[z * split_floats];
    }
    if (h == 1) half[c] = v;
    __syncthreads();
    if (rank > 0) {
        const int j = threadIdx.x;
        if (j < 64) gs[j] = scale * ((gp[0][j] + gp[1][j]) + (gp[2][j] + gp[3][j]));
        __syncthreads();
    }
    if (h == 1 || k >= K) return;
    v += half[c];
    if (rank > 0) {
        const float* ar = a + static_cast<size_t>(k) * rank;
        float l = 0.0f;
#pragma unroll 8
        for (int j = 0; j < rank; ++j) l = fmaf(gs[j], __ldg(ar + j), l);
        v += l;
    }
    row_store(out + row * K + k, v);
}

// Launch under the tail of the kernel before (programmatic dependent launch).
template <typename... Params, typename... Args>
int rows_launch(void (*kern)(Params...), dim3 grid, unsigned threads, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...));
}

// f with the row count as a constant, 1..8.
template <typename F>
int rows_dispatch(int M, F&& f) {
    switch (M) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        case 4: return f(std::integral_constant<int, 4>());
        case 5: return f(std::integral_constant<int, 5>());
        case 6: return f(std::integral_constant<int, 6>());
        case 7: return f(std::integral_constant<int, 7>());
        case 8: return f(std::integral_constant<int, 8>());
    }
    return static_cast<int>(cudaErrorInvalidValue);
}

}  // namespace

int rows_logits_tiles(int N) { return (N + kRowsCols - 1) / kRowsCols; }

int launch_rows_logits(const void* x, bool bf16, const uint32_t* packed, const float* scales, const long long* targets,
                       float* z, float* zt, float* smax, float* ssum, int M, int N, int K, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(rows_logits_tiles(N)));
    return rows_dispatch(M, [&](auto mr) {
        constexpr int MR = decltype(mr)::value;
        return bf16 ? rows_launch(rows_logits_kernel<MR, __nv_bfloat16>, grid, 256, stream,
                                  static_cast<const __nv_bfloat16*>(x), packed, scales, targets, z, zt, smax, ssum, N, K)
                    : rows_launch(rows_logits_kernel<MR, float>, grid, 256, stream, static_cast<const float*>(x), packed,
                                  scales, targets, z, zt, smax, ssum, N, K);
    });
}

int launch_rows_loss(const float* smax, const float* ssum, const float* zt, const long long* targets,
                     const float* row_scale, float* loss, float* lse, float* coef, int M, int N, cudaStream_t stream) {
    return rows_launch(rows_loss_kernel, dim3(static_cast<unsigned>(M)), 512, stream, smax, ssum, zt, targets, row_scale,
                       loss, lse, coef, N, rows_logits_tiles(N));
}

// Splits of n: about two blocks per SM (one wave), at least 32 n each.
int rows_wt_splits(int N, int K, int sm_count) {
    const long long blocks = (K / 8 + kWtWords - 1) / kWtWords;
    long long s = 2ll * sm_count / blocks;
    if (s > (N + 31) / 32) s = (N + 31) / 32;
    return static_cast<int>(s < 1 ? 1 : s);
}

int launch_rows_wt(const void* d, bool bf16, const float* coef, const long long* targets, const uint32_t* packed,
                   const float* scales, float* partial, int splits, int M, int N, int K, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>((K / 8 + kWtWords - 1) / kWtWords), static_cast<unsigned>(splits));
    return rows_dispatch(M, [&](auto mr) {
        constexpr int MR = decltype(mr)::value;
        return bf16 ? rows_launch(rows_wt_kernel<MR, __nv_bfloat16>, grid, kWtThreads, stream,
                                  static_cast<const __nv_bfloat16*>(d), coef, targets, packed, scales, partial, N, K)
                    : rows_launch(rows_wt_kernel<MR, float>, grid, kWtThreads, stream, static_cast<const float*>(d), coef,
                                  targets, packed, scales, partial, N, K);
    });
}

// Ranges of n per block of rows: enough blocks for the SMs, at least 256 n each.
int rows_proj_splits(int M, int N, int rank, int sm_count) {
    const long long blocks = static_cast<long long>((M + kProjRows - 1) / kProjRows) * ((rank + kProjRanks - 1) / kProjRanks);
    long long s = sm_count / blocks;
    if (s > N / 256) s = N / 256;
    return static_cast<int>(s < 1 ? 1 : s > 64 ? 64 : s);
}

int launch_rows_proj(const void* dy, bool bf16, const float* b, float* g, int splits, int M, int N, int rank,
                     cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>((M + kProjRows - 1) / kProjRows),
                    static_cast<unsigned>((rank + kProjRanks - 1) / kProjRanks), static_cast<unsigned>(splits));
    return bf16 ? rows_launch(rows_proj_kernel<__nv_bfloat16>, grid, 256, stream, static_cast<const __nv_bfloat16*>(dy), b, g,
                              M, N, rank)
                : rows_launch(rows_proj_kernel<float>, grid, 256, stream, static_cast<const float*>(dy), b, g, M, N, rank);
}

int launch_rows_finish(const float* partial, int splits, long long split_floats, const float* g, int gsplits,
                       const float* a, int rank, float scale, void* out, bool bf16, int M, int K, cudaStream_t stream) {
    if (M < 1 || M > 32768) return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>((K + 127) / 128), static_cast<unsigned>(M));
    return bf16 ? rows_launch(rows_finish_kernel<__nv_bfloat16>, grid, 256, stream, partial, splits, split_floats, g, gsplits,
                              a, rank, scale, static_cast<__nv_bfloat16*>(out), M, K)
                : rows_launch(rows_finish_kernel<float>, grid, 256, stream, partial, splits, split_floats, g, gsplits, a, rank,
                              scale, static_cast<float*>(out), M, K);
}

}  // namespace q4
