// add_rms_norm_quant: the residual's addition, the root-mean-square norm and the per-token int8 quantisation of a row in one pass.
//
//   h = x + residual;  r = 1 / sqrt(mean(h^2) + eps);  u = h * gamma (* smooth);  step = max|u| / 127
//   q = rint(u / step);  scale = step * r;  residual_out = h;  normed_out = h * r * gamma
//
// The int8 value of h * r * gamma * smooth at its own scale does not depend on r, which is one number for the row: u / step is the
// quotient with r cancelled.  So the sum of squares and the maximum come out of the same pass over the registers and one block
// reduction serves both, and q does not hang on the order in which the squares are summed.  The sum, the statistics and u are fp32;
// each output is rounded once.
//
// Bound by memory: x and residual are read once, every output is written once.  A row stays in registers between the reduction and
// the stores.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gmm_common.h"

namespace gmm {
namespace {

struct NormParams {
    const void *x, *residual, *gamma;
    const float *smooth;
    int8_t *q;
    float *scale;
    void *residual_out, *normed_out;
    long long ld_x, ld_residual, ld_q, ld_residual_out, ld_normed;
    int rows, h;
    float eps;
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements at once: one load or store of N * sizeof(T) bytes, which p is aligned to.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack { T v[N]; };

template <typename T, int N>
__device__ __forceinline__ void load_floats(const void *base, long long at, float (&f)[N])
{
    const Pack<T, N> p = *reinterpret_cast<const Pack<T, N> *>(reinterpret_cast<const T *>(base) + at);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_float<T>(p.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_floats(void *base, long long at, const float (&f)[N])
{
    Pack<T, N> p;
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = from_float<T>(f[i]);
    *reinterpret_cast<Pack<T, N> *>(reinterpret_cast<T *>(base) + at) = p;
}

// Sum of `sum` and largest of `mag` (bits of magnitudes: as unsigned numbers they order like them, and a NaN is the largest of all,
// so that it is not passed over) of the block, in every thread.
template <int THREADS>
__device__ __forceinline__ void block_reduce(float &sum, uint32_t &mag, float2 *red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    mag = __reduce_max_sync(0xffffffffu, mag);
    if (THREADS == 32) return;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(sum, __uint_as_float(mag));
    __syncthreads();
    constexpr int W = THREADS / 32;
    const float2 v = red[(threadIdx.x & 31) % W];
    sum = v.x;
    mag = __float_as_uint(v.y);
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    mag = __reduce_max_sync(0xffffffffu, mag);
}

// rint(u / step), 0 where there is no step to divide by.
__device__ __forceinline__ int quantise(float u, float step)
{
    if (!(step > 0.0f && step < __int_as_float(0x7f800000))) return 0;
    return max(-127, min(127, __float2int_rn(__fdiv_rn(u, step))));
}

// One CTA per row.  A thread holds NCH packs of V elements, THREADS packs apart; REG: the row fits, else it is read again.
template <typename T, typename G, int V, int NCH, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_quant_kernel(const NormParams p)
{
    __shared__ float2 red[THREADS / 32];
    const long long row = blockIdx.x;
    const int packs = p.h / V;
    float h[NCH][V];
    float sum = 0.0f;
    uint32_t mag = 0;
    for (int c0 = 0; c0 < packs; c0 += THREADS * NCH) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = c0 + i * THREADS + threadIdx.x;
            if (c >= packs) break;
            load_floats<T, V>(p.x, row * p.ld_x + (long long)c * V, h[i]);
            if (p.residual) {
                float t[V];
                load_floats<T, V>(p.residual, row * p.ld_residual + (long long)c * V, t);
#pragma unroll
                for (int e = 0; e < V; ++e) h[i][e] = __fadd_rn(h[i][e], t[e]);
            }
            float g[V];
            load_floats<G, V>(p.gamma, (long long)c * V, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float u = __fmul_rn(h[i][e], g[e]);
                if (p.smooth) u = __fmul_rn(u, p.smooth[c * V + e]);
                sum = __fmaf_rn(h[i][e], h[i][e], sum);
                mag = max(mag, __float_as_uint(u) & 0x7fffffffu);
            }
        }
    }
    block_reduce<THREADS>(sum, mag, red);
    const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)p.h), p.eps)));
    const float step = __fdiv_rn(__uint_as_float(mag), 127.0f);
    if (threadIdx.x == 0) p.scale[row] = step == 0.0f ? 0.0f : __fmul_rn(step, r);
    const bool again = packs > THREADS * NCH;
    for (int c0 = 0; c0 < packs; c0 += THREADS * NCH) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = c0 + i * THREADS + threadIdx.x;
            if (c >= packs) break;
            if (again) {
                load_floats<T, V>(p.x, row * p.ld_x + (long long)c * V, h[i]);
                if (p.residual) {
                    float t[V];
                    load_floats<T, V>(p.residual, row * p.ld_residual + (long long)c * V, t);
#pragma unroll
                    for (int e = 0; e < V; ++e) h[i][e] = __fadd_rn(h[i][e], t[e]);
                }
            }
            float g[V], y[V];
            Pack<int8_t, V> q;
            load_floats<G, V>(p.gamma, (long long)c * V, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float u = __fmul_rn(h[i][e], g[e]);
                y[e] = __fmul_rn(u, r);
                if (p.smooth) u = __fmul_rn(u, p.smooth[c * V + e]);
                q.v[e] = (int8_t)quantise(u, step);
            }
            *reinterpret_cast<Pack<int8_t, V> *>(p.q + row * p.ld_q + (long long)c * V) = q;
            if (p.residual_out) store_floats<T, V>(p.residual_out, row * p.ld_residual_out + (long long)c * V, h[i]);
            if (p.normed_out) store_floats<T, V>(p.normed_out, row * p.ld_normed + (long long)c * V, y);
        }
    }
}

template <typename T, typename G, int V>
void launch_rows(const NormParams &p, cudaStream_t stream)
{
    norm_quant_kernel<T, G, V, 4, 256><<<p.rows, 256, 0, stream>>>(p);
}

template <typename T, typename G>
void launch_typed(const NormParams &p, cudaStream_t stream)
{
    constexpr int V = 16 / (int)sizeof(T);
    // 16 bytes of T and V bytes of q at a time, where every row of every tensor starts on such a boundary
    const auto fits = [](const void *base, long long ld, int bytes, int align) {
        return !base || (((uintptr_t)base | (uintptr_t)(ld * bytes)) & (uintptr_t)(align - 1)) == 0;
    };
    const bool wide = p.h % V == 0 && fits(p.x, p.ld_x, sizeof(T), 16) && fits(p.residual, p.ld_residual, sizeof(T), 16) &&
                      fits(p.residual_out, p.ld_residual_out, sizeof(T), 16) && fits(p.normed_out, p.ld_normed, sizeof(T), 16) &&
                      fits(p.gamma, 0, 0, V * (int)sizeof(G)) && fits(p.smooth, 0, 0, 16) && fits(p.q, p.ld_q, 1, V);
    if (wide) launch_rows<T, G, V>(p, stream);
    else launch_rows<T, G, 1>(p, stream);
}

}  // namespace

cudaError_t norm_quant_launch(const NormQuantProblem &n, cudaStream_t stream)
{
    if (n.rows <= 0) return cudaSuccess;
    NormParams p;
    p.x = n.x; p.residual = n.residual; p.gamma = n.gamma; p.smooth = n.smooth;
    p.q = n.q; p.scale = n.scale; p.residual_out = n.residual_out; p.normed_out = n.normed_out;
    p.ld_x = n.ld_x; p.ld_residual = n.ld_residual; p.ld_q = n.ld_q; p.ld_residual_out = n.ld_residual_out; p.ld_normed = n.ld_normed;
    p.rows = (int)n.rows; p.h = (int)n.h; p.eps = n.eps;
    const bool g32 = n.gamma_dtype == kF32;
    switch (n.dtype) {
        case kF32: launch_typed<float, float>(p, stream); break;
        case kF16: g32 ? launch_typed<__half, float>(p, stream) : launch_typed<__half, __half>(p, stream); break;
        case kBF16: g32 ? launch_typed<__nv_bfloat16, float>(p, stream) : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, stream); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace gmm
