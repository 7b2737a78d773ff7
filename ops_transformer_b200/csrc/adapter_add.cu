// adapter_add: low-rank adapters of many requests on top of a projection that they share.
//
//   out[t] = base[t] + scaling[i] * (x[t] a[i]^T) b[i]^T,  i = ids[t]
//
// Two kernels: v[t] = scaling * x[t] a[i]^T in fp32 (workspace), then out[t] = base[t] + v[t] b[i]^T, rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gmm_common.h"

namespace gmm {
namespace {

struct AdapterParams {
    const void *base, *x, *a, *b;
    const float *x_scale, *scaling;
    const int *ids;
    void *out;
    float *v;                       // [rows, rank]
    long long ld_base, ld_x, ld_out;
    int rows, k, n, adapters, rank;
};

__device__ __forceinline__ float to_float(int8_t v) { return (float)v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One warp per (row, rank component).
template <typename T, typename X>
__global__ void __launch_bounds__(128) adapter_shrink_kernel(const AdapterParams p)
{
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (at >= (long long)p.rows * p.rank) return;
    const int row = (int)(at / p.rank), j = (int)(at % p.rank);
    const int i = p.ids[row];
    if (i < 0 || i >= p.adapters) return;
    const X *x = reinterpret_cast<const X *>(p.x) + row * p.ld_x;
    const T *a = reinterpret_cast<const T *>(p.a) + ((long long)i * p.rank + j) * p.k;
    float sum = 0.0f;
    for (int c = lane; c < p.k; c += 32) sum = __fmaf_rn(to_float(x[c]), to_float(a[c]), sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
        if (p.x_scale) sum = __fmul_rn(sum, p.x_scale[row]);
        if (p.scaling) sum = __fmul_rn(sum, p.scaling[i]);
        p.v[at] = sum;
    }
}

// One CTA per row and 128 columns.
template <typename T>
__global__ void __launch_bounds__(128) adapter_expand_kernel(const AdapterParams p)
{
    const int row = blockIdx.x, c = blockIdx.y * 128 + threadIdx.x;
    if (c >= p.n) return;
    const int i = p.ids[row];
    float sum = to_float(reinterpret_cast<const T *>(p.base)[row * p.ld_base + c]);
    if (i >= 0 && i < p.adapters) {
        const T *b = reinterpret_cast<const T *>(p.b) + ((long long)i * p.n + c) * p.rank;
        const float *v = p.v + (long long)row * p.rank;
        float delta = 0.0f;
        for (int j = 0; j < p.rank; ++j) delta = __fmaf_rn(v[j], to_float(b[j]), delta);
        sum = __fadd_rn(sum, delta);
    }
    reinterpret_cast<T *>(p.out)[row * p.ld_out + c] = from_float<T>(sum);
}

template <typename T>
cudaError_t launch_typed(const AdapterParams &p, bool x_i8, cudaStream_t stream)
{
    const long long dots = (long long)p.rows * p.rank;
    if (x_i8) adapter_shrink_kernel<T, int8_t><<<(unsigned)((dots + 3) / 4), 128, 0, stream>>>(p);
    else adapter_shrink_kernel<T, T><<<(unsigned)((dots + 3) / 4), 128, 0, stream>>>(p);
    adapter_expand_kernel<T><<<dim3((unsigned)p.rows, (unsigned)((p.n + 127) / 128)), 128, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

size_t adapter_workspace_bytes(const AdapterProblem &p) { return 256 + ((size_t)p.rows * p.rank * 4 + 255) / 256 * 256; }

cudaError_t adapter_launch(const AdapterProblem &a, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (a.rows <= 0) return cudaSuccess;
    if (!workspace || workspace_bytes < adapter_workspace_bytes(a)) return cudaErrorInvalidValue;
    AdapterParams p;
    p.base = a.base; p.x = a.x; p.a = a.a; p.b = a.b;
    p.x_scale = a.x_scale; p.scaling = a.scaling; p.ids = a.ids; p.out = a.out;
    p.v = reinterpret_cast<float *>(static_cast<char *>(workspace) + 256);
    p.ld_base = a.ld_base; p.ld_x = a.ld_x; p.ld_out = a.ld_out;
    p.rows = (int)a.rows; p.k = (int)a.k; p.n = (int)a.n; p.adapters = (int)a.adapters; p.rank = (int)a.rank;
    return a.dtype == kF16 ? launch_typed<__half>(p, a.x_i8, stream) : launch_typed<__nv_bfloat16>(p, a.x_i8, stream);
}

}  // namespace gmm
