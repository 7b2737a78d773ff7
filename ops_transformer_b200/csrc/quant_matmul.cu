// quant_matmul: y = ((x w) * scale) * per_token_scale + bias of int8 matrices, without groups.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gmm_common.h"

namespace gmm {
namespace {

struct MatmulParams {
    const int8_t *x, *w;
    long long ld_x, ws_k, ws_n, ld_y;
    const void *scale, *bias;
    int scale_dtype, bias_dtype, y_dtype;
    const float *token_scale;
    void *y;
    int m, k, n;
};

__device__ __forceinline__ float load_as_float(const void *p, int dtype, long long i)
{
    if (dtype == kF32) return static_cast<const float *>(p)[i];
    if (dtype == kF16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// One result per thread.
__global__ void __launch_bounds__(256) quant_matmul_simple_kernel(const MatmulParams p)
{
    const long long c = (long long)blockIdx.x * 32 + threadIdx.x % 32, t = (long long)blockIdx.y * 8 + threadIdx.x / 32;
    if (c >= p.n || t >= p.m) return;
    const int8_t *x = p.x + t * p.ld_x, *w = p.w + c * p.ws_n;
    int acc = 0;
    for (int k = 0; k < p.k; ++k) acc += (int)x[k] * (int)w[k * p.ws_k];
    float v = __fmul_rn(__int2float_rn(acc), load_as_float(p.scale, p.scale_dtype, c));
    if (p.token_scale) v = __fmul_rn(v, p.token_scale[t]);
    if (p.bias) v = __fadd_rn(v, load_as_float(p.bias, p.bias_dtype, c));
    const long long at = t * p.ld_y + c;
    if (p.y_dtype == kF32) static_cast<float *>(p.y)[at] = v;
    else if (p.y_dtype == kF16) static_cast<__half *>(p.y)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p.y)[at] = __float2bfloat16_rn(v);
}

}  // namespace

size_t quant_matmul_workspace_bytes(const QuantMatmulProblem &) { return 256; }

cudaError_t quant_matmul_launch(const QuantMatmulProblem &q, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (q.m <= 0) return cudaSuccess;
    if (!workspace || workspace_bytes < quant_matmul_workspace_bytes(q)) return cudaErrorInvalidValue;
    const cudaError_t e = cudaMemsetAsync(workspace, 0, 256, stream);
    if (e != cudaSuccess) return e;
    MatmulParams p;
    p.x = q.x; p.w = q.w; p.ld_x = q.ld_x; p.ld_y = q.ld_y;
    p.ws_k = q.w_nk ? 1 : q.ld_w; p.ws_n = q.w_nk ? q.ld_w : 1;
    p.scale = q.scale; p.bias = q.bias; p.scale_dtype = q.scale_dtype; p.bias_dtype = q.bias_dtype; p.y_dtype = q.y_dtype;
    p.token_scale = q.token_scale; p.y = q.y;
    p.m = (int)q.m; p.k = (int)q.k; p.n = (int)q.n;
    for (long long t0 = 0; t0 < q.m; t0 += 65535ll * 8) {   // a grid's second dimension
        MatmulParams part = p;
        part.x += t0 * p.ld_x;
        if (p.token_scale) part.token_scale += t0;
        part.y = static_cast<char *>(p.y) + t0 * p.ld_y * (p.y_dtype == kF32 ? 4 : 2);
        part.m = (int)(q.m - t0 < 65535ll * 8 ? q.m - t0 : 65535ll * 8);
        quant_matmul_simple_kernel<<<dim3((unsigned)((q.n + 31) / 32), (unsigned)((part.m + 7) / 8)), 256, 0, stream>>>(part);
    }
    return cudaGetLastError();
}

}  // namespace gmm
