// sandwich_norm_quant: the norm behind a block, its gate, the scaled residual sum, and the norm in front of the next block in 8 bits.
//
//   n = x * rsqrt(mean(x^2) + post_eps) * post_gamma;  s = residual_scale * residual + block_scale * act(gate) * n
//   r = rsqrt(mean(s^2) + eps);  u = s * gamma (* smooth);  step = max|u| / 127;  q = rint(u / step);  scale = step * r
//
// r cancels in u / step, so the second norm's sum of squares and the largest |u| come out of one pass; the first norm's sum has to be there
// before.  Statistics, s and u are fp32; each output is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gmm_common.h"
#include "norm_common.h"

namespace gmm {
namespace {

struct SandwichParams {
    const void *x, *residual, *gamma, *post_gamma, *gate;
    const float *smooth;
    int8_t *q;
    float *scale;
    void *residual_out, *normed_out;
    long long ld_x, ld_residual, ld_gate, ld_q, ld_residual_out, ld_normed;
    int rows, h, gate_step, gate_act;
    bool gamma32;
    float inv_h, residual_scale, block_scale, eps, post_eps;
};

// The division's error is within 2 units, expf's within 1, and an exponential that overflows gives 0.
__device__ __forceinline__ float gate_value(float g, int act)
{
    if (act == kGateSigmoid) return __fdividef(1.0f, __fadd_rn(1.0f, expf(-g)));
    return act == kGateTanh ? tanhf(g) : g;
}

template <typename T>
__device__ __forceinline__ float load_gamma(const void *g, bool f32, int e)
{
    return f32 ? static_cast<const float *>(g)[e] : to_float<T>(static_cast<const T *>(g)[e]);
}

// Any strides, addresses and lengths: one element at a time, the inputs read anew in each of up to three passes.  Every thread stores only
// elements that it alone reads, behind its last look at them, so that outputs may be inputs.
template <typename T, typename X>
__global__ void __launch_bounds__(256) sandwich_any_kernel(const SandwichParams p)
{
    __shared__ float2 red[2][32];
    const long long row = blockIdx.x;
    const X *x = static_cast<const X *>(p.x) + row * p.ld_x;
    const T *residual = static_cast<const T *>(p.residual) + row * p.ld_residual, *gate = static_cast<const T *>(p.gate) + row * p.ld_gate;
    float norm = 1.0f;
    if (p.post_gamma) {
        float sum = 0.0f, unused = 0.0f;
        for (int e = threadIdx.x; e < p.h; e += 256) {
            const float v = to_float<X>(x[e]);
            sum = __fmaf_rn(v, v, sum);
        }
        block_reduce(sum, unused, red[0]);
        norm = rsqrtf(__fmaf_rn(sum, p.inv_h, p.post_eps));
    }
    const auto stream_at = [&](int e) {
        float n = to_float<X>(x[e]);
        if (p.post_gamma) n = __fmul_rn(__fmul_rn(n, norm), load_gamma<T>(p.post_gamma, p.gamma32, e));
        if (p.gate) n = __fmul_rn(n, gate_value(to_float<T>(gate[e * p.gate_step]), p.gate_act));
        return __fmaf_rn(p.residual_scale, to_float<T>(residual[e]), __fmul_rn(p.block_scale, n));
    };
    float r = 0.0f, step = 0.0f;
    if (p.gamma) {
        float sum = 0.0f, mag = 0.0f;
        for (int e = threadIdx.x; e < p.h; e += 256) {
            const float s = stream_at(e);
            sum = __fmaf_rn(s, s, sum);
            if (!p.q) continue;
            float u = __fmul_rn(s, load_gamma<T>(p.gamma, p.gamma32, e));
            if (p.smooth) u = __fmul_rn(u, p.smooth[e]);
            mag = max_mag(mag, u, u);
        }
        block_reduce(sum, mag, red[1]);
        r = rsqrtf(__fmaf_rn(sum, p.inv_h, p.eps));
        step = step_of(mag);
    }
    Quantiser quant;
    quant.set(step);
    if (p.q && threadIdx.x == 0) p.scale[row] = step == 0.0f ? 0.0f : __fmul_rn(step, r);
    for (int e = threadIdx.x; e < p.h; e += 256) {
        const float s = stream_at(e);
        if (p.residual_out) static_cast<T *>(p.residual_out)[row * p.ld_residual_out + e] = from_float<T>(s);
        if (!p.gamma) continue;
        float u = __fmul_rn(s, load_gamma<T>(p.gamma, p.gamma32, e));
        if (p.normed_out) static_cast<T *>(p.normed_out)[row * p.ld_normed + e] = from_float<T>(__fmul_rn(u, r));
        if (p.smooth) u = __fmul_rn(u, p.smooth[e]);
        if (p.q) p.q[row * p.ld_q + e] = (int8_t)quant.one(u);
    }
}

template <typename T, typename X>
cudaError_t launch_typed(const SandwichParams &p, cudaStream_t stream)
{
    sandwich_any_kernel<T, X><<<p.rows, 256, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t sandwich_norm_launch(const SandwichNormProblem &n, cudaStream_t stream)
{
    if (n.rows <= 0) return cudaSuccess;
    SandwichParams p;
    p.x = n.x; p.residual = n.residual; p.gamma = n.gamma; p.post_gamma = n.post_gamma; p.gate = n.gate; p.smooth = n.smooth;
    p.q = n.q; p.scale = n.scale; p.residual_out = n.residual_out; p.normed_out = n.normed_out;
    p.ld_x = n.ld_x; p.ld_residual = n.ld_residual; p.ld_gate = n.ld_gate; p.ld_q = n.ld_q; p.ld_residual_out = n.ld_residual_out;
    p.ld_normed = n.ld_normed;
    p.rows = (int)n.rows; p.h = (int)n.h; p.gate_step = n.gate_step; p.gate_act = n.gate_act;
    p.gamma32 = n.gamma_dtype == kF32;
    p.inv_h = 1.0f / (float)n.h; p.residual_scale = n.residual_scale; p.block_scale = n.block_scale; p.eps = n.eps; p.post_eps = n.post_eps;
    switch (n.dtype) {
        case kF32: return launch_typed<float, float>(p, stream);
        case kF16: return n.x_dtype == kF32 ? launch_typed<__half, float>(p, stream) : launch_typed<__half, __half>(p, stream);
        case kBF16: return n.x_dtype == kF32 ? launch_typed<__nv_bfloat16, float>(p, stream) : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace gmm
