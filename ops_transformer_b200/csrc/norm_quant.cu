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
// Bound by memory where there are many rows: x and residual are read once, every output is written once, and a row stays in registers
// between the reduction and the stores.  4096 x 7168 bf16 with a residual and all outputs: 264 MB in 47.5 us, 5.6 TB/s, where a copy on
// the same GPU reaches 6.6.  Without residual and the 16-bit outputs 33 us, 2.6 TB/s: 22.9 million instructions against 29.8 for three
// times the bytes, in two thirds of the issue slots, with the stalls spread over arithmetic and the block's barrier.  Few rows cost a row's
// chain of load, reduction and store: 16 x 7168 3.4 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "gmm_common.h"
#include "norm_common.h"

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
    float inv_h, eps;
};

__device__ __forceinline__ float rms_scale(float sum, const NormParams &p) { return rsqrtf(__fmaf_rn(sum, p.inv_h, p.eps)); }

// One CTA per row; a thread holds NCH packs of 16 bytes, blockDim.x apart, in fp32 between the reduction and the stores (rows that do
// not fit are read again).  WHOLE: rows start on packs.  Else every row starts `lead` elements into one, the same in all tensors (their
// rows are equally far apart, counted in elements modulo a pack), and only the stores of its first and last pack go one element at a time.
//
// STREAM: the CTA takes every gridDim.x-th row (which fits).  While it works on one, the packs of the next are copied to shared memory,
// each by the thread that will read it, so nothing but the thread's own copies is waited for and loads are under way all the time.
// 4096 x 7168: 47.5 us, 64 without; 16384 x 512: 15.8, 17.5; rows on no boundary, whose masks cost instructions, 4096 x 5001: 61, 63.
template <typename T, typename G, int NCH, bool WHOLE, int MAXT, int MINB, bool STREAM>
__global__ void __launch_bounds__(MAXT, MINB) norm_quant_kernel(const NormParams p)
{
    constexpr int V = 16 / (int)sizeof(T);
    extern __shared__ uint4 ahead[];   // STREAM: [2][NCH][threads]
    __shared__ float2 red[2][32];
    const int threads = blockDim.x;
    const G *gamma = reinterpret_cast<const G *>(p.gamma);
    const uint32_t mine = STREAM ? (uint32_t)__cvta_generic_to_shared(ahead) + threadIdx.x * 16 : 0;
    const auto lead_of = [&](long long row) { return WHOLE ? 0 : (int)((row * p.ld_x) & (V - 1)); };
    // Elements from the row's first pack on that lie inside x and residual: a row's first and last pack hold elements of its neighbours
    // (or what is between the rows), which are read with it and dropped, but behind the tensor's end there may be nothing to read.
    const auto room_of = [&](long long row, int lead) {
        const long long behind = (p.rows - 1 - row) * (p.residual ? min(p.ld_x, p.ld_residual) : p.ld_x);
        return lead + p.h + (int)min(behind, 1024ll);
    };
    const auto fetch = [&](long long row) {
        const int lead = lead_of(row), room = room_of(row, lead);
        const T *x = reinterpret_cast<const T *>(p.x) + row * p.ld_x - lead, *res = reinterpret_cast<const T *>(p.residual) + row * p.ld_residual - lead;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = threadIdx.x + i * threads;
            if (WHOLE ? c * V < p.h : c * V < lead + p.h && (c + 1) * V <= room) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + i * threads * 16), "l"(x + (long long)c * V) : "memory");
                if (p.residual)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + (NCH + i) * threads * 16), "l"(res + (long long)c * V) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (STREAM) fetch(blockIdx.x);
    int parity = 0;
    for (long long row = blockIdx.x; row < p.rows; row += STREAM ? (long long)gridDim.x : (long long)p.rows) {
        const int lead = lead_of(row), end = lead + p.h, room = room_of(row, lead);
        const int packs = (end + V - 1) / V;
        const bool again = !STREAM && packs > threads * NCH;
        const T *x = reinterpret_cast<const T *>(p.x) + row * p.ld_x - lead;
        const T *residual = reinterpret_cast<const T *>(p.residual) + row * p.ld_residual - lead;
        T *residual_out = reinterpret_cast<T *>(p.residual_out) + row * p.ld_residual_out - lead;
        T *normed_out = reinterpret_cast<T *>(p.normed_out) + row * p.ld_normed - lead;
        int8_t *q_out = p.q + row * p.ld_q - lead;
        const auto full = [&](int c) { return WHOLE || (c * V >= lead && (c + 1) * V <= end); };
        const auto get = [&](const T *from, int c, int at) {
            if (!WHOLE && (c + 1) * V > room) {
                const auto one = [&](int e) { return c * V + e >= lead && c * V + e < end ? to_float<T>(from[c * V + e]) : 0.0f; };
                f32x2 f[V / 2];
#pragma unroll
                for (int e = 0; e < V; e += 2) f[e / 2] = pair2(one(e), one(e + 1));
                return pack<T>(f);   // exact: the values come from T
            }
            uint4 u;
            if (STREAM) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(mine + at * threads * 16) : "memory");
            else u = *reinterpret_cast<const uint4 *>(from + (long long)c * V);
            return u;
        };
        const auto load_h = [&](int c, int i, f32x2 *h) {
            unpack<T>(get(x, c, i), h);
            if (p.residual) {
                f32x2 t[V / 2];
                unpack<T>(get(residual, c, NCH + i), t);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) h[e] = fma2(h[e], pair2(1.0f, 1.0f), t[e]);
            }
            if (!full(c)) {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const float2 v = unpair2(h[e / 2]);
                    h[e / 2] = pair2(c * V + e >= lead && c * V + e < end ? v.x : 0.0f, c * V + e + 1 >= lead && c * V + e + 1 < end ? v.y : 0.0f);
                }
            }
        };
        // h * gamma in the place of h
        const auto weigh = [&](int c, f32x2 *h) {
            f32x2 g[V / 2];
            if constexpr (!WHOLE) load_anywhere<G, V>(gamma, c * V - lead, p.h, g);
            else if constexpr (sizeof(G) == 4) load_fp32<V>(gamma + c * V, g);
            else unpack<G>(__ldg(reinterpret_cast<const uint4 *>(gamma + c * V)), g);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) h[e] = mul2(h[e], g[e]);
        };
        const auto smooth = [&](int c, const f32x2 *u, f32x2 *to) {
            f32x2 m[V / 2];
            if constexpr (WHOLE) load_fp32<V>(p.smooth + c * V, m);
            else load_anywhere<float, V>(p.smooth, c * V - lead, p.h, m);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) to[e] = mul2(u[e], m[e]);
        };
        const auto store = [&](T *to, int c, const f32x2 *f) {
            if (full(c)) {
                *reinterpret_cast<uint4 *>(to + (long long)c * V) = pack<T>(f);
                return;
            }
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c * V + e >= lead && c * V + e < end) to[c * V + e] = from_float<T>(element(f, e));
        };
        f32x2 u[NCH][V / 2];
        f32x2 sum2 = 0;
        float mag = 0.0f;
        if (STREAM) asm volatile("cp.async.wait_group 0;" ::: "memory");
        // A row that streams fits: one turn, which threads without a pack of it take too, since the next row may have one for them.
        for (int c0 = threadIdx.x; c0 < packs || (STREAM && c0 < threads); c0 += threads * NCH) {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                if (c0 + i * threads < packs) load_h(c0 + i * threads, i, u[i]);
            }
            if (STREAM && row + gridDim.x < p.rows) fetch(row + gridDim.x);   // the thread has read what this fills
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int c = c0 + i * threads;
                if (c >= packs) break;
#pragma unroll
                for (int e = 0; e < V / 2; ++e) sum2 = fma2(u[i][e], u[i][e], sum2);
                // a row that is read again keeps its inputs, which residual_out may be, until then
                if (p.residual_out && !again) store(residual_out, c, u[i]);
                weigh(c, u[i]);
                f32x2 m[V / 2];
#pragma unroll
                for (int e = 0; e < V / 2; ++e) m[e] = u[i][e];
                if (p.smooth) smooth(c, u[i], m);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 v = unpair2(m[e]);
                    mag = max_mag(mag, v.x, v.y);
                }
            }
        }
        const float2 parts = unpair2(sum2);
        float sum = parts.x + parts.y;
        block_reduce(sum, mag, red[parity]);
        parity ^= 1;
        const float r = rms_scale(sum, p), step = step_of(mag);
        Quantiser quant;
        quant.set(step);
        if (threadIdx.x == 0) p.scale[row] = step == 0.0f ? 0.0f : __fmul_rn(step, r);
        const auto finish = [&](bool by_rcp) {
            for (int c0 = threadIdx.x; c0 < packs; c0 += threads * NCH) {
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const int c = c0 + i * threads;
                    if (c >= packs) break;
                    if (again) {
                        load_h(c, i, u[i]);
                        if (p.residual_out) store(residual_out, c, u[i]);
                        weigh(c, u[i]);
                    }
                    if (p.normed_out) {
                        f32x2 y[V / 2];
#pragma unroll
                        for (int e = 0; e < V / 2; ++e) y[e] = mul2(u[i][e], pair2(r, r));
                        store(normed_out, c, y);
                    }
                    if (p.smooth) smooth(c, u[i], u[i]);
                    uint32_t q[V / 4];
#pragma unroll
                    for (int e = 0; e < V / 4; ++e) q[e] = quant.four(u[i] + 2 * e, by_rcp);
                    int8_t *to = q_out + (long long)c * V;
                    if (full(c)) {
                        if (V == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(q[0], q[V / 4 - 1]);
                        else *reinterpret_cast<uint32_t *>(to) = q[0];
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            if (c * V + e >= lead && c * V + e < end) to[e] = (int8_t)(q[e / 4] >> (e % 4 * 8));
                    }
                }
            }
        };
        if (quant.rcp != 0.0f) finish(true);
        else finish(false);
    }
}

// Any strides and addresses: one element at a time.
template <typename T, typename G>
__global__ void __launch_bounds__(256) norm_quant_any_kernel(const NormParams p)
{
    __shared__ float2 red[32];
    const long long row = blockIdx.x;
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.ld_x, *residual = reinterpret_cast<const T *>(p.residual) + row * p.ld_residual;
    const G *gamma = reinterpret_cast<const G *>(p.gamma);
    const auto load = [&](int e) { return p.residual ? __fadd_rn(to_float<T>(x[e]), to_float<T>(residual[e])) : to_float<T>(x[e]); };
    float sum = 0.0f, mag = 0.0f;
    for (int e = threadIdx.x; e < p.h; e += 256) {
        const float h = load(e);
        float u = __fmul_rn(h, to_float<G>(gamma[e]));
        if (p.smooth) u = __fmul_rn(u, p.smooth[e]);
        sum = __fmaf_rn(h, h, sum);
        mag = max_mag(mag, u, u);
    }
    block_reduce(sum, mag, red);
    const float r = rms_scale(sum, p), step = step_of(mag);
    Quantiser quant;
    quant.set(step);
    if (threadIdx.x == 0) p.scale[row] = step == 0.0f ? 0.0f : __fmul_rn(step, r);
    for (int e = threadIdx.x; e < p.h; e += 256) {
        const float h = load(e);
        float u = __fmul_rn(h, to_float<G>(gamma[e]));
        if (p.residual_out) reinterpret_cast<T *>(p.residual_out)[row * p.ld_residual_out + e] = from_float<T>(h);
        if (p.normed_out) reinterpret_cast<T *>(p.normed_out)[row * p.ld_normed + e] = from_float<T>(__fmul_rn(u, r));
        if (p.smooth) u = __fmul_rn(u, p.smooth[e]);
        p.q[row * p.ld_q + e] = (int8_t)quant.one(u);
    }
}

template <typename T, typename G, bool WHOLE>
void launch_packed(const NormParams &p, cudaStream_t stream)
{
    constexpr int V = 16 / (int)sizeof(T);
    const int packs = (p.h + (WHOLE ? 0 : V - 1) + V - 1) / V;
    const auto warps = [](int n) { return (n + 31) / 32 * 32; };
    // Few rows: as many threads as a row has packs, for the shortest chain (16 x 7168: 3.4 us, 4.7 with four packs a thread).  More: four
    // packs a thread, for more rows on an SM (400 x 7168: 7.1 us, 8.7 with one); from more rows than find a place on the SMs together on,
    // the CTAs go through them with the next row's loads under way.
    const int four = warps((packs + 3) / 4), smem = 2 * 4 * 16 * four;
    const int fit = 1024 / four < 200 * 1024 / (smem + 1024) ? 1024 / four : 200 * 1024 / (smem + 1024), places = 148 * fit;
    if (packs <= 4 * 256 && p.rows > places) {
        const auto kernel = norm_quant_kernel<T, G, 4, WHOLE, 256, 4, true>;
        kernel<<<places, four, smem, stream>>>(p);
    } else if (packs <= 1024 && (p.rows <= 2 * 148 || packs <= 64)) norm_quant_kernel<T, G, 1, WHOLE, 1024, 1, false><<<p.rows, warps(packs), 0, stream>>>(p);
    else if (packs <= 4 * 256) norm_quant_kernel<T, G, 4, WHOLE, 256, 3, false><<<p.rows, four, 0, stream>>>(p);
    else norm_quant_kernel<T, G, 4, WHOLE, 1024, 1, false><<<p.rows, packs >= 4096 ? 1024 : four, 0, stream>>>(p);
}

template <typename T, typename G>
void launch_typed(const NormParams &p, cudaStream_t stream)
{
    constexpr int V = 16 / (int)sizeof(T);
    // Packs need every tensor to begin on one (V elements of its own type) and its rows to be as far apart as x's, modulo a pack.
    const auto fits = [&](const void *base, long long ld, int bytes) {
        return !base || (((uintptr_t)base & (uintptr_t)(V * bytes < 16 ? V * bytes - 1 : 15)) == 0 && (ld - p.ld_x) % V == 0);
    };
    const bool packed = fits(p.x, p.ld_x, sizeof(T)) && fits(p.residual, p.ld_residual, sizeof(T)) && fits(p.residual_out, p.ld_residual_out, sizeof(T)) &&
                        fits(p.normed_out, p.ld_normed, sizeof(T)) && fits(p.q, p.ld_q, 1) && fits(p.gamma, p.ld_x, sizeof(G)) &&
                        fits(p.smooth, p.ld_x, 4);
    if (!packed) norm_quant_any_kernel<T, G><<<p.rows, 256, 0, stream>>>(p);
    else if (p.h % V == 0 && p.ld_x % V == 0) launch_packed<T, G, true>(p, stream);
    else launch_packed<T, G, false>(p, stream);
}

}  // namespace

cudaError_t norm_quant_launch(const NormQuantProblem &n, cudaStream_t stream)
{
    if (n.rows <= 0) return cudaSuccess;
    NormParams p;
    p.x = n.x; p.residual = n.residual; p.gamma = n.gamma; p.smooth = n.smooth;
    p.q = n.q; p.scale = n.scale; p.residual_out = n.residual_out; p.normed_out = n.normed_out;
    p.ld_x = n.ld_x; p.ld_residual = n.ld_residual; p.ld_q = n.ld_q; p.ld_residual_out = n.ld_residual_out; p.ld_normed = n.ld_normed;
    p.rows = (int)n.rows; p.h = (int)n.h; p.inv_h = 1.0f / (float)n.h; p.eps = n.eps;
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
