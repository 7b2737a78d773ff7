// sandwich_norm_quant: the norm behind a block, its gate, the scaled residual sum, and the norm in front of the next block in 8 bits.
//
//   n = x * rsqrt(mean(x^2) + post_eps) * post_gamma;  s = residual_scale * residual + block_scale * act(gate) * n
//   r = rsqrt(mean(s^2) + eps);  u = s * gamma (* smooth);  step = max|u| / 127;  q = rint(u / step);  scale = step * r
//
// r cancels in u / step, so the second norm's sum of squares and the largest |u| come out of one pass; the first norm's sum has to be there
// before.  Statistics, s and u are fp32; each output is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dependent.h"
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
    // of the kernel with waits
    int fetched;                // rows whose copies are made: all but in a test
    bool clear_status;          // else it has been, before the launch
    long long wait_limit;
    int *status;
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

// The status record, by a call's first block.  That is among the first to start, and a wait of the default limit runs out about a second after.
// (A store under a predicate: behind a branch it costs the kernel of many rows registers, 4096 x 7168 54.4 us for 53.4.)
__device__ __forceinline__ void clear_status(const SandwichParams &p)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.eq.u32 p, %1, 0;\n"
        "@p st.global.v4.b32 [%0], {%2, %2, %2, %2};\n"
        "}\n" ::"l"(p.status), "r"(blockIdx.x | threadIdx.x | !p.clear_status), "r"(0));
}

// Any strides, addresses and lengths: one element at a time, the inputs read anew in each of up to three passes.  Every thread stores only
// elements that it alone reads, behind its last look at them, so that outputs may be inputs.
template <typename T, typename X>
__global__ void __launch_bounds__(256) sandwich_any_kernel(const SandwichParams p)
{
    __shared__ float2 red[2][32];
    dependent_wait();
    dependent_release();
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
    if (threadIdx.x == 0) {
        if (p.q) p.scale[row] = step == 0.0f ? 0.0f : __fmul_rn(step, r);
        if (row == 0 && p.clear_status) *reinterpret_cast<int4 *>(p.status) = make_int4(0, 0, 0, 0);
    }
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

// The same for few rows, in batches of loads that wait for nothing between them.
template <typename T, typename X>
__global__ void __launch_bounds__(1024, 1) sandwich_any_few_kernel(const SandwichParams p)
{
    constexpr int N = 4;    // elements of a batch
    __shared__ float2 red[2][32];
    dependent_wait();
    dependent_release();
    clear_status(p);
    const long long row = blockIdx.x;
    const int threads = blockDim.x;
    const X *x = static_cast<const X *>(p.x) + row * p.ld_x;
    const T *residual = static_cast<const T *>(p.residual) + row * p.ld_residual, *gate = static_cast<const T *>(p.gate) + row * p.ld_gate;
    float norm = 1.0f;
    if (p.post_gamma) {
        float sum = 0.0f, unused = 0.0f;
        for (int e0 = threadIdx.x; e0 < p.h; e0 += N * threads) {
            float v[N];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = e0 + i * threads < p.h ? to_float<X>(x[e0 + i * threads]) : 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) sum = __fmaf_rn(v[i], v[i], sum);
        }
        block_reduce(sum, unused, red[0]);
        norm = rsqrtf(__fmaf_rn(sum, p.inv_h, p.post_eps));
    }
    // A batch of the stream and of what multiplies it behind the norm; all loads come before the first conversion.
    float s[N], g[N], m[N];
    const auto load = [&](int e0) {
        const auto at = [&](int i) { return min(e0 + i * threads, p.h - 1); };   // what is beyond the row is loaded for nothing
        X xs[N];
        T rs[N], gates[N], post[N], next[N];
        float post32[N], next32[N];
#pragma unroll
        for (int i = 0; i < N; ++i) xs[i] = x[at(i)];
#pragma unroll
        for (int i = 0; i < N; ++i) rs[i] = residual[at(i)];
        const auto load_gammas = [&](const void *from, T (&v)[N], float (&v32)[N]) {
            if (!from) return;
            if (p.gamma32) {
#pragma unroll
                for (int i = 0; i < N; ++i) v32[i] = static_cast<const float *>(from)[at(i)];
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = static_cast<const T *>(from)[at(i)];
            }
        };
        load_gammas(p.post_gamma, post, post32);
        load_gammas(p.gamma, next, next32);
        if (p.gate) {
#pragma unroll
            for (int i = 0; i < N; ++i) gates[i] = gate[at(i) * p.gate_step];
        }
        if (p.smooth) {
#pragma unroll
            for (int i = 0; i < N; ++i) m[i] = p.smooth[at(i)];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float n = to_float<X>(xs[i]);
            if (p.post_gamma) n = __fmul_rn(__fmul_rn(n, norm), p.gamma32 ? post32[i] : to_float<T>(post[i]));
            if (p.gate) n = __fmul_rn(n, gate_value(to_float<T>(gates[i]), p.gate_act));
            s[i] = __fmaf_rn(p.residual_scale, to_float<T>(rs[i]), __fmul_rn(p.block_scale, n));
            g[i] = p.gamma32 ? next32[i] : to_float<T>(next[i]);
        }
    };
    float r = 0.0f, step = 0.0f;
    if (p.gamma) {
        float sum = 0.0f, mag = 0.0f;
        for (int e0 = threadIdx.x; e0 < p.h; e0 += N * threads) {
            load(e0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (e0 + i * threads >= p.h) break;
                sum = __fmaf_rn(s[i], s[i], sum);
                const float u = p.smooth ? __fmul_rn(__fmul_rn(s[i], g[i]), m[i]) : __fmul_rn(s[i], g[i]);
                if (p.q) mag = max_mag(mag, u, u);
            }
        }
        block_reduce(sum, mag, red[1]);
        r = rsqrtf(__fmaf_rn(sum, p.inv_h, p.eps));
        step = step_of(mag);
    }
    Quantiser quant;
    quant.set(step);
    if (p.q && threadIdx.x == 0) p.scale[row] = step == 0.0f ? 0.0f : __fmul_rn(step, r);
    for (int e0 = threadIdx.x; e0 < p.h; e0 += N * threads) {
        load(e0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = e0 + i * threads;
            if (e >= p.h) break;
            if (p.residual_out) static_cast<T *>(p.residual_out)[row * p.ld_residual_out + e] = from_float<T>(s[i]);
            if (!p.gamma) continue;
            float u = __fmul_rn(s[i], g[i]);
            if (p.normed_out) static_cast<T *>(p.normed_out)[row * p.ld_normed + e] = from_float<T>(__fmul_rn(u, r));
            if (p.smooth) u = __fmul_rn(u, m[i]);
            if (p.q) p.q[row * p.ld_q + e] = (int8_t)quant.one(u);
        }
    }
}

// V values of a vector over the channels from `at` on, as pairs.
template <typename G, int V, bool WHOLE>
__device__ __forceinline__ void load_channels(const void *vec, int at, int h, f32x2 *f)
{
    const G *g = static_cast<const G *>(vec);
    if constexpr (!WHOLE) load_anywhere<G, V, true>(g, at, h, f);
    else if constexpr (sizeof(G) == 4) load_fp32<V, true>(g + at, f);
    else unpack<G>(load16<true>(reinterpret_cast<const uint4 *>(g + at)), f);
}

template <typename T, int V, bool WHOLE>
__device__ __forceinline__ void load_gammas(const void *vec, bool gamma32, int at, int h, f32x2 *f)
{
    if (gamma32) load_channels<float, V, WHOLE>(vec, at, h, f);
    else load_channels<T, V, WHOLE>(vec, at, h, f);
}

// One CTA per row; a thread holds NCH packs of V elements (16 bytes of T), blockDim.x apart, in fp32 from the first look at x to the last
// store.  WHOLE: rows start on packs.  Else every row starts `lead` elements into one, the same in all tensors, and only what lies in a row's
// first and last pack is masked and stored one element at a time.  Its time is a row's chain of load, sum, load, sum and store (16 x 2048 2.7 us,
// 128 x 7168 4.9); the second loads stand behind the first sum, although none of them needs it.
template <typename T, typename X, int NCH, bool WHOLE, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) sandwich_kernel(const SandwichParams p)
{
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float2 red[2][32];
    dependent_wait();
    dependent_release();
    clear_status(p);
    const int threads = blockDim.x;
    const bool rows_gate = p.gate && p.ld_gate != 0 && p.gate_step != 0;
    const long long row = blockIdx.x;
    const int lead = WHOLE ? 0 : (int)((row * p.ld_x) & (V - 1)), end = lead + p.h, packs = (end + V - 1) / V;
    // Elements from the row's first pack on that there are to read: a row's edge packs hold elements of its neighbours, which are read with it
    // and dropped, but behind the last row's end there may be nothing.
    const long long apart = min(min(p.ld_x, p.ld_residual), rows_gate ? p.ld_gate : p.ld_x);
    const int room = end + (int)min((p.rows - 1 - row) * apart, 1024ll);
    const X *x = static_cast<const X *>(p.x) + row * p.ld_x - lead;
    const T *residual = static_cast<const T *>(p.residual) + row * p.ld_residual - lead, *gate = static_cast<const T *>(p.gate) + row * p.ld_gate - lead;
    const auto full = [&](int c) { return WHOLE || (c * V >= lead && (c + 1) * V <= end); };
    const auto inside = [&](int e) { return e >= lead && e < end; };
    const auto load = [&](auto type, const auto *from, int c, f32x2 *f) {   // a pack of a row
        typedef decltype(type) S;
        constexpr int N = (int)sizeof(S) * V / 16;
        if (!WHOLE && (c + 1) * V > room) {
            const auto one = [&](int e) { return inside(e) ? to_float<S>(from[e]) : 0.0f; };
#pragma unroll
            for (int e = 0; e < V; e += 2) f[e / 2] = pair2(one(c * V + e), one(c * V + e + 1));
            return;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) unpack<S>(*(reinterpret_cast<const uint4 *>(from + (long long)c * V) + j), f + j * (V / 2 / N));
    };
    const auto mask = [&](int c, f32x2 *f) {
        if (full(c)) return;
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const float2 v = unpair2(f[e / 2]);
            f[e / 2] = pair2(inside(c * V + e) ? v.x : 0.0f, inside(c * V + e + 1) ? v.y : 0.0f);
        }
    };
    const auto gammas = [&](const void *g, int c, f32x2 *f) { load_gammas<T, V, WHOLE>(g, p.gamma32, c * V - lead, p.h, f); };
    const auto store = [&](T *to, int c, const f32x2 *f) {
        if (full(c)) {
            *reinterpret_cast<uint4 *>(to + (long long)c * V) = pack<T>(f);
            return;
        }
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (inside(c * V + e)) to[c * V + e] = from_float<T>(element(f, e));
    };

    // the block's output, and the norm behind it
    f32x2 u[NCH][V / 2];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = threadIdx.x + i * threads;
        if (c >= packs) break;
        load(X(), x, c, u[i]);
        mask(c, u[i]);
    }
    float factor = p.block_scale;
    if (p.post_gamma) {
        f32x2 sum2 = 0;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            if (threadIdx.x + i * threads >= packs) break;
#pragma unroll
            for (int e = 0; e < V / 2; ++e) sum2 = fma2(u[i][e], u[i][e], sum2);
        }
        const float2 parts = unpair2(sum2);
        float sum = parts.x + parts.y, unused = 0.0f;
        block_reduce(sum, unused, red[0]);
        factor = __fmul_rn(factor, rsqrtf(__fmaf_rn(sum, p.inv_h, p.post_eps)));
    }
    if (p.gate && p.gate_step == 0) factor = __fmul_rn(factor, gate_value(to_float<T>(static_cast<const T *>(p.gate)[row * p.ld_gate]), p.gate_act));

    // the residual stream, and the sums of the next norm
    f32x2 sum2 = 0;
    float mag = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = threadIdx.x + i * threads;
        if (c >= packs) break;
        f32x2 f[V / 2];
#pragma unroll
        for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], pair2(factor, factor));
        if (p.post_gamma) {
            gammas(p.post_gamma, c, f);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], f[e]);
        }
        if (p.gate && p.gate_step != 0) {
            if (rows_gate) load(T(), gate, c, f);
            else load_channels<T, V, WHOLE>(p.gate, c * V - lead, p.h, f);
            if (p.gate_act != kGateNone) {
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 g = unpair2(f[e]);
                    f[e] = pair2(gate_value(g.x, p.gate_act), gate_value(g.y, p.gate_act));
                }
            }
#pragma unroll
            for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], f[e]);
        }
        load(T(), residual, c, f);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) u[i][e] = fma2(f[e], pair2(p.residual_scale, p.residual_scale), u[i][e]);
        mask(c, u[i]);
        if (p.residual_out) store(static_cast<T *>(p.residual_out) + row * p.ld_residual_out - lead, c, u[i]);
        if (!p.gamma) continue;
#pragma unroll
        for (int e = 0; e < V / 2; ++e) sum2 = fma2(u[i][e], u[i][e], sum2);
        gammas(p.gamma, c, f);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], f[e]);
        if (!p.q) continue;
#pragma unroll
        for (int e = 0; e < V / 2; ++e) f[e] = u[i][e];
        if (p.smooth) {
            f32x2 m[V / 2];
            load_channels<float, V, WHOLE>(p.smooth, c * V - lead, p.h, m);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) f[e] = mul2(f[e], m[e]);
        }
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            const float2 v = unpair2(f[e]);
            mag = max_mag(mag, v.x, v.y);
        }
    }
    if (p.gamma) {
        const float2 parts = unpair2(sum2);
        float sum = parts.x + parts.y;
        block_reduce(sum, mag, red[1]);
        const float r = rsqrtf(__fmaf_rn(sum, p.inv_h, p.eps)), step = step_of(mag);
        Quantiser quant;
        quant.set(step);
        if (p.q && threadIdx.x == 0) p.scale[row] = step == 0.0f ? 0.0f : __fmul_rn(step, r);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = threadIdx.x + i * threads;
            if (c >= packs) break;
            if (p.normed_out) {
                f32x2 y[V / 2];
#pragma unroll
                for (int e = 0; e < V / 2; ++e) y[e] = mul2(u[i][e], pair2(r, r));
                store(static_cast<T *>(p.normed_out) + row * p.ld_normed - lead, c, y);
            }
            if (!p.q) continue;
            if (p.smooth) {
                f32x2 m[V / 2];
                load_channels<float, V, WHOLE>(p.smooth, c * V - lead, p.h, m);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], m[e]);
            }
            uint32_t q[V / 4];
#pragma unroll
            for (int e = 0; e < V / 4; ++e) q[e] = quant.four(u[i] + 2 * e, quant.rcp != 0.0f);
            int8_t *to = p.q + row * p.ld_q - lead + (long long)c * V;
            if (full(c)) {
                if (V == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(q[0], q[V / 4 - 1]);
                else *reinterpret_cast<uint32_t *>(to) = q[0];
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (inside(c * V + e)) to[e] = (int8_t)(q[e / 4] >> (e % 4 * 8));
            }
        }
    }
}


// Many rows: one CTA per SM, in which groups of threads take a row each.  What multiplies the channels is laid out once in shared memory, in
// fp32 and with everything folded in that a row does not change (the norm's weight, the activated gate, the block's scale), so that a row's
// turn has no loads but its own.  Those come as one bulk copy a tensor, for the next row as soon as the group holds this one in registers.
// (With a 16-byte cp.async for each pack an SM takes in 16 bytes per ns however many are under way: 4096 x 7168 in 80 us.)  A group's
// threads hold two packs each; four would leave too few rows in turn for the chain load, sum, load, sum, store of each.
// 4096 x 7168, fp32 x, bf16 stream: 53.4 us with int8 rows (264 MB, 4.9 TB/s), 48.1 with bf16 rows and a gate (294 MB, 6.1 TB/s).  Quantising
// costs what the difference is: max, step and rounding are the issue slots' work.  5001 channels, whose rows begin anywhere, take 52.6 and 5008
// take 42.9: eight single reads of a factor for two wide ones, and rows' ends element by element.  600 x 16384 24.3.
constexpr int kGroupPacks = 2, kMaxGroups = 14, kMaxDepth = 3;    // of the 15 named barriers that are left
constexpr long long kWaitLimitCycles = 1ll << 31, kDrainLimitCycles = 1ll << 22;   // about a second, two milliseconds
constexpr int kGroupThreads = 1024;
// Packs that a row can touch, and floats of a vector of factors.
template <int V, bool WHOLE> __host__ __device__ inline int most_packs(int h) { return WHOLE ? h / V : (h + 2 * V - 2) / V; }
template <int V, bool WHOLE> __host__ __device__ inline int factor_floats(int h) { return WHOLE ? h : V * (most_packs<V, WHOLE>(h) + 2); }

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool mbar_try(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok;
}
// What a wait that has run out leaves behind.
__device__ __noinline__ void gave_up(volatile int *late, int *status, int role, uint32_t parity)
{
    *late = 1;
    if (atomicCAS(status, kStatusOk, kStatusWaitTimeout) == kStatusOk) {
        status[1] = (int)blockIdx.x;
        status[2] = role;
        status[3] = (int)parity;
    }
}
// Bounded: false when the copies have not come, which the status says, or when another wait of the CTA has run out.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, volatile int *late, const SandwichParams &p, int role)
{
    if (mbar_try(bar, parity)) return true;
    for (const long long t0 = clock64(); !*late;) {
        if (mbar_try(bar, parity)) return true;
        if (clock64() - t0 > p.wait_limit) gave_up(late, p.status, role, parity);
    }
    return false;
}
__device__ __forceinline__ void bulk_copy(void *to, const void *from, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)), "l"(from), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void group_sync(int group, int threads)
{
    if (threads > 32) asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
    else __syncwarp();
}

__device__ __forceinline__ void group_reduce(float &sum, float &mag, float2 *red, int group, int threads)
{
    uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(mag) & 0x7fffffffu);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threads > 32) {
        const int lane = threadIdx.x & 31, warps = threads >> 5, warp = (int)(threadIdx.x >> 5) - group * warps;
        red += group * warps;
        if (lane == 0) red[warp] = make_float2(sum, __uint_as_float(m));
        group_sync(group, threads);
        const float2 v = lane < warps ? red[lane] : make_float2(0.0f, 0.0f);
        sum = v.x;
        m = __reduce_max_sync(0xffffffffu, __float_as_uint(v.y));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    mag = __uint_as_float(m);
}

// WHOLE as above; EXACT: every thread of a group has all of its packs; GATED: a gate for each element.
template <typename T, typename X, bool WHOLE, bool EXACT, bool GATED>
__global__ void __launch_bounds__(kGroupThreads, 1) sandwich_rows_kernel(const SandwichParams p, int threads, int groups, int depth)
{
    constexpr int V = 16 / (int)sizeof(T), XW = (int)sizeof(X) * V / 16, N = kGroupPacks;
    extern __shared__ uint4 smem[];     // the groups' rows (x, residual, gate); block's, next norm's and smoothing's factors
    __shared__ float2 red[4][32];
    __shared__ alignas(8) uint64_t x_landed[kMaxGroups][kMaxDepth], rest_landed[kMaxGroups][kMaxDepth];
    __shared__ volatile int late;   // a wait has run out: from then on nothing is fetched, and what has not come is NaN
    const float nan = __int_as_float(0x7fffffff);
    if (threadIdx.x == 0) late = 0;
    const bool channel_gate = !GATED && p.gate && p.gate_step != 0;
    const int most = most_packs<V, WHOLE>(p.h), row_packs = most * (XW + (GATED ? 2 : 1)), plane = most + 2, vec = factor_floats<V, WHOLE>(p.h);
    float *by_block = reinterpret_cast<float *>(smem + (size_t)groups * depth * row_packs), *by_gamma = by_block + vec, *by_smooth = by_gamma + (p.gamma ? vec : 0);
    const int group = (int)threadIdx.x / threads, tid = (int)threadIdx.x - group * threads;
    uint4 *all = smem + (size_t)group * depth * row_packs;
    const auto lead_of = [&](long long row) { return WHOLE ? 0 : (int)((row * p.ld_x) & (V - 1)); };
    // A row from the pack on in which it begins, to the 16 bytes in which it ends (which lie in the row's own memory pages, whatever else is
    // in them).  By one thread, when all of the group have read what is there.
    const auto fetch = [&](const auto *from, long long row, long long ld, uint4 *to, uint64_t *bar) {
        const int lead = lead_of(row);
        bulk_copy(to, from + row * ld - lead, ((lead + p.h) * (uint32_t)sizeof(*from) + 15) / 16 * 16, bar);
    };
    const auto expect = [&](uint64_t *bar, long long row, int bytes, int n) {   // n rows of elements of so many bytes
        const uint32_t all = ((lead_of(row) + p.h) * (uint32_t)bytes + 15) / 16 * 16 * n;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(all) : "memory");
    };
    const auto fetch_x = [&](long long row, int at) {
        expect(&x_landed[group][at], row, sizeof(X), 1);
        fetch(static_cast<const X *>(p.x), row, p.ld_x, all + at * row_packs, &x_landed[group][at]);
    };
    const auto fetch_rest = [&](long long row, int at) {
        uint4 *to = all + at * row_packs + most * XW;
        expect(&rest_landed[group][at], row, sizeof(T), GATED ? 2 : 1);
        fetch(static_cast<const T *>(p.residual), row, p.ld_residual, to, &rest_landed[group][at]);
        if (GATED) fetch(static_cast<const T *>(p.gate), row, p.ld_gate, to + most, &rest_landed[group][at]);
    };
    const long long step = (long long)gridDim.x * groups;
    long long row = (long long)blockIdx.x * groups + group;
    if (tid == 0) {
        for (int d = 0; d < depth; ++d) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&x_landed[group][d])) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&rest_landed[group][d])) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    dependent_wait();
    dependent_release();
    if (tid == 0) {
        for (int d = 0; d < depth && row + d * step < p.fetched; ++d) {
            fetch_x(row + d * step, d);
            fetch_rest(row + d * step, d);
        }
    }
    // The factors, so that a warp reads no bank twice.  WHOLE: four floats of every pack together.  Else, since a pack begins at any channel,
    // every V-th channel together, a zero before and behind, for the packs that reach beyond a row's ends.
    const auto place = [&](float *to, int c, const f32x2 *f) {
        if constexpr (WHOLE) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float2 u = unpair2(f[e / 2]), v = unpair2(f[e / 2 + 1]);
                reinterpret_cast<float4 *>(to)[e / 4 * most + c] = make_float4(u.x, u.y, v.x, v.y);
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) to[e * plane + c + 1] = element(f, e);
        }
    };
    for (int c = (int)threadIdx.x - (WHOLE ? 0 : 1); c < (WHOLE ? most : plane - 1); c += blockDim.x) {
        f32x2 post[V / 2], g[V / 2], gamma[V / 2], smooth[V / 2];
#pragma unroll
        for (int e = 0; e < V / 2; ++e) post[e] = g[e] = pair2(1.0f, 1.0f);
        if (p.post_gamma) load_gammas<T, V, WHOLE>(p.post_gamma, p.gamma32, c * V, p.h, post);
        if (channel_gate) load_channels<T, V, WHOLE>(p.gate, c * V, p.h, g);
        if (p.gamma) load_gammas<T, V, WHOLE>(p.gamma, p.gamma32, c * V, p.h, gamma);
        if (p.smooth) load_channels<float, V, WHOLE>(p.smooth, c * V, p.h, smooth);
        if (p.gamma) place(by_gamma, c, gamma);
        if (p.smooth) place(by_smooth, c, smooth);
        if (channel_gate && p.gate_act != kGateNone) {
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                const float2 v = unpair2(g[e]);
                g[e] = pair2(gate_value(v.x, p.gate_act), gate_value(v.y, p.gate_act));
            }
        }
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            post[e] = mul2(mul2(post[e], pair2(p.block_scale, p.block_scale)), g[e]);
            const float2 v = unpair2(post[e]);
            if (!WHOLE) post[e] = pair2((unsigned)(c * V + 2 * e) < (unsigned)p.h ? v.x : 0.0f, (unsigned)(c * V + 2 * e + 1) < (unsigned)p.h ? v.y : 0.0f);
        }
        place(by_block, c, post);
    }
    clear_status(p);
    __syncthreads();
    uint32_t phase = 0;
    int at = 0;     // the buffer that the row is in
    bool gone = false;      // for good: behind a row that was not fetched a barrier's parity says nothing
    for (int parity = 0; row < p.rows; row += step, parity ^= 1) {
        const long long next = row + depth * step;   // what comes in its place
        const uint4 *mine = all + at * row_packs;
        const int lead = lead_of(row), packs = WHOLE ? most : (lead + p.h + V - 1) / V;
        const auto has = [&](int i) { return EXACT || tid + i * threads < packs; };
        const auto full = [&](int c) { return WHOLE || (c * V >= lead && (c + 1) * V <= lead + p.h); };
        const auto inside = [&](int e) { return e >= lead && e < lead + p.h; };
        const auto mask = [&](int c, f32x2 *f) {
            if (full(c)) return;
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float2 v = unpair2(f[e / 2]);
                f[e / 2] = pair2(inside(c * V + e) ? v.x : 0.0f, inside(c * V + e + 1) ? v.y : 0.0f);
            }
        };
        const auto factors = [&](const float *from, int c, f32x2 *f) {
            if constexpr (WHOLE) {
#pragma unroll
                for (int e = 0; e < V; e += 4) unpack<float>(reinterpret_cast<const uint4 *>(from)[e / 4 * most + c], f + e / 2);
            } else {
                const auto one = [&](int j) { return from[((j - lead) & (V - 1)) * plane + c + 1 - (j < lead)]; };
#pragma unroll
                for (int e = 0; e < V; e += 2) f[e / 2] = pair2(one(e), one(e + 1));
            }
        };
        const auto store = [&](T *to, int c, const f32x2 *f) {
            if (full(c)) {
                *reinterpret_cast<uint4 *>(to + c * V) = pack<T>(f);
                return;
            }
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (inside(c * V + e)) to[c * V + e] = from_float<T>(element(f, e));
        };

        // the block's output, and the norm behind it
        f32x2 u[N][V / 2];
        gone = gone || !mbar_wait(&x_landed[group][at], phase, &late, p, 1000);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * threads;
#pragma unroll
            for (int j = 0; j < XW; ++j) unpack<X>(has(i) ? mine[c * XW + j] : make_uint4(0, 0, 0, 0), u[i] + j * (V / 2 / XW));
            if (has(i)) mask(c, u[i]);
        }
        float factor = 1.0f;
        if (p.post_gamma) {
            f32x2 sum2 = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < V / 2; ++e) sum2 = fma2(u[i][e], u[i][e], sum2);
            const float2 parts = unpair2(sum2);
            float sum = gone ? nan : parts.x + parts.y, unused = 0.0f;
            group_reduce(sum, unused, red[parity], group, threads);
            factor = __fmul_rn(factor, rsqrtf(__fmaf_rn(sum, p.inv_h, p.post_eps)));
        } else {
            group_sync(group, threads);
        }
        if (tid == 0 && next < p.fetched && !late) fetch_x(next, at);
        if (p.gate && p.gate_step == 0) factor = __fmul_rn(factor, gate_value(to_float<T>(static_cast<const T *>(p.gate)[row * p.ld_gate]), p.gate_act));

        // the residual stream, and the sums of the next norm
        gone = gone || !mbar_wait(&rest_landed[group][at], phase, &late, p, 1001);
        if (gone) factor = nan;     // and so all that follows
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!has(i)) break;
            const int c = tid + i * threads;
            f32x2 f[V / 2], r[V / 2];
            factors(by_block, c, f);
            unpack<T>(mine[most * XW + c], r);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], mul2(f[e], pair2(factor, factor)));
            if (GATED) {
                unpack<T>(mine[most * (XW + 1) + c], f);
                if (p.gate_act != kGateNone) {
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) {
                        const float2 g = unpair2(f[e]);
                        f[e] = pair2(gate_value(g.x, p.gate_act), gate_value(g.y, p.gate_act));
                    }
                }
#pragma unroll
                for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], f[e]);
            }
#pragma unroll
            for (int e = 0; e < V / 2; ++e) u[i][e] = fma2(r[e], pair2(p.residual_scale, p.residual_scale), u[i][e]);
            mask(c, u[i]);
        }
        if (p.residual_out) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (has(i)) store(static_cast<T *>(p.residual_out) + row * p.ld_residual_out - lead, tid + i * threads, u[i]);
        }
        f32x2 sum2 = 0;
        float mag = 0.0f;
        if (p.gamma) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!has(i)) break;
                f32x2 f[V / 2];
                factors(by_gamma, tid + i * threads, f);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    sum2 = fma2(u[i][e], u[i][e], sum2);
                    u[i][e] = mul2(u[i][e], f[e]);
                }
            }
        }
        if (p.q) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!has(i)) break;
                f32x2 f[V / 2];
                if (p.smooth) factors(by_smooth, tid + i * threads, f);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 v = unpair2(p.smooth ? mul2(u[i][e], f[e]) : u[i][e]);
                    mag = max_mag(mag, v.x, v.y);
                }
            }
        }
        const float2 parts = unpair2(sum2);
        float sum = parts.x + parts.y;
        if (p.gamma) group_reduce(sum, mag, red[2 + parity], group, threads);
        else group_sync(group, threads);
        if (tid == 0 && next < p.fetched && !late) fetch_rest(next, at);
        if (++at == depth) { at = 0; phase ^= 1; }
        if (!p.gamma) continue;
        const float r = rsqrtf(__fmaf_rn(sum, p.inv_h, p.eps));
        if (p.normed_out) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!has(i)) break;
                f32x2 y[V / 2];
#pragma unroll
                for (int e = 0; e < V / 2; ++e) y[e] = mul2(u[i][e], pair2(r, r));
                store(static_cast<T *>(p.normed_out) + row * p.ld_normed - lead, tid + i * threads, y);
            }
        }
        if (!p.q) continue;
        const float of_row = step_of(mag);
        Quantiser quant;
        quant.set(of_row);
        if (tid == 0) p.scale[row] = of_row == 0.0f ? 0.0f : __fmul_rn(of_row, r);
        const auto finish = [&](bool by_rcp) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = tid + i * threads;
                if (!has(i)) break;
                if (p.smooth) {
                    f32x2 f[V / 2];
                    factors(by_smooth, c, f);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], f[e]);
                }
                uint32_t q[V / 4];
#pragma unroll
                for (int e = 0; e < V / 4; ++e) q[e] = quant.four(u[i] + 2 * e, by_rcp);
                int8_t *to = p.q + row * p.ld_q - lead + c * V;
                if (full(c)) {
                    if (V == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(q[0], q[V / 4 - 1]);
                    else *reinterpret_cast<uint32_t *>(to) = q[0];
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (inside(c * V + e)) to[e] = (int8_t)(q[e / 4] >> (e % 4 * 8));
                }
            }
        };
        if (quant.rcp != 0.0f) finish(true);
        else finish(false);
    }
    // Copies that were not waited for must not land in shared memory that is no longer this CTA's.  One of a barrier's two parities is the past
    // phase's, and no wait; the other one comes with the copies, or not at all where none are under way.
    if (tid == 0 && late) {
        for (int i = 0; i < 4 * depth; ++i) {
            uint64_t *bar = (i & 2 ? rest_landed : x_landed)[group] + i / 4;
            for (const long long t0 = clock64(); !mbar_try(bar, i & 1) && clock64() - t0 < kDrainLimitCycles;) {}
        }
    }
}

// Threads of a group and groups of a CTA; 0 where a row does not fit.
struct Groups {
    int threads, groups, depth, smem;
};
template <typename T, typename X, bool WHOLE>
Groups groups_of(const SandwichParams &p)
{
    constexpr int V = 16 / (int)sizeof(T), XW = (int)sizeof(X) * V / 16;
    const int packs = most_packs<V, WHOLE>(p.h), room = 224 * 1024;
    Groups g;
    g.threads = ((packs + kGroupPacks - 1) / kGroupPacks + 31) / 32 * 32;
    const int factors = 4 * factor_floats<V, WHOLE>(p.h) * (1 + (p.gamma != nullptr) + (p.smooth != nullptr));
    const int row = (XW + (p.gate && p.ld_gate && p.gate_step ? 2 : 1)) * 16 * packs;
    g.groups = kGroupThreads / g.threads;
    if (g.groups > kMaxGroups) g.groups = kMaxGroups;
    if (g.groups > (room - factors) / row) g.groups = room > factors ? (room - factors) / row : 0;
    g.depth = g.groups > 0 ? (room - factors) / (g.groups * row) : 0;   // rows of a group that there is room for
    if (g.depth > kMaxDepth) g.depth = kMaxDepth;
    g.smem = factors + g.groups * g.depth * row;
    return g;
}

template <typename T, typename X, bool WHOLE, bool EXACT, bool GATED>
cudaError_t launch_rows(const SandwichParams &p, const Groups &g, cudaStream_t stream)
{
    const auto kernel = sandwich_rows_kernel<T, X, WHOLE, EXACT, GATED>;
    static unsigned long long done_mask = 0;   // once per device; the attribute is idempotent, so a race only repeats the call
    int dev = 0;
    cudaGetDevice(&dev);
    if (!((done_mask >> (dev & 63)) & 1ull)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
        if (e != cudaSuccess) return e;
        done_mask |= 1ull << (dev & 63);
    }
    const int ctas = (p.rows + g.groups - 1) / g.groups;
    return launch_dependent(kernel, dim3(ctas < 148 ? ctas : 148), g.threads * g.groups, g.smem, 1, stream, p, g.threads, g.groups, g.depth);
}

template <typename T, typename X>
cudaError_t launch_any(const SandwichParams &p, cudaStream_t stream)
{
    // Few rows: up to 1024 threads with eight elements or more each.  Many: small CTAs, of which an SM holds more (128 rows of 7168 on no pack
    // 9.8 us against 17.5 with those, 16 of 40000 33 and 107, 300 of 40000 142 and 183, but 4096 of 7168 173 and 130).
    const int wanted = (p.h + 7) / 8, most = p.rows <= 148 ? 1024 : 256, threads = wanted > most ? most : (wanted + 31) / 32 * 32;
    if (p.rows <= 4 * 148) return launch_dependent(sandwich_any_few_kernel<T, X>, dim3(p.rows), threads, 0, 1, stream, p);
    return launch_dependent(sandwich_any_kernel<T, X>, dim3(p.rows), 256, 0, 1, stream, p);
}

template <typename T, typename X, bool WHOLE>
cudaError_t launch_packed(const SandwichParams &p, cudaStream_t stream)
{
    constexpr int V = 16 / (int)sizeof(T);
    const int packs = most_packs<V, WHOLE>(p.h);
    const auto warps = [](int n) { return (n + 31) / 32 * 32; };
    // Few rows: as many threads as a row has packs, for the shortest chain.  The kernel of many rows has the factors to lay out first and
    // gains where every SM has rows enough in turn, later for short rows, of which an SM holds more CTAs (this one / that one, us, bf16 and
    // an fp32 x: 148 x 7168 6.0 / 8.1, 200 x 7168 9.6 / 8.2, 1184 x 4096 14.8 / 15.6, 2368 x 4096 25.8 / 22.8, 4096 x 2048 19.6 / 22.5,
    // 16384 x 2048 64.5 / 57.6, 16384 x 1424 49.8 / 47.3, 16384 x 768 26.8 / 32.0).
    const long long work = (long long)p.rows * packs;
    if (packs <= 256 && (packs <= 128 || work <= 148 * 8192))
        return launch_dependent(sandwich_kernel<T, X, 1, WHOLE, 256, 8>, dim3(p.rows), warps(packs), 0, 1, stream, p);
    if (packs <= 1024 && (p.rows <= 148 || (packs <= 512 && work <= 148 * 4096)))
        return launch_dependent(sandwich_kernel<T, X, 1, WHOLE, 1024, 1>, dim3(p.rows), warps(packs), 0, 1, stream, p);
    const Groups g = groups_of<T, X, WHOLE>(p);
    if (g.groups > 0) {
        const bool gated = p.gate && p.ld_gate && p.gate_step;
        if (WHOLE && packs == kGroupPacks * g.threads) return gated ? launch_rows<T, X, WHOLE, WHOLE, true>(p, g, stream) : launch_rows<T, X, WHOLE, WHOLE, false>(p, g, stream);
        return gated ? launch_rows<T, X, WHOLE, false, true>(p, g, stream) : launch_rows<T, X, WHOLE, false, false>(p, g, stream);
    }
    if (packs <= 4 * 1024) return launch_dependent(sandwich_kernel<T, X, 4, WHOLE, 1024, 1>, dim3(p.rows), warps((packs + 3) / 4), 0, 1, stream, p);
    return launch_any<T, X>(p, stream);
}

template <typename T, typename X>
cudaError_t launch_typed(const SandwichParams &p, cudaStream_t stream)
{
    constexpr int V = 16 / (int)sizeof(T);
    // Packs need every tensor to begin on one (V elements of its own type, at most 16 bytes) and its rows to be as far apart as x's, modulo
    // a pack.
    const auto fits = [&](const void *base, long long ld, int bytes) {
        return !base || (((uintptr_t)base & (uintptr_t)(V * bytes < 16 ? V * bytes - 1 : 15)) == 0 && (ld - p.ld_x) % V == 0);
    };
    const bool rows_gate = p.gate && p.gate_step && p.ld_gate, channel_gate = p.gate && p.gate_step && !p.ld_gate;
    const bool packed = fits(p.x, p.ld_x, sizeof(X)) && fits(p.residual, p.ld_residual, sizeof(T)) && fits(p.residual_out, p.ld_residual_out, sizeof(T)) &&
                        fits(p.normed_out, p.ld_normed, sizeof(T)) && fits(p.q, p.ld_q, 1) && fits(p.gamma, p.ld_x, p.gamma32 ? 4 : sizeof(T)) &&
                        fits(p.post_gamma, p.ld_x, p.gamma32 ? 4 : sizeof(T)) && fits(p.smooth, p.ld_x, 4) &&
                        (!rows_gate || fits(p.gate, p.ld_gate, sizeof(T))) && (!channel_gate || fits(p.gate, p.ld_x, sizeof(T)));
    if (packed) return p.h % V == 0 && p.ld_x % V == 0 ? launch_packed<T, X, true>(p, stream) : launch_packed<T, X, false>(p, stream);
    return launch_any<T, X>(p, stream);
}

}  // namespace

cudaError_t sandwich_norm_launch(const SandwichNormProblem &n, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (n.rows <= 0) return cudaSuccess;
    if (!workspace || workspace_bytes < kSandwichNormWorkspace) return cudaErrorInvalidValue;
    SandwichParams p;
    p.x = n.x; p.residual = n.residual; p.gamma = n.gamma; p.post_gamma = n.post_gamma; p.gate = n.gate; p.smooth = n.smooth;
    p.q = n.q; p.scale = n.scale; p.residual_out = n.residual_out; p.normed_out = n.normed_out;
    p.ld_x = n.ld_x; p.ld_residual = n.ld_residual; p.ld_gate = n.ld_gate; p.ld_q = n.ld_q; p.ld_residual_out = n.ld_residual_out;
    p.ld_normed = n.ld_normed;
    p.rows = (int)n.rows; p.h = (int)n.h; p.gate_step = n.gate_step; p.gate_act = n.gate_act;
    p.gamma32 = n.gamma_dtype == kF32;
    p.inv_h = 1.0f / (float)n.h; p.residual_scale = n.residual_scale; p.block_scale = n.block_scale; p.eps = n.eps; p.post_eps = n.post_eps;
    p.status = static_cast<int *>(workspace);
    p.wait_limit = n.opt.wait_limit_cycles > 0 ? n.opt.wait_limit_cycles : kWaitLimitCycles;
    p.fetched = p.rows > n.opt.test_skip_k_blocks ? p.rows - n.opt.test_skip_k_blocks : 0;
    // A caller's limit may be short: nothing but the stream orders another block's record behind the clearing then.
    p.clear_status = n.opt.wait_limit_cycles <= 0;
    if (!p.clear_status) {
        const cudaError_t e = cudaMemsetAsync(workspace, 0, 16, stream);
        if (e != cudaSuccess) return e;
    }
    switch (n.dtype) {
        case kF32: return launch_typed<float, float>(p, stream);
        case kF16: return n.x_dtype == kF32 ? launch_typed<__half, float>(p, stream) : launch_typed<__half, __half>(p, stream);
        case kBF16: return n.x_dtype == kF32 ? launch_typed<__nv_bfloat16, float>(p, stream) : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace gmm
