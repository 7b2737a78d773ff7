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

// V values of a vector over the channels from `at` on, as pairs.
template <typename G, int V, bool WHOLE>
__device__ __forceinline__ void load_channels(const void *vec, int at, int h, f32x2 *f)
{
    const G *g = static_cast<const G *>(vec);
    if constexpr (!WHOLE) load_anywhere<G, V>(g, at, h, f);
    else if constexpr (sizeof(G) == 4) load_fp32<V>(g + at, f);
    else unpack<G>(__ldg(reinterpret_cast<const uint4 *>(g + at)), f);
}

// One CTA per row; a thread holds NCH packs of V elements (16 bytes of T), blockDim.x apart, in fp32 from the first look at x to the last
// store.  WHOLE: rows start on packs.  Else every row starts `lead` elements into one, the same in all tensors, and only what lies in a row's
// first and last pack is masked and stored one element at a time.
//
// STREAM: the CTA takes every gridDim.x-th row.  While it works on one, the packs of the next are copied to shared memory, each by the
// thread that will read it, x as soon as it is in registers and the rest behind the first reduction.
template <typename T, typename X, int NCH, bool WHOLE, int MAXT, int MINB, bool STREAM>
__global__ void __launch_bounds__(MAXT, MINB) sandwich_kernel(const SandwichParams p)
{
    constexpr int V = 16 / (int)sizeof(T), XW = (int)sizeof(X) * V / 16;   // loads of a pack of x
    extern __shared__ uint4 ahead[];    // STREAM: [(XW + 1 or 2) * NCH][threads]: x, residual, gate
    __shared__ float2 red[4][32];
    const int threads = blockDim.x;
    const uint32_t mine = STREAM ? (uint32_t)__cvta_generic_to_shared(ahead) + threadIdx.x * 16 : 0;
    const bool rows_gate = p.gate && p.ld_gate != 0 && p.gate_step != 0;
    const auto lead_of = [&](long long row) { return WHOLE ? 0 : (int)((row * p.ld_x) & (V - 1)); };
    // Elements from the row's first pack on that there are to read (see add_rms_norm_quant): a row's edge packs hold elements of its
    // neighbours, which are read with it and dropped, but behind the last row's end there may be nothing.
    const auto room_of = [&](long long row, int lead) {
        long long ld = min(p.ld_x, p.ld_residual);
        if (rows_gate) ld = min(ld, p.ld_gate);
        return lead + p.h + (int)min((p.rows - 1 - row) * ld, 1024ll);
    };
    const auto slot = [&](int s) { return mine + (uint32_t)(s * threads) * 16; };
    const auto copy = [&](int s, const void *from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot(s)), "l"(from) : "memory"); };
    const auto there = [&](int c, int lead, int room) { return WHOLE ? c * V < p.h : c * V < lead + p.h && (c + 1) * V <= room; };
    const auto fetch_x = [&](long long row) {
        const int lead = lead_of(row), room = room_of(row, lead);
        const X *x = static_cast<const X *>(p.x) + row * p.ld_x - lead;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = threadIdx.x + i * threads;
            if (!there(c, lead, room)) continue;
#pragma unroll
            for (int j = 0; j < XW; ++j) copy(i * XW + j, reinterpret_cast<const uint4 *>(x + (long long)c * V) + j);
        }
    };
    const auto fetch_rest = [&](long long row, int i) {
        const int lead = lead_of(row), room = room_of(row, lead), c = threadIdx.x + i * threads;
        if (!there(c, lead, room)) return;
        copy(NCH * XW + i, static_cast<const T *>(p.residual) + row * p.ld_residual - lead + (long long)c * V);
        if (rows_gate) copy(NCH * (XW + 1) + i, static_cast<const T *>(p.gate) + row * p.ld_gate - lead + (long long)c * V);
    };
    const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    const auto await_older = [] { asm volatile("cp.async.wait_group 1;" ::: "memory"); };
    if (STREAM) {
        fetch_x(blockIdx.x);
        commit();
#pragma unroll
        for (int i = 0; i < NCH; ++i) fetch_rest(blockIdx.x, i);
        commit();
    }
    int parity = 0;
    for (long long row = blockIdx.x; row < p.rows; row += STREAM ? (long long)gridDim.x : (long long)p.rows) {
        const long long next = row + gridDim.x;
        const int lead = lead_of(row), end = lead + p.h, room = room_of(row, lead), packs = (end + V - 1) / V;
        const X *x = static_cast<const X *>(p.x) + row * p.ld_x - lead;
        const T *residual = static_cast<const T *>(p.residual) + row * p.ld_residual - lead, *gate = static_cast<const T *>(p.gate) + row * p.ld_gate - lead;
        const auto full = [&](int c) { return WHOLE || (c * V >= lead && (c + 1) * V <= end); };
        const auto inside = [&](int e) { return e >= lead && e < end; };
        // a pack of a row of S: N loads of it, out of the slots from s on
        const auto load = [&](auto type, const auto *from, int c, int s, f32x2 *f) {
            typedef decltype(type) S;
            constexpr int N = (int)sizeof(S) * V / 16;
            if (!WHOLE && (c + 1) * V > room) {
                const auto one = [&](int e) { return inside(e) ? to_float<S>(from[e]) : 0.0f; };
#pragma unroll
                for (int e = 0; e < V; e += 2) f[e / 2] = pair2(one(c * V + e), one(c * V + e + 1));
                return;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                uint4 u;
                if (STREAM) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(slot(s + j)) : "memory");
                else u = *(reinterpret_cast<const uint4 *>(from + (long long)c * V) + j);
                unpack<S>(u, f + j * (V / 2 / N));
            }
        };
        const auto mask = [&](int c, f32x2 *f) {
            if (full(c)) return;
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float2 v = unpair2(f[e / 2]);
                f[e / 2] = pair2(inside(c * V + e) ? v.x : 0.0f, inside(c * V + e + 1) ? v.y : 0.0f);
            }
        };
        const auto gammas = [&](const void *g, int c, f32x2 *f) {
            if (p.gamma32) load_channels<float, V, WHOLE>(g, c * V - lead, p.h, f);
            else load_channels<T, V, WHOLE>(g, c * V - lead, p.h, f);
        };
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
        if (STREAM) await_older();
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = threadIdx.x + i * threads;
            if (c >= packs) break;
            load(X(), x, c, i * XW, u[i]);
            mask(c, u[i]);
        }
        if (STREAM) {
            if (next < p.rows) fetch_x(next);   // the thread has read what this fills
            commit();
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
            block_reduce(sum, unused, red[parity]);
            factor = __fmul_rn(factor, rsqrtf(__fmaf_rn(sum, p.inv_h, p.post_eps)));
        }
        if (p.gate && p.gate_step == 0) factor = __fmul_rn(factor, gate_value(to_float<T>(static_cast<const T *>(p.gate)[row * p.ld_gate]), p.gate_act));

        // the residual stream, and the sums of the next norm
        if (STREAM) await_older();
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
                if (rows_gate) load(T(), gate, c, NCH * (XW + 1) + i, f);
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
            load(T(), residual, c, NCH * XW + i, f);
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
        if (STREAM) {
#pragma unroll
            for (int i = 0; i < NCH; ++i)
                if (next < p.rows) fetch_rest(next, i);
            commit();
        }
        if (p.gamma) {
            const float2 parts = unpair2(sum2);
            float sum = parts.x + parts.y;
            block_reduce(sum, mag, red[2 + parity]);
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
        parity ^= 1;
    }
}

// Many rows that start on packs: one CTA per SM, in which groups of threads take a row each.  What multiplies the channels is laid out once
// in shared memory, in fp32 and with everything folded in that a row does not change (the norm's weight, the activated gate, the block's
// scale), so that a row's turn has no loads but its own.  Those come as one bulk copy a tensor, for the next row as soon as the group holds
// this one in registers.  (With a 16-byte cp.async for each pack, the form of the other kernels, an SM takes in 16 bytes per ns however many
// are under way: 4096 x 7168 in 80 us.)  A group's threads hold four packs each.
constexpr int kGroupPacks = 2, kMaxGroups = 14, kMaxDepth = 3;    // of the 15 named barriers that are left
constexpr long long kWaitLimitCycles = 1ll << 31;  // about a second
__host__ __device__ constexpr int group_threads_most(int elem) { return 1024; }

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// Bounded: false when the copies have not come.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity)
{
    uint32_t ok = 0;
    const long long t0 = clock64();
    while (true) {
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if (clock64() - t0 > kWaitLimitCycles) return false;
    }
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

// EXACT: every thread of a group has all of its packs.  GATED: a gate for each element.
template <typename T, typename X, bool EXACT, bool GATED>
__global__ void __launch_bounds__(group_threads_most(sizeof(T)), 1) sandwich_rows_kernel(const SandwichParams p, int threads, int groups, int depth)
{
    constexpr int V = 16 / (int)sizeof(T), XW = (int)sizeof(X) * V / 16, N = kGroupPacks;
    extern __shared__ uint4 smem[];     // the groups' rows (x, residual, gate); block's, next norm's and smoothing's factors [h]
    __shared__ float2 red[4][32];
    __shared__ alignas(8) uint64_t x_landed[kMaxGroups][kMaxDepth], rest_landed[kMaxGroups][kMaxDepth];
    const bool channel_gate = !GATED && p.gate && p.gate_step != 0;
    const int packs = p.h / V, row_packs = packs * (XW + (GATED ? 2 : 1));
    float *by_block = reinterpret_cast<float *>(smem + (size_t)groups * depth * row_packs), *by_gamma = by_block + p.h, *by_smooth = by_gamma + (p.gamma ? p.h : 0);
    const int group = (int)threadIdx.x / threads, tid = (int)threadIdx.x - group * threads;
    uint4 *all = smem + (size_t)group * depth * row_packs;
    const uint32_t bytes = (uint32_t)packs * 16;
    const auto expect = [](uint64_t *bar, uint32_t n) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory"); };
    // by one thread, when all of the group have read what is there
    const auto fetch_x = [&](long long row, int at) {
        expect(&x_landed[group][at], bytes * XW);
        bulk_copy(all + at * row_packs, static_cast<const X *>(p.x) + row * p.ld_x, bytes * XW, &x_landed[group][at]);
    };
    const auto fetch_rest = [&](long long row, int at) {
        uint4 *to = all + at * row_packs + packs * XW;
        expect(&rest_landed[group][at], bytes * (GATED ? 2 : 1));
        bulk_copy(to, static_cast<const T *>(p.residual) + row * p.ld_residual, bytes, &rest_landed[group][at]);
        if (GATED) bulk_copy(to + packs, static_cast<const T *>(p.gate) + row * p.ld_gate, bytes, &rest_landed[group][at]);
    };
    const long long step = (long long)gridDim.x * groups;
    long long row = (long long)blockIdx.x * groups + group;
    if (tid == 0) {
        for (int d = 0; d < depth; ++d) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&x_landed[group][d])) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&rest_landed[group][d])) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int d = 0; d < depth && row + d * step < p.rows; ++d) {
            fetch_x(row + d * step, d);
            fetch_rest(row + d * step, d);
        }
    }
    for (int e = threadIdx.x; e < p.h; e += blockDim.x) {
        float f = p.block_scale;
        if (p.post_gamma) f = __fmul_rn(f, load_gamma<T>(p.post_gamma, p.gamma32, e));
        if (channel_gate) f = __fmul_rn(f, gate_value(to_float<T>(static_cast<const T *>(p.gate)[e]), p.gate_act));
        const int at = (e % V / 4 * packs + e / V) * 4 + e % 4;   // four floats of every pack together, so that a warp reads no bank twice
        by_block[at] = f;
        if (p.gamma) by_gamma[at] = load_gamma<T>(p.gamma, p.gamma32, e);
        if (p.smooth) by_smooth[at] = p.smooth[e];
    }
    const auto has = [&](int i) { return EXACT || tid + i * threads < packs; };
    const auto factors = [&](const float *from, int c, f32x2 *f) {
#pragma unroll
        for (int e = 0; e < V; e += 4) unpack<float>(reinterpret_cast<const uint4 *>(from)[e / 4 * packs + c], f + e / 2);
    };
    __syncthreads();
    uint32_t phase = 0;
    int at = 0;     // the buffer that the row is in
    for (int parity = 0; row < p.rows; row += step, parity ^= 1) {
        const long long next = row + depth * step;   // what comes in its place
        const uint4 *mine = all + at * row_packs;
        const auto give_up = [&] {   // never while the GPU is well; what there is to see of it is a row of NaN
            if (tid == 0 && p.q) p.scale[row] = __int_as_float(0x7fffffff);
            if (tid == 0 && p.residual_out) static_cast<T *>(p.residual_out)[row * p.ld_residual_out] = from_float<T>(__int_as_float(0x7fffffff));
        };
        // the block's output, and the norm behind it
        f32x2 u[N][V / 2];
        if (!mbar_wait(&x_landed[group][at], phase)) return give_up();
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < XW; ++j) unpack<X>(has(i) ? mine[(tid + i * threads) * XW + j] : make_uint4(0, 0, 0, 0), u[i] + j * (V / 2 / XW));
        float factor = 1.0f;
        if (p.post_gamma) {
            f32x2 sum2 = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < V / 2; ++e) sum2 = fma2(u[i][e], u[i][e], sum2);
            const float2 parts = unpair2(sum2);
            float sum = parts.x + parts.y, unused = 0.0f;
            group_reduce(sum, unused, red[parity], group, threads);
            factor = rsqrtf(__fmaf_rn(sum, p.inv_h, p.post_eps));
        } else {
            group_sync(group, threads);
        }
        if (tid == 0 && next < p.rows) fetch_x(next, at);
        if (p.gate && p.gate_step == 0) factor = __fmul_rn(factor, gate_value(to_float<T>(static_cast<const T *>(p.gate)[row * p.ld_gate]), p.gate_act));

        // the residual stream, and the sums of the next norm
        if (!mbar_wait(&rest_landed[group][at], phase)) return give_up();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!has(i)) break;
            const int c = tid + i * threads;
            f32x2 f[V / 2], r[V / 2];
            factors(by_block, c, f);
            unpack<T>(mine[packs * XW + c], r);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) u[i][e] = mul2(u[i][e], mul2(f[e], pair2(factor, factor)));
            if (GATED) {
                unpack<T>(mine[packs * (XW + 1) + c], f);
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
        }
        if (p.residual_out) {
            uint4 *to = reinterpret_cast<uint4 *>(static_cast<T *>(p.residual_out) + row * p.ld_residual_out) + tid;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (has(i)) to[i * threads] = pack<T>(u[i]);
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
        if (tid == 0 && next < p.rows) fetch_rest(next, at);
        if (++at == depth) { at = 0; phase ^= 1; }
        if (!p.gamma) continue;
        const float r = rsqrtf(__fmaf_rn(sum, p.inv_h, p.eps));
        if (p.normed_out) {
            uint4 *normed = reinterpret_cast<uint4 *>(static_cast<T *>(p.normed_out) + row * p.ld_normed) + tid;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!has(i)) break;
                f32x2 y[V / 2];
#pragma unroll
                for (int e = 0; e < V / 2; ++e) y[e] = mul2(u[i][e], pair2(r, r));
                normed[i * threads] = pack<T>(y);
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
                int8_t *to = p.q + row * p.ld_q + c * V;
                if (V == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(q[0], q[V / 4 - 1]);
                else *reinterpret_cast<uint32_t *>(to) = q[0];
            }
        };
        if (quant.rcp != 0.0f) finish(true);
        else finish(false);
    }
}

// Threads of a group and groups of a CTA; 0 where a row does not fit.
struct Groups {
    int threads, groups, depth, smem;
};
template <typename T, typename X>
Groups groups_of(const SandwichParams &p)
{
    constexpr int V = 16 / (int)sizeof(T), XW = (int)sizeof(X) * V / 16;
    const int packs = p.h / V, most = group_threads_most(sizeof(T)), room = 224 * 1024;
    Groups g;
    g.threads = ((packs + kGroupPacks - 1) / kGroupPacks + 31) / 32 * 32;
    const int factors = 4 * p.h * (1 + (p.gamma != nullptr) + (p.smooth != nullptr));
    const int row = (XW + (p.gate && p.ld_gate && p.gate_step ? 2 : 1)) * 16 * packs;
    g.groups = most / g.threads;
    if (g.groups > kMaxGroups) g.groups = kMaxGroups;
    if (g.groups > (room - factors) / row) g.groups = room > factors ? (room - factors) / row : 0;
    g.depth = g.groups > 0 ? (room - factors) / (g.groups * row) : 0;   // rows of a group that there is room for
    if (g.depth > kMaxDepth) g.depth = kMaxDepth;
    g.smem = factors + g.groups * g.depth * row;
    return g;
}

template <typename T, typename X, bool WHOLE>
cudaError_t launch_packed(const SandwichParams &p, cudaStream_t stream)
{
    constexpr int V = 16 / (int)sizeof(T), XW = (int)sizeof(X) * V / 16;
    const int packs = (p.h + (WHOLE ? 0 : V - 1) + V - 1) / V;
    const auto warps = [](int n) { return (n + 31) / 32 * 32; };
    // Few rows: as many threads as a row has packs, for the shortest chain.  More: four packs a thread, for more rows on an SM, and the next
    // row's loads under way; the CTAs that find a place on the SMs together go through the rows.
    const int four = warps((packs + 3) / 4);
    if (packs <= 1024 && (p.rows <= 2 * 148 || packs <= 64)) {
        sandwich_kernel<T, X, 1, WHOLE, 1024, 1, false><<<p.rows, warps(packs), 0, stream>>>(p);
        return cudaGetLastError();
    }
    int dev = 0;
    cudaGetDevice(&dev);
    // once per device; the attribute is idempotent, so a race only repeats the call
    static unsigned long long done_mask = 0;
    const bool first = !((done_mask >> (dev & 63)) & 1ull);
    if constexpr (WHOLE) {
        const Groups g = groups_of<T, X>(p);
        if (g.groups > 0) {
            const bool exact = packs == kGroupPacks * g.threads, gated = p.gate && p.ld_gate && p.gate_step;
            const auto kernel = exact ? gated ? sandwich_rows_kernel<T, X, true, true> : sandwich_rows_kernel<T, X, true, false>
                                : gated ? sandwich_rows_kernel<T, X, false, true> : sandwich_rows_kernel<T, X, false, false>;
            const unsigned long long bit = 1ull << (dev & 63);
            static unsigned long long done[4] = {};   // as above
            unsigned long long &mask = done[2 * exact + gated];
            if (!(mask & bit)) {
                const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
                if (e != cudaSuccess) return e;
                mask |= bit;
            }
            const int ctas = (p.rows + g.groups - 1) / g.groups;
            kernel<<<ctas < 148 ? ctas : 148, g.threads * g.groups, g.smem, stream>>>(p, g.threads, g.groups, g.depth);
            return cudaGetLastError();
        }
    } else if (packs <= 4 * 512) {
        const int smem = (XW + (p.gate && p.ld_gate && p.gate_step ? 2 : 1)) * 4 * 16 * four;
        const int fit = 1024 / four < 220 * 1024 / (smem + 2048) ? 1024 / four : 220 * 1024 / (smem + 2048);
        const auto kernel = sandwich_kernel<T, X, 4, WHOLE, 512, 2, true>;
        if (first) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * 4 * 16 * 512);
            if (e != cudaSuccess) return e;
            done_mask |= 1ull << (dev & 63);
        }
        kernel<<<p.rows < 148 * fit ? p.rows : 148 * fit, four, smem, stream>>>(p);
        return cudaGetLastError();
    }
    if (packs <= 4 * 1024) {
        sandwich_kernel<T, X, 4, WHOLE, 1024, 1, false><<<p.rows, four, 0, stream>>>(p);
    } else {
        sandwich_any_kernel<T, X><<<p.rows, 256, 0, stream>>>(p);
    }
    return cudaGetLastError();
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
