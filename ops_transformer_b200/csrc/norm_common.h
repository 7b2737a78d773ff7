// What the kernels that work on rows share: packs of values as pairs of floats, the reduction over a block, the int8 step and
// its quotients.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gmm_common.h"

namespace gmm {
namespace {

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of T as pairs of floats, and back with one rounding each.  Values stay in pairs throughout: taken apart and put together
// again, they cost as many register moves as arithmetic.
template <typename T> __device__ __forceinline__ void unpack(const uint4 &u, f32x2 *f);
template <> __device__ __forceinline__ void unpack<float>(const uint4 &u, f32x2 *f)
{
    f[0] = pair2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = pair2(__uint_as_float(u.z), __uint_as_float(u.w));
}
template <> __device__ __forceinline__ void unpack<__half>(const uint4 &u, f32x2 *f)
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[i] = pair2(t.x, t.y);
    }
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4 &u, f32x2 *f)
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pair2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ uint4 pack(const f32x2 *f);
template <> __device__ __forceinline__ uint4 pack<float>(const f32x2 *f)
{
    const float2 a = unpair2(f[0]), b = unpair2(f[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
}
template <> __device__ __forceinline__ uint4 pack<__half>(const f32x2 *f)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpair2(f[i]);
        const __half2 t = __floats2half2_rn(v.x, v.y);
        w[i] = *reinterpret_cast<const uint32_t *>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <> __device__ __forceinline__ uint4 pack<__nv_bfloat16>(const f32x2 *f)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpair2(f[i]);
        const __nv_bfloat162 t = __floats2bfloat162_rn(v.x, v.y);
        w[i] = *reinterpret_cast<const uint32_t *>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float element(const f32x2 *f, int e)
{
    const float2 v = unpair2(f[e / 2]);
    return e % 2 ? v.y : v.x;
}

// Largest magnitude of three; a NaN is larger than all numbers, so that it is not passed over.
__device__ __forceinline__ float max_mag(float m, float a, float b)
{
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
    return r;
}

// Sum of `sum` and largest of `mag` over the block, in every thread; at most 32 warps.  The magnitudes are compared as unsigned
// numbers, which order like them (NaN last).
__device__ __forceinline__ void block_reduce(float &sum, float &mag, float2 *red)
{
    uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(mag) & 0x7fffffffu);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps > 1) {
        if (lane == 0) red[threadIdx.x >> 5] = make_float2(sum, __uint_as_float(m));
        __syncthreads();
        const float2 v = lane < warps ? red[lane] : make_float2(0.0f, 0.0f);
        sum = v.x;
        m = __reduce_max_sync(0xffffffffu, __float_as_uint(v.y));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    mag = __uint_as_float(m);
}

// How a row is divided by its step.  rcp: the correctly rounded reciprocal where the quotient can be formed with it, else 0.
struct Quantiser {
    float step, rcp;
    __device__ __forceinline__ void set(float s)
    {
        step = s;
        rcp = s > 1e-30f && s < 1e30f ? __frcp_rn(s) : 0.0f;
    }
    __device__ __forceinline__ uint32_t one(float u) const
    {
        if (!(step > 0.0f && step < __int_as_float(0x7f800000))) return 0u;
        return (uint32_t)max(-127, min(127, __float2int_rn(__fdiv_rn(u, step))));
    }
    // rint(u / step) of two values, in the low bytes.  q = u * rcp, twice q += (u - q * step) * rcp: after the first correction q is a
    // faithful rounding of the quotient, and with an exact residual and a correctly rounded reciprocal the second one yields the
    // correctly rounded quotient (Markstein's theorem), at most 127 in magnitude.  Adding 1.5 * 2^23 rounds it to an integer, ties to
    // even, in the low bits.
    __device__ __forceinline__ f32x2 two(f32x2 u) const
    {
        const f32x2 r = pair2(rcp, rcp), ns = pair2(-step, -step);
        f32x2 q = mul2(u, r);
        q = fma2(fma2(q, ns, u), r, q);
        q = fma2(fma2(q, ns, u), r, q);
        return fma2(q, pair2(1.0f, 1.0f), pair2(12582912.0f, 12582912.0f));
    }
    __device__ __forceinline__ uint32_t four(const f32x2 *u, bool by_rcp) const
    {
        if (by_rcp) {
            const f32x2 a = two(u[0]), b = two(u[1]);
            return __byte_perm(__byte_perm((uint32_t)a, (uint32_t)(a >> 32), 0x0040), __byte_perm((uint32_t)b, (uint32_t)(b >> 32), 0x0040), 0x5410);
        }
        return __byte_perm(__byte_perm(one(element(u, 0)), one(element(u, 1)), 0x0040),
                           __byte_perm(one(element(u, 2)), one(element(u, 3)), 0x0040), 0x5410);
    }
};

// m / 127, correctly rounded as in Quantiser::two; the rest of the range by division.
__device__ __forceinline__ float step_of(float m)
{
    if (!(m > 1e-28f && m < 1e30f)) return __fdiv_rn(m, 127.0f);
    const float r = 1.0f / 127.0f;
    float q = __fmul_rn(m, r);
    q = __fmaf_rn(__fmaf_rn(-q, 127.0f, m), r, q);
    return __fmaf_rn(__fmaf_rn(-q, 127.0f, m), r, q);
}

// 16 bytes.  LATE: not to be read before a wait for the kernel before, behind which the compiler would let a load of constants go.
template <bool LATE, typename P> __device__ __forceinline__ P load16(const P *p) { return LATE ? *p : __ldg(p); }

// V elements from `at` on, which stands anywhere: 16-bit weights out of two aligned packs where these lie inside, else one by one.
template <typename G, int V, bool LATE = false>
__device__ __forceinline__ void load_anywhere(const G *g, int at, int h, f32x2 *f)
{
    if constexpr (sizeof(G) == 2 && V == 8) {
        const int lo = at & ~7, shift = at & 7;
        if (at >= 0 && lo + 16 <= h) {
            const uint4 a = load16<LATE>(reinterpret_cast<const uint4 *>(g + lo)), b = load16<LATE>(reinterpret_cast<const uint4 *>(g + lo + 8));
            uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            if (shift & 4) { w[0] = w[2]; w[1] = w[3]; w[2] = w[4]; w[3] = w[5]; w[4] = w[6]; w[5] = w[7]; }
            if (shift & 2) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = w[4]; w[4] = w[5]; }
            const uint32_t bits = (shift & 1) * 16;
            unpack<G>(make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                                 __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits)), f);
            return;
        }
    }
    const auto one = [&](int e) { return e >= 0 && e < h ? to_float<G>(g[e]) : 0.0f; };
#pragma unroll
    for (int e = 0; e < V; e += 2) f[e / 2] = pair2(one(at + e), one(at + e + 1));
}
template <int V, bool LATE = false>
__device__ __forceinline__ void load_fp32(const float *g, f32x2 *f)
{
#pragma unroll
    for (int e = 0; e < V; e += 4) {
        const float4 v = load16<LATE>(reinterpret_cast<const float4 *>(g + e));
        f[e / 2] = pair2(v.x, v.y);
        f[e / 2 + 1] = pair2(v.z, v.w);
    }
}

}  // namespace
}  // namespace gmm
