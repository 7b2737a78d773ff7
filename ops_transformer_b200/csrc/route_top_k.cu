// route_top_k: the choice of experts of a mixture-of-experts layer.
//
//   s = sigmoid(l) or softmax(l);  c = s + bias;  groups ranked by max c or by the sum of their two largest c, the best ones stay;
//   ids = the k largest c that stay, ties to the lowest id;  weights = s[ids] (/ their sum) * scale
// Where neither a bias nor a sum of two scores decides, the logits stand for c: both score functions grow with them, so only the k
// scores that are returned are computed (and with `renormalize` softmax needs no sum over all experts, since it cancels).
//
// One warp per row.  A group's experts lie in `sub` neighbouring lanes (sub * groups <= 32, sub a power of two), `per` consecutive ones
// in each: lower experts are in lower lanes and lower registers, so the first of equal candidates has the lowest id, and a group is
// ranked by shuffles among its lanes.  Candidates are compared as unsigned keys that order like their values; key 0 is no candidate.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gmm_common.h"

namespace gmm {
namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kWarps = 4;

struct RouteParams {
    const void *logits;
    long long ld;
    const float *bias;
    const int8_t *token_mask;
    int rows, experts, top_k;
    int groups, group_size, topk_group, sub, per;
    float scale;
    float *weights;
    void *ids;
};

template <typename T> __device__ __forceinline__ float load_logit(const void *p, long long at);
template <> __device__ __forceinline__ float load_logit<float>(const void *p, long long at) { return __ldg(reinterpret_cast<const float *>(p) + at); }
template <> __device__ __forceinline__ float load_logit<__half>(const void *p, long long at) { return __half2float(reinterpret_cast<const __half *>(p)[at]); }
template <> __device__ __forceinline__ float load_logit<__nv_bfloat16>(const void *p, long long at) { return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[at]); }

__device__ __forceinline__ float minus_inf() { return __int_as_float(0xff800000); }

// Orders like v for all v above minus infinity; adding zero makes the two zeros equal.
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
}

__device__ __forceinline__ float sigmoid(float l) { return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-l))); }
// exp(l - top); the largest logit gives 1 also where it is infinite.
__device__ __forceinline__ float exp_below(float l, float top) { return l == top ? 1.0f : expf(__fsub_rn(l, top)); }

// SCORED: c is computed for every expert, else it is the logit.  R: experts per lane, at least p.per.
template <typename T, typename I, int R, bool SIGMOID, bool SCORED, bool TOP2, bool RENORM>
__global__ void __launch_bounds__(32 * kWarps) route_kernel(const RouteParams p)
{
    const int lane = threadIdx.x & 31;
    const int row = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    float *weights = p.weights + (long long)row * p.top_k;
    I *ids = reinterpret_cast<I *>(p.ids) + (long long)row * p.top_k;
    if (p.token_mask && p.token_mask[row] == 0) {
        if (lane < p.top_k) { weights[lane] = 0.0f; ids[lane] = (I)-1; }
        return;
    }
    const int group = lane / p.sub, inside = (lane % p.sub) * p.per;
    const int first = group * p.group_size + inside;
    const int mine = group < p.groups ? max(0, min(p.per, p.group_size - inside)) : 0;
    float l[R];
    uint32_t key[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        l[i] = i < mine ? load_logit<T>(p.logits, (long long)row * p.ld + first + i) : minus_inf();
        if (!(l[i] > minus_inf())) l[i] = minus_inf();   // NaN too
    }
    float top = 0.0f, total = 1.0f;
    if (!SIGMOID) {
        top = l[0];
#pragma unroll
        for (int i = 1; i < R; ++i) top = fmaxf(top, l[i]);
        top = warp_max(top);
        if (SCORED) {   // the choice hangs on the last bit of this sum, which 64 bits make independent of the order of its terms
            double t = 0.0;
#pragma unroll
            for (int i = 0; i < R; ++i) t += l[i] > minus_inf() ? (double)exp_below(l[i], top) : 0.0;
            total = (float)warp_sum(t);
        } else if (!RENORM) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) t += l[i] > minus_inf() ? exp_below(l[i], top) : 0.0f;
            total = warp_sum(t);
        }
    }
    const auto score = [&](float v) { return SIGMOID ? sigmoid(v) : !SCORED && RENORM ? exp_below(v, top) : __fdiv_rn(exp_below(v, top), total); };
    float best = minus_inf(), second = minus_inf();
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float c = l[i];
        if (SCORED && c > minus_inf()) {
            c = score(c);
            if (p.bias) c = __fadd_rn(c, __ldg(p.bias + first + i));
        }
        key[i] = c > minus_inf() ? key_of(c) : 0u;
        if (!(c > minus_inf())) c = minus_inf();
        if (TOP2) second = fmaxf(second, fminf(best, c));
        best = fmaxf(best, c);
    }
    if (p.groups > 1) {
        for (int o = 1; o < p.sub; o <<= 1) {
            const float ob = __shfl_xor_sync(kAll, best, o);
            if (TOP2) second = fmaxf(fmaxf(second, __shfl_xor_sync(kAll, second, o)), fminf(best, ob));
            best = fmaxf(best, ob);
        }
        const float rank = TOP2 && second > minus_inf() ? __fadd_rn(best, second) : best;
        int better = 0;
        for (int g = 0; g < p.groups; ++g) {
            const float r = __shfl_sync(kAll, rank, g * p.sub);
            better += r > rank || (r == rank && g < group);
        }
        if (better >= p.topk_group) {
#pragma unroll
            for (int i = 0; i < R; ++i) key[i] = 0u;
        }
    }
    // k rounds: the largest key of the warp, the first one of equal ones
    float chosen = 0.0f;
    int id = -1;
    for (int j = 0; j < p.top_k; ++j) {
        uint32_t m = key[0];
#pragma unroll
        for (int i = 1; i < R; ++i) m = max(m, key[i]);
        const uint32_t warp_m = __reduce_max_sync(kAll, m);
        if (warp_m == 0) break;
        const int owner = __ffs(__ballot_sync(kAll, m == warp_m)) - 1;
        float v = 0.0f;
        int at = 0;
        if (lane == owner) {
            bool found = false;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (!found && key[i] == warp_m) {
                    found = true;
                    at = first + i;
                    v = l[i];
                    key[i] = 0u;
                }
            }
        }
        v = __shfl_sync(kAll, v, owner);
        at = __shfl_sync(kAll, at, owner);
        if (lane == j) { chosen = v; id = at; }
    }
    float w = id >= 0 ? score(chosen) : 0.0f;
    if (RENORM) {
        const float sum = warp_sum(w);
        w = sum > 0.0f ? __fdiv_rn(w, sum) : 0.0f;
    }
    if (lane < p.top_k) {
        weights[lane] = __fmul_rn(w, p.scale);
        ids[lane] = (I)id;
    }
}

template <typename T, typename I, int R, bool SIGMOID, bool RENORM>
void launch_scored(const RouteParams &p, bool scored, bool top2, cudaStream_t stream)
{
    const unsigned grid = (unsigned)((p.rows + kWarps - 1) / kWarps);
    if (!scored) route_kernel<T, I, R, SIGMOID, false, false, RENORM><<<grid, 32 * kWarps, 0, stream>>>(p);
    else if (!top2) route_kernel<T, I, R, SIGMOID, true, false, RENORM><<<grid, 32 * kWarps, 0, stream>>>(p);
    else route_kernel<T, I, R, SIGMOID, true, true, RENORM><<<grid, 32 * kWarps, 0, stream>>>(p);
}

template <typename T, typename I, int R>
void launch_rows(const RouteParams &p, const RouteTopKProblem &r, cudaStream_t stream)
{
    const bool top2 = r.n_group > 1 && r.group_score == kGroupTop2, scored = r.bias || top2;
    if (r.scoring == kScoreSigmoid) {
        if (r.renormalize) launch_scored<T, I, R, true, true>(p, scored, top2, stream);
        else launch_scored<T, I, R, true, false>(p, scored, top2, stream);
    } else {
        if (r.renormalize) launch_scored<T, I, R, false, true>(p, scored, top2, stream);
        else launch_scored<T, I, R, false, false>(p, scored, top2, stream);
    }
}

template <typename T, typename I>
cudaError_t launch_typed(const RouteParams &p, const RouteTopKProblem &r, cudaStream_t stream)
{
    if (p.per <= 2) launch_rows<T, I, 2>(p, r, stream);
    else if (p.per <= 8) launch_rows<T, I, 8>(p, r, stream);
    else launch_rows<T, I, 64>(p, r, stream);
    return cudaGetLastError();
}

}  // namespace

cudaError_t route_top_k_launch(const RouteTopKProblem &r, cudaStream_t stream)
{
    if (r.rows <= 0) return cudaSuccess;
    RouteParams p;
    p.logits = r.logits; p.ld = r.ld; p.bias = r.bias; p.token_mask = r.token_mask;
    p.rows = (int)r.rows; p.experts = r.experts; p.top_k = r.top_k;
    p.groups = r.n_group; p.group_size = r.experts / r.n_group; p.topk_group = r.topk_group;
    p.sub = 32;
    while (p.sub * p.groups > 32) p.sub >>= 1;
    p.per = (p.group_size + p.sub - 1) / p.sub;   // below 2 * 1024 / 32: more than half of the lanes have a group
    p.scale = r.scale; p.weights = r.weights; p.ids = r.ids;
    switch (r.dtype) {
        case kF32: return r.ids_i64 ? launch_typed<float, int64_t>(p, r, stream) : launch_typed<float, int32_t>(p, r, stream);
        case kF16: return r.ids_i64 ? launch_typed<__half, int64_t>(p, r, stream) : launch_typed<__half, int32_t>(p, r, stream);
        case kBF16: return r.ids_i64 ? launch_typed<__nv_bfloat16, int64_t>(p, r, stream) : launch_typed<__nv_bfloat16, int32_t>(p, r, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace gmm
