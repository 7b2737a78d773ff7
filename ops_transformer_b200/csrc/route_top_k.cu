// route_top_k: the choice of experts of a mixture-of-experts layer.
//
//   s = sigmoid(l) or softmax(l);  c = s + bias;  groups ranked by max c or by the sum of their two largest c, the best ones stay;
//   ids = the k largest c that stay, ties to the lowest id;  weights = s[ids] (/ their sum) * scale
// Where neither a bias nor a sum of two scores decides, the logits stand for c: both score functions grow with them, so only the k
// scores that are returned are computed (and with `renormalize` softmax needs no sum over all experts, since it cancels).
//
// One warp per row.  A group's experts lie in `sub` neighbouring lanes (sub * groups <= 32, sub a power of two), `per` consecutive ones
// in each: lower experts are in lower lanes and lower registers, and a group is ranked by shuffles among its lanes.  Candidates are
// compared as unsigned keys that order like their values; key 0 is no candidate.
//
// The k-th largest of the lanes' maxima bounds the k-th largest key from below, and few keys reach it: those are gathered, one to a lane,
// and each counts how many stand before it (larger, or equal with a lower id), which is its place in the result.  Taking the largest key
// k times over instead, with the owner's registers searched every time, was 25 us for 16384 rows of 256; it is left for rows where more
// than 32 keys reach the bound (many equal ones, or a large k).
//
// Bound by instructions: some 800 a row and warp for 256 experts in eight groups (16384 rows 15 us, where reading the logits takes 2.7),
// softmax without groups and bias 11.3 us, 128 experts 9.6 us, 64 8.4.  Few rows cost a warp's chain: 2.8 us for 16.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gmm_common.h"

namespace gmm {
namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kWarps = 4;

struct RouteParams {
    const void *logits;
    int dtype;
    long long ld;
    const float *bias;
    const int8_t *token_mask;
    int rows, experts, top_k;
    int groups, group_size, topk_group, sub, sub_log, per;
    bool whole;                // every lane's experts fill its registers and start on a boundary of their own size (at most 16 bytes)
    bool renormalize, ids_i64;
    float scale;
    float *weights;
    void *ids;
};

__device__ __forceinline__ float minus_inf() { return __int_as_float(0xff800000); }

// R values of a lane with as wide loads as there are.
template <typename T, int R>
__device__ __forceinline__ void load_wide(const T *from, float (&l)[R])
{
    constexpr int BYTES = R * (int)sizeof(T), STEP = BYTES < 16 ? BYTES : 16, N = STEP / (int)sizeof(T);
    struct alignas(STEP) Pack { T v[N]; };
#pragma unroll
    for (int i = 0; i < R; i += N) {
        const Pack q = *reinterpret_cast<const Pack *>(from + i);
#pragma unroll
        for (int e = 0; e < N; ++e) l[i + e] = (float)q.v[e];
    }
}
template <typename T, int R>
__device__ __forceinline__ void load_logits(const RouteParams &p, long long at, int mine, float (&l)[R])
{
    const T *from = reinterpret_cast<const T *>(p.logits) + at;
    if (p.whole) {
        load_wide<T, R>(from, l);
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) l[i] = i < mine ? (float)from[i] : minus_inf();
    }
}

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

__device__ __forceinline__ float sigmoid(float l) { return __frcp_rn(__fadd_rn(1.0f, expf(-l))); }
// exp(l - top); the largest logit gives 1 also where it is infinite.
__device__ __forceinline__ float exp_below(float l, float top) { return l == top ? 1.0f : expf(__fsub_rn(l, top)); }

__device__ __forceinline__ void put(const RouteParams &p, long long at, float w, int id)
{
    p.weights[at] = w;
    if (p.ids_i64) reinterpret_cast<int64_t *>(p.ids)[at] = id;
    else reinterpret_cast<int32_t *>(p.ids)[at] = id;
}

// Sigmoid to within 3e-7 in five instructions; the exact one takes thirty.
__device__ __forceinline__ float sigmoid_about(float l)
{
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(l, -1.44269504f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.0f, e)));
    return r;
}

// The choice by sigmoid scores plus a bias, from scores that are only about right.  Such a score is off by less than 6e-7 from the one that
// the definition rounds (both count their own errors: 3e-7 here; exp, sum and quotient there), a sum with the bias by a unit of its last
// place more.  Groups that differ by more than these errors together stay or go as with exact scores; and the k-th largest lane maximum,
// less the errors, bounds the k-th largest exact choice from below.  So the few experts that reach it are the only ones whose exact score
// is needed, and each has a lane of its own for that (16384 rows of 256 in eight groups: 15.0 us, 17.1 with exact scores throughout).
// False, with nothing written, where two groups are too close, where infinities are about or more than 32 experts reach the bound: then
// every score is computed exactly.
template <int R, bool TOP2>
__device__ __forceinline__ bool route_about(const RouteParams &p, const float (&l)[R], const float (&bias)[R], int group, int first, long long out,
                                            unsigned long long *list_key, float *list_logit, int *list_id)
{
    const int lane = threadIdx.x & 31;
    float c[R], best = minus_inf(), second = minus_inf();
#pragma unroll
    for (int i = 0; i < R; ++i) {
        c[i] = sigmoid_about(l[i]);
        if (p.bias) c[i] = __fadd_rn(c[i], bias[i]);
        c[i] = l[i] > minus_inf() && c[i] > minus_inf() ? c[i] : minus_inf();   // NaN too
        if (TOP2) second = fmaxf(second, fminf(best, c[i]));
        best = fmaxf(best, c[i]);
    }
    float top = best;
    bool stays = true;
    if (p.groups > 1) {
        for (int o = 1; o < p.sub; o <<= 1) {
            const float ob = __shfl_xor_sync(kAll, best, o);
            if (TOP2) second = fmaxf(fmaxf(second, __shfl_xor_sync(kAll, second, o)), fminf(best, ob));
            best = fmaxf(best, ob);
        }
        const float rank = TOP2 && second > minus_inf() ? __fadd_rn(best, second) : best;
        // What two groups' ranks may be off by together.  The largest choices of groups that are close are of one size; the parts of a sum
        // may be far larger than it, and another group's larger than this one's: there it goes by the largest parts of the row.
        float size = fabsf(rank);
        if (TOP2) {
            const float parts = second > minus_inf() ? fabsf(best) + fabsf(second) : fabsf(best);
            size = __uint_as_float(__reduce_max_sync(kAll, best > minus_inf() ? __float_as_uint(parts) : 0u));
        }
        const float margin = 3e-6f + 1e-6f * size;
        const float above = __fadd_rn(rank, margin), below = __fsub_rn(rank, margin);
        int surely = 0, maybe = -1;   // groups that are, that may be better; it is no better than itself
#pragma unroll 8
        for (int g = 0; g < p.groups; ++g) {
            const float r = __shfl_sync(kAll, rank, g << p.sub_log);
            surely += r > above;
            maybe += r > below;
        }
        stays = maybe < p.topk_group;
        const bool gone = surely >= p.topk_group || !(rank > minus_inf());
        // an infinite rank has no margin
        if (__any_sync(kAll, group < p.groups && ((!stays && !gone) || rank > 1e30f))) return false;
        stays = stays && !gone;
    }
    uint32_t rest = stays && top > minus_inf() ? key_of(top) : 0u, last = 0u;
    bool all = false;   // fewer lanes than k have a candidate
    for (int j = 0; j < p.top_k; ++j) {
        const uint32_t m = __reduce_max_sync(kAll, rest);
        if (m == 0u) { all = true; break; }
        last = m;
        if (rest == m) rest = 0u;
    }
    const float kth = __uint_as_float(last ^ (last & 0x80000000u ? 0x80000000u : 0xffffffffu));
    if (last != 0u && !(fabsf(kth) < 1e30f)) return false;
    // a lane whose group is gone compares with something that nothing reaches
    const float lowest = -3.402823466e38f, bound = !stays ? __int_as_float(0x7fc00000) : all ? lowest : kth - (1.5e-6f + 4e-7f * fabsf(kth));
    int count = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) count += c[i] >= bound;
    int before = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(kAll, before, o);
        if (lane >= o) before += t;
    }
    const int found = __shfl_sync(kAll, before, 31);
    if (found > 32) return false;
    before -= count;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (c[i] >= bound) {
            list_logit[before] = l[i];
            list_id[before] = first + i;
            ++before;
        }
    }
    __syncwarp();
    float exact = 0.0f;
    int id = -1, place = lane;
    unsigned long long own = 0ull;
    if (lane < found) {
        id = list_id[lane];
        exact = sigmoid(list_logit[lane]);
        const float choice = p.bias ? __fadd_rn(exact, __ldg(p.bias + id)) : exact;
        own = (unsigned long long)key_of(choice) << 32 | (uint32_t)~id;
    }
    list_key[lane] = own;
    __syncwarp();
    if (lane < found) {
        place = 0;
        for (int q = 0; q < found; q += 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) place += list_key[q + e] > own;
        }
    }
    float w = place < p.top_k && id >= 0 ? exact : 0.0f;
    if (p.renormalize) {
        const float sum = warp_sum(w);
        w = sum > 0.0f ? __fdiv_rn(w, sum) : 0.0f;
    }
    if (place < p.top_k) put(p, out + place, __fmul_rn(w, p.scale), id);
    return true;
}

// SCORED: c is computed for every expert, else it is the logit.  R: experts per lane, at least p.per.
template <int R, bool SIGMOID, bool SCORED, bool TOP2>
__global__ void __launch_bounds__(32 * kWarps) route_kernel(const RouteParams p)
{
    __shared__ unsigned long long list_key[kWarps][32];   // key, then the id with its bits inverted: equal keys order by the lower id
    __shared__ float list_logit[kWarps][32];
    __shared__ int list_id[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x * kWarps + warp;
    if (row >= p.rows) return;
    const long long out = (long long)row * p.top_k;
    if (p.token_mask && p.token_mask[row] == 0) {
        if (lane < p.top_k) put(p, out + lane, 0.0f, -1);
        return;
    }
    const int group = lane >> p.sub_log, inside = (lane & (p.sub - 1)) * p.per;
    const int first = group * p.group_size + inside;
    const int mine = group < p.groups ? max(0, min(p.per, p.group_size - inside)) : 0;
    float l[R];
    const long long at = (long long)row * p.ld + first;
    if (p.dtype == kF32) load_logits<float, R>(p, at, mine, l);
    else if (p.dtype == kBF16) load_logits<__nv_bfloat16, R>(p, at, mine, l);
    else load_logits<__half, R>(p, at, mine, l);
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (!(l[i] > minus_inf())) l[i] = minus_inf();   // NaN too
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
        } else if (!p.renormalize) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) t += l[i] > minus_inf() ? exp_below(l[i], top) : 0.0f;
            total = warp_sum(t);
        }
    }
    // without SCORED and with renormalisation the sum over all experts cancels: total stays 1
    const auto score = [&](float v) { return SIGMOID ? sigmoid(v) : __fdiv_rn(exp_below(v, top), total); };
    float bias[R];
    if (SCORED && p.bias) {
        if (p.whole) {
            load_wide<float, R>(p.bias + first, bias);
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i) bias[i] = i < mine ? __ldg(p.bias + first + i) : 0.0f;
        }
    }
    if constexpr (SIGMOID && SCORED) {
        if (route_about<R, TOP2>(p, l, bias, group, first, out, list_key[warp], list_logit[warp], list_id[warp])) return;
        __syncwarp();
    }
    float best = minus_inf(), second = minus_inf();
    uint32_t key[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float c = l[i];
        if (SCORED) {
            c = score(c);
            if (p.bias) c = __fadd_rn(c, bias[i]);
            c = l[i] > minus_inf() && c > minus_inf() ? c : minus_inf();
        }
        key[i] = c > minus_inf() ? key_of(c) : 0u;
        if (TOP2) second = fmaxf(second, fminf(best, c));
        best = fmaxf(best, c);
    }
    uint32_t top_key = best > minus_inf() ? key_of(best) : 0u;
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
            top_key = 0u;
#pragma unroll
            for (int i = 0; i < R; ++i) key[i] = 0u;
        }
    }
    // a bound that at least k keys reach, or all there are
    uint32_t bound = 1u;
    {
        uint32_t rest = top_key;
        for (int j = 0; j < p.top_k; ++j) {
            const uint32_t m = __reduce_max_sync(kAll, rest);
            if (m == 0u) { bound = 1u; break; }
            bound = m;
            if (rest == m) rest = 0u;
        }
    }
    int count = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) count += key[i] >= bound;
    int before = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(kAll, before, o);
        if (lane >= o) before += t;
    }
    const int found = __shfl_sync(kAll, before, 31);
    before -= count;
    float chosen = 0.0f;
    int id = -1, place = lane;
    if (found <= 32) {
        list_key[warp][lane] = 0ull;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (key[i] >= bound) {
                list_key[warp][before] = (unsigned long long)key[i] << 32 | (uint32_t)~(first + i);
                list_logit[warp][before] = l[i];
                ++before;
            }
        }
        __syncwarp();
        const unsigned long long own = list_key[warp][lane];
        place = 0;
        for (int q = 0; q < found; q += 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) place += list_key[warp][q + e] > own;
        }
        if (lane < found) {
            chosen = list_logit[warp][lane];
            id = ~(int)(uint32_t)own;
        } else {
            place = lane;   // at least `found`: a slot for which there is no expert
        }
    } else {
        // k rounds: the largest key of the warp, the first one of equal ones
        for (int j = 0; j < p.top_k; ++j) {
            uint32_t m = key[0];
#pragma unroll
            for (int i = 1; i < R; ++i) m = max(m, key[i]);
            const uint32_t warp_m = __reduce_max_sync(kAll, m);
            const int owner = __ffs(__ballot_sync(kAll, m == warp_m)) - 1;
            float v = 0.0f;
            int it = 0;
            if (lane == owner) {
                bool done = false;
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    if (!done && key[i] == warp_m) {
                        done = true;
                        it = first + i;
                        v = l[i];
                        key[i] = 0u;
                    }
                }
            }
            v = __shfl_sync(kAll, v, owner);
            it = __shfl_sync(kAll, it, owner);
            if (lane == j) { chosen = v; id = it; }
        }
    }
    float w = place < p.top_k && id >= 0 ? score(chosen) : 0.0f;
    if (p.renormalize) {
        const float sum = warp_sum(w);
        w = sum > 0.0f ? __fdiv_rn(w, sum) : 0.0f;
    }
    if (place < p.top_k) put(p, out + place, __fmul_rn(w, p.scale), id);
}

template <int R, bool SIGMOID>
void launch_scored(const RouteParams &p, bool scored, bool top2, cudaStream_t stream)
{
    const unsigned grid = (unsigned)((p.rows + kWarps - 1) / kWarps);
    if (!scored) route_kernel<R, SIGMOID, false, false><<<grid, 32 * kWarps, 0, stream>>>(p);
    else if (!top2) route_kernel<R, SIGMOID, true, false><<<grid, 32 * kWarps, 0, stream>>>(p);
    else route_kernel<R, SIGMOID, true, true><<<grid, 32 * kWarps, 0, stream>>>(p);
}

template <int R>
void launch_rows(RouteParams &p, const RouteTopKProblem &r, cudaStream_t stream)
{
    const int bytes = R * (r.dtype == kF32 ? 4 : 2), step = bytes < 16 ? bytes : 16;
    const long long pitch = r.ld * (r.dtype == kF32 ? 4 : 2);
    p.whole = p.per == R && p.sub * R == p.group_size && p.sub * p.groups == 32 && (((uintptr_t)r.logits | (uintptr_t)pitch) & (uintptr_t)(step - 1)) == 0 &&
              ((uintptr_t)r.bias & 15) == 0;
    const bool top2 = r.n_group > 1 && r.group_score == kGroupTop2, scored = r.bias || top2;
    if (r.scoring == kScoreSigmoid) launch_scored<R, true>(p, scored, top2, stream);
    else launch_scored<R, false>(p, scored, top2, stream);
}

}  // namespace

cudaError_t route_top_k_launch(const RouteTopKProblem &r, cudaStream_t stream)
{
    if (r.rows <= 0) return cudaSuccess;
    RouteParams p;
    p.logits = r.logits; p.dtype = r.dtype; p.ld = r.ld; p.bias = r.bias; p.token_mask = r.token_mask;
    p.rows = (int)r.rows; p.experts = r.experts; p.top_k = r.top_k;
    p.groups = r.n_group; p.group_size = r.experts / r.n_group; p.topk_group = r.topk_group;
    p.sub = 32;
    p.sub_log = 5;
    while (p.sub * p.groups > 32) { p.sub >>= 1; --p.sub_log; }
    p.per = (p.group_size + p.sub - 1) / p.sub;   // below 2 * 1024 / 32: more than half of the lanes have a group
    p.renormalize = r.renormalize; p.ids_i64 = r.ids_i64;
    p.scale = r.scale; p.weights = r.weights; p.ids = r.ids;
    if (p.per <= 2) launch_rows<2>(p, r, stream);
    else if (p.per <= 4) launch_rows<4>(p, r, stream);
    else if (p.per <= 8) launch_rows<8>(p, r, stream);
    else if (p.per <= 16) launch_rows<16>(p, r, stream);
    else launch_rows<64>(p, r, stream);
    return cudaGetLastError();
}

}  // namespace gmm
