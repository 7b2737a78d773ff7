// expert_balance: how a router's choices load the experts, the loss that evens them out, and its gradient.
//
//   p = softmax(l), or sigmoid(l) / sum of the row's;  per sequence of T tokens: counts c[e], P[e] = sum of p[e] over its tokens
//   loss = sum over the sequences of weight * sum_e c[e] P[e],  weight = coefficient * experts / (top_k * T^2 * sequences with a token)
//   d loss / d l[e] = weight * p[e] * (c[e] - sum_j p[j] c[j])   (sigmoid: times 1 - sigmoid(l[e]))
//
// The loss needs the counts of all tokens, so its gradient reads the logits a second time and forms p anew: 1 KB a row from memory against
// the same to write p and read it back.  A warp holds a row, a lane its share of the experts; sums over tokens are made in a fixed order
// (a lane's rows one after the other, then the warps, then the blocks), so that a call gives the same bits every time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gmm_common.h"

namespace gmm {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct BalanceParams {
    const void *logits;
    long long ld;
    const int8_t *mask;
    const int *cu;
    const void *ids;
    bool ids_i64;
    int top_k, rows, experts, sequences;
    float coefficient;
    float *loss, *weight;
    long long *counts;
    const float *grad_loss;
    void *grad;
    long long ld_grad;
    // workspace of the loss: what a block of rows adds to a sequence stands in the piece `block + sequence`, which is another one for every
    // block and sequence that meet, since both only grow on the way through the rows
    int chunk, blocks;                  // rows of a block, blocks
    int *ticket;
    int *piece_tokens;                  // [blocks + sequences]
    int *piece_counts;                  // [blocks + sequences, experts]
    float *piece_sums;                  // the same
    int *seq_tokens;                    // [sequences]
    double *seq_dots;                   // [sequences, ceil(experts / 32)]
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr float kInf = __builtin_huge_valf();

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The expert of a lane's i-th value: V neighbours at a time.
template <int V>
__device__ __forceinline__ int expert_of(int i, int lane) { return (i / V * 32 + lane) * V + i % V; }

// A row's logits; minus infinity where there is no expert.  V: values of one 16-byte load, or 1.
template <typename T, int PER, int V>
__device__ __forceinline__ void load_row(const T *row, int experts, int lane, float (&l)[PER])
{
#pragma unroll
    for (int i = 0; i < PER; i += V) {
        const int e = expert_of<V>(i, lane);
        if constexpr (V > 1) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (e < experts) u = *reinterpret_cast<const uint4 *>(row + e);
            const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
            for (int j = 0; j < V; ++j) l[i + j] = e < experts ? to_float<T>(t[j]) : -kInf;
        } else {
            l[i] = e < experts ? to_float<T>(row[e]) : -kInf;
        }
    }
}

// p in the place of a row's logits, and for the sigmoid's gradient 1 - sigmoid.  An expert whose logit is NaN or minus infinity is not
// there; a row without one is all zeros.
template <bool SIGMOID, int PER>
__device__ __forceinline__ void scores(float (&l)[PER], float (&rest)[PER])
{
    float total = 0.0f;
    if constexpr (SIGMOID) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float t = expf(-fabsf(l[i])), big = __fdividef(1.0f, 1.0f + t), small = __fmul_rn(t, big);   // of |l| and -|l|
            const bool there = l[i] > -kInf;
            rest[i] = !there ? 0.0f : l[i] >= 0.0f ? small : big;
            l[i] = !there ? 0.0f : l[i] >= 0.0f ? big : small;
            total += l[i];
        }
    } else {
        float top = -kInf;
#pragma unroll
        for (int i = 0; i < PER; ++i) top = fmaxf(top, l[i]);   // passes NaN over
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            l[i] = !(l[i] > -kInf) ? 0.0f : l[i] == top ? 1.0f : expf(l[i] - top);
            total += l[i];
        }
    }
    total = warp_sum(total);
    const float inv = total > 0.0f ? __frcp_rn(total) : 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) l[i] = __fmul_rn(l[i], inv);
}

// Rows of sequence s, cut to those that there are.
__device__ __forceinline__ int seq_begin(const BalanceParams &p, int s) { return p.cu ? min(max(p.cu[s], 0), p.rows) : 0; }
__device__ __forceinline__ int seq_end(const BalanceParams &p, int s) { return p.cu ? min(max(p.cu[s + 1], 0), p.rows) : p.rows; }
// The first sequence that ends behind `row`.
__device__ __forceinline__ int seq_of(const BalanceParams &p, int row)
{
    int lo = 0, hi = p.sequences;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (seq_end(p, mid) > row) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ float weight_of(const BalanceParams &p, int tokens, int sequences)
{
    return tokens > 0 ? (float)((double)p.coefficient * p.experts / ((double)p.top_k * tokens * tokens * sequences)) : 0.0f;
}

// What the rows of a block add to the sequences that they belong to.  ALL: one block holds all rows of the one sequence, and finishes.
template <typename T, bool SIGMOID, int PER, int V, bool ALL>
__global__ void __launch_bounds__(kThreads) balance_rows_kernel(const BalanceParams p)
{
    extern __shared__ float sums[];     // [warps][experts], then the counts [experts]
    __shared__ int warp_tokens[kWarps];
    __shared__ double warp_dots[kWarps];
    int *counts = reinterpret_cast<int *>(sums + kWarps * p.experts);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, block = blockIdx.x;
    if (!ALL && block == 0 && tid == 0) *p.ticket = 0;
    const int row0 = block * p.chunk, row1 = min(row0 + p.chunk, p.rows);
    for (int s = ALL ? 0 : seq_of(p, row0); s < p.sequences; ++s) {
        const int begin = max(seq_begin(p, s), row0), end = min(seq_end(p, s), row1);
        if (!ALL && seq_begin(p, s) >= row1) break;
        if (!ALL && begin >= end) continue;
        for (int e = tid; e < p.experts; e += kThreads) counts[e] = 0;
        __syncthreads();
        float sum[PER] = {};
        int tokens = 0;
        for (int row = begin + warp; row < end; row += kWarps) {
            if (p.mask && p.mask[row] == 0) continue;
            ++tokens;
            float l[PER], rest[PER];
            load_row<T, PER, V>(static_cast<const T *>(p.logits) + row * p.ld, p.experts, lane, l);
            scores<SIGMOID, PER>(l, rest);
#pragma unroll
            for (int i = 0; i < PER; ++i) sum[i] += l[i];
        }
        const long long id0 = (long long)begin * p.top_k;
        const long long pairs = (long long)(end - begin) * p.top_k;
        for (long long i = tid; i < pairs; i += kThreads) {
            if (p.mask && p.mask[begin + i / p.top_k] == 0) continue;
            const long long id = p.ids_i64 ? static_cast<const long long *>(p.ids)[id0 + i] : static_cast<const int *>(p.ids)[id0 + i];
            if (id >= 0 && id < p.experts) atomicAdd(counts + id, 1);
        }
        if (lane == 0) warp_tokens[warp] = tokens;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = expert_of<V>(i, lane);
            if (e < p.experts) sums[warp * p.experts + e] = sum[i];
        }
        __syncthreads();
        tokens = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) tokens += warp_tokens[w];
        double dot = 0.0;
        for (int e = tid; e < p.experts; e += kThreads) {
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) total += sums[w * p.experts + e];
            if (ALL) {
                p.counts[e] = counts[e];
                dot += (double)total * counts[e];
            } else {
                p.piece_sums[(long long)(block + s) * p.experts + e] = total;
                p.piece_counts[(long long)(block + s) * p.experts + e] = counts[e];
            }
        }
        if (ALL) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            if (lane == 0) warp_dots[warp] = dot;
            __syncthreads();
            if (tid == 0) {
                dot = 0.0;
                for (int w = 0; w < kWarps; ++w) dot += warp_dots[w];
                const float weight = weight_of(p, tokens, 1);
                p.weight[0] = weight;
                *p.loss = (float)(dot * weight);
            }
            return;
        }
        if (tid == 0) p.piece_tokens[block + s] = tokens;
        __syncthreads();
    }
}

// The pieces of a sequence, 32 experts a block; the block that comes last makes the loss of all.
__global__ void __launch_bounds__(kThreads) balance_finish_kernel(const BalanceParams p)
{
    __shared__ float sums[kWarps][32];
    __shared__ int counts[kWarps][32], tokens_of[kWarps];
    __shared__ double warp_dots[kWarps];
    __shared__ int last, some;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.y, parts = gridDim.x;
    const int e = blockIdx.x * 32 + lane, begin = seq_begin(p, s), end = seq_end(p, s);
    const int first = begin / p.chunk, behind = begin < end ? (end - 1) / p.chunk + 1 : first;
    float sum = 0.0f;
    int count = 0, tokens = 0;
    for (int b = first + warp; b < behind; b += kWarps) {
        if (e < p.experts) {
            sum += p.piece_sums[(long long)(b + s) * p.experts + e];
            count += p.piece_counts[(long long)(b + s) * p.experts + e];
        }
        tokens += p.piece_tokens[b + s];
    }
    sums[warp][lane] = sum;
    counts[warp][lane] = count;
    if (lane == 0) tokens_of[warp] = tokens;
    if (tid == 0) some = 0;
    __syncthreads();
    if (warp == 0) {
        sum = 0.0f;
        count = tokens = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            sum += sums[w][lane];
            count += counts[w][lane];
            tokens += tokens_of[w];
        }
        if (e < p.experts) p.counts[(long long)s * p.experts + e] = count;
        double dot = (double)sum * count;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (lane == 0) {
            p.seq_dots[(long long)s * parts + blockIdx.x] = dot;
            if (blockIdx.x == 0) p.seq_tokens[s] = tokens;
            __threadfence();
            last = atomicAdd(p.ticket, 1) == p.sequences * parts - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    int mine = 0;
    for (int i = tid; i < p.sequences; i += kThreads) mine += __ldcg(p.seq_tokens + i) > 0;
    if (mine) atomicAdd(&some, mine);
    __syncthreads();
    double loss = 0.0;
    for (int i = tid; i < p.sequences; i += kThreads) {
        const float weight = weight_of(p, __ldcg(p.seq_tokens + i), some);
        p.weight[i] = weight;
        double dot = 0.0;
        for (int j = 0; j < parts; ++j) dot += __ldcg(p.seq_dots + (long long)i * parts + j);
        loss += dot * weight;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
    if (lane == 0) warp_dots[warp] = loss;
    __syncthreads();
    if (tid == 0) {
        loss = 0.0;
        for (int w = 0; w < kWarps; ++w) loss += warp_dots[w];
        *p.loss = (float)loss;
    }
}

template <typename T, bool SIGMOID, int PER, int V>
__global__ void __launch_bounds__(kThreads) balance_grad_kernel(const BalanceParams p)
{
    const int lane = threadIdx.x & 31, row0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * p.chunk, row1 = min(row0 + p.chunk, p.rows);
    if (row0 >= row1) return;
    const float grad_loss = p.grad_loss ? *p.grad_loss : 1.0f;
    int s = seq_of(p, row0), known = -1;
    float load[PER], factor = 0.0f;
    for (int row = row0; row < row1; ++row) {
        while (s < p.sequences && seq_end(p, s) <= row) ++s;
        const bool token = s < p.sequences && row >= seq_begin(p, s) && !(p.mask && p.mask[row] == 0);
        float l[PER] = {};
        if (token) {
            if (known != s) {
                // Counts less a whole number near their mean: the difference from the row's mean of them, which is what the gradient is made
                // of, does not lose its places to what they all have in common.
                known = s;
                const long long *counts = p.counts + (long long)s * p.experts;
                float total = 0.0f;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int e = expert_of<V>(i, lane);
                    if (e < p.experts) total += (float)counts[e];
                }
                const long long base = (long long)(warp_sum(total) / (float)p.experts);
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int e = expert_of<V>(i, lane);
                    load[i] = e < p.experts ? (float)(counts[e] - base) : 0.0f;
                }
                factor = __fmul_rn(p.weight[s], grad_loss);
            }
            float rest[PER];
            load_row<T, PER, V>(static_cast<const T *>(p.logits) + row * p.ld, p.experts, lane, l);
            scores<SIGMOID, PER>(l, rest);
            float mean = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) mean = __fmaf_rn(l[i], load[i], mean);
            mean = warp_sum(mean);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                l[i] = __fmul_rn(__fmul_rn(l[i], load[i] - mean), factor);
                if (SIGMOID) l[i] = __fmul_rn(l[i], rest[i]);
            }
        }
        T *to = static_cast<T *>(p.grad) + row * p.ld_grad;
#pragma unroll
        for (int i = 0; i < PER; i += V) {
            const int e = expert_of<V>(i, lane);
            if (e >= p.experts) continue;
            if constexpr (V > 1) {
                uint4 u;
                T *t = reinterpret_cast<T *>(&u);
#pragma unroll
                for (int j = 0; j < V; ++j) t[j] = from_float<T>(l[i + j]);
                *reinterpret_cast<uint4 *>(to + e) = u;
            } else {
                to[e] = from_float<T>(l[i]);
            }
        }
    }
}

constexpr int kAllRows = 64;    // most rows that one block takes by itself

int chunk_of(int64_t rows)      // rows of a block: two blocks an SM, at least one row a warp
{
    const int64_t each = (rows + 2 * 148 - 1) / (2 * 148);
    return (int)((each + kWarps - 1) / kWarps * kWarps);
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// fn(kernel traits) for the type, the scoring and the way that rows are loaded.
template <int N> struct Int { static constexpr int value = N; };
template <bool B> struct Flag { static constexpr bool value = B; };
template <typename T> struct Type { typedef T type; };

template <typename T, bool SIGMOID, typename Fn>
cudaError_t dispatch_width(int experts, bool packs, Fn fn)
{
    constexpr int V = 16 / (int)sizeof(T);
    if (packs) {
        if (experts <= 32 * V) return fn(Type<T>(), Flag<SIGMOID>(), Int<V>(), Int<V>());
        if (experts <= 64 * V) return fn(Type<T>(), Flag<SIGMOID>(), Int<2 * V>(), Int<V>());
        if (experts <= 512) return fn(Type<T>(), Flag<SIGMOID>(), Int<16>(), Int<V>());
        return fn(Type<T>(), Flag<SIGMOID>(), Int<32>(), Int<V>());
    }
    if (experts <= 64) return fn(Type<T>(), Flag<SIGMOID>(), Int<2>(), Int<1>());
    if (experts <= 160) return fn(Type<T>(), Flag<SIGMOID>(), Int<5>(), Int<1>());
    if (experts <= 256) return fn(Type<T>(), Flag<SIGMOID>(), Int<8>(), Int<1>());
    return fn(Type<T>(), Flag<SIGMOID>(), Int<32>(), Int<1>());
}
template <typename Fn>
cudaError_t dispatch(const BalanceProblem &b, bool packs, Fn fn)
{
    const bool sigmoid = b.scoring == kScoreSigmoid;
    switch (b.dtype) {
        case kF32: return sigmoid ? dispatch_width<float, true>(b.experts, packs, fn) : dispatch_width<float, false>(b.experts, packs, fn);
        case kF16: return sigmoid ? dispatch_width<__half, true>(b.experts, packs, fn) : dispatch_width<__half, false>(b.experts, packs, fn);
        case kBF16: return sigmoid ? dispatch_width<__nv_bfloat16, true>(b.experts, packs, fn) : dispatch_width<__nv_bfloat16, false>(b.experts, packs, fn);
        default: return cudaErrorInvalidValue;
    }
}

bool in_packs(const void *p, int64_t ld, const BalanceProblem &b)
{
    const int bytes = b.dtype == kF32 ? 4 : 2;
    return !((uintptr_t)p & 15) && ld * bytes % 16 == 0 && b.experts * bytes % 16 == 0;
}

BalanceParams params_of(const BalanceProblem &b)
{
    BalanceParams p = {};
    p.logits = b.logits; p.ld = b.ld; p.mask = b.token_mask; p.cu = b.cu_seqlens;
    p.ids = b.ids; p.ids_i64 = b.ids_i64; p.top_k = b.top_k; p.rows = (int)b.rows; p.experts = b.experts; p.sequences = (int)b.sequences;
    p.coefficient = b.coefficient;
    p.loss = b.loss; p.weight = b.weight; p.counts = reinterpret_cast<long long *>(b.counts);
    p.grad_loss = b.grad_loss; p.grad = b.grad; p.ld_grad = b.ld_grad;
    return p;
}

struct Layout {
    size_t tokens, counts, sums, seq_tokens, seq_dots, bytes;
    int chunk, blocks;
    explicit Layout(const BalanceProblem &b)
    {
        chunk = b.rows > 0 ? chunk_of(b.rows) : kWarps;
        blocks = (int)((b.rows + chunk - 1) / chunk);
        const size_t pieces = (size_t)blocks + (size_t)b.sequences, parts = ((size_t)b.experts + 31) / 32;
        tokens = 256;
        counts = tokens + align256(pieces * 4);
        sums = counts + align256(pieces * b.experts * 4);
        seq_tokens = sums + align256(pieces * b.experts * 4);
        seq_dots = seq_tokens + align256((size_t)b.sequences * 4);
        bytes = seq_dots + align256((size_t)b.sequences * parts * 8);
    }
};

bool one_block(const BalanceProblem &b) { return !b.cu_seqlens && b.rows <= kAllRows; }

}  // namespace

size_t balance_workspace_bytes(const BalanceProblem &b) { return one_block(b) ? 0 : Layout(b).bytes; }

cudaError_t balance_launch(const BalanceProblem &b, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    BalanceParams p = params_of(b);
    const bool all = one_block(b);
    const int smem = (kWarps + 1) * b.experts * 4;
    int blocks = 1;
    if (all) {
        p.chunk = kAllRows;
    } else {
        const Layout at(b);
        if (!workspace || workspace_bytes < at.bytes) return cudaErrorInvalidValue;
        char *ws = static_cast<char *>(workspace);
        p.chunk = at.chunk; p.blocks = at.blocks;
        p.ticket = reinterpret_cast<int *>(ws);
        p.piece_tokens = reinterpret_cast<int *>(ws + at.tokens);
        p.piece_counts = reinterpret_cast<int *>(ws + at.counts);
        p.piece_sums = reinterpret_cast<float *>(ws + at.sums);
        p.seq_tokens = reinterpret_cast<int *>(ws + at.seq_tokens);
        p.seq_dots = reinterpret_cast<double *>(ws + at.seq_dots);
        blocks = at.blocks > 0 ? at.blocks : 1;   // no rows: the ticket is cleared all the same
    }
    cudaError_t e = dispatch(b, in_packs(b.logits, b.ld, b), [&](auto type, auto sigmoid, auto per, auto v) {
        typedef typename decltype(type)::type T;
        const auto kernel = all ? balance_rows_kernel<T, decltype(sigmoid)::value, decltype(per)::value, decltype(v)::value, true>
                                : balance_rows_kernel<T, decltype(sigmoid)::value, decltype(per)::value, decltype(v)::value, false>;
        kernel<<<blocks, kThreads, smem, stream>>>(p);
        return cudaGetLastError();
    });
    if (e != cudaSuccess || all) return e;
    balance_finish_kernel<<<dim3((unsigned)(b.experts + 31) / 32, (unsigned)b.sequences), kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

cudaError_t balance_grad_launch(const BalanceProblem &b, cudaStream_t stream)
{
    if (b.rows <= 0) return cudaSuccess;
    BalanceParams p = params_of(b);
    // rows of a warp: four blocks an SM
    const int64_t warps = 4 * 148 * kWarps;
    p.chunk = (int)((b.rows + warps - 1) / warps);
    const int64_t blocks = (b.rows + (int64_t)p.chunk * kWarps - 1) / ((int64_t)p.chunk * kWarps);
    return dispatch(b, in_packs(b.logits, b.ld, b) && in_packs(b.grad, b.ld_grad, b), [&](auto type, auto sigmoid, auto per, auto v) {
        typedef typename decltype(type)::type T;
        balance_grad_kernel<T, decltype(sigmoid)::value, decltype(per)::value, decltype(v)::value><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
        return cudaGetLastError();
    });
}

}  // namespace gmm
