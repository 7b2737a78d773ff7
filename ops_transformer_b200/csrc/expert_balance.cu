// expert_balance: how a router's choices load the experts, the loss that evens them out, and its gradient.
//
//   p = softmax(l), or sigmoid(l) / sum of the row's;  per sequence of T tokens: counts c[e], P[e] = sum of p[e] over its tokens
//   loss = sum over the sequences of weight * sum_e c[e] P[e],  weight = coefficient * experts / (top_k * T^2 * sequences with a token)
//   d loss / d l[e] = weight * p[e] * (c[e] - sum_j p[j] c[j])   (sigmoid: times 1 - sigmoid(l[e]))
//
// The loss needs the counts of all tokens, so its gradient reads the logits a second time and forms p anew: 1 KB a row from memory against
// the same to write p and read it back.  A group of 8, 16 or 32 lanes holds a row, a lane 16 of its experts or so: fewer lanes make fewer
// steps of sums and maxima across them, and of all that a row costs once.  Sums over tokens are made in a fixed order (a lane's rows one
// after the other, then the groups, then the pieces), so that a call gives the same bits every time.
//
// Measured, us (forward, gradient): 16 x 64 bf16 2.2, 2.0; 256 x 256 bf16 4.0, 2.3; 4096 x 256 bf16 7.3, 3.8; 4096 x 1024 bf16 13.3, 8.7; 16384 x 256 fp32 in 16
// sequences 12.7, 9.1; 65536 x 256 bf16 17.5, 17.7 (2 TB/s and 3.8).  Loads' latency bounds the large ones: with no scores and no ids to work
// on 65536 rows take 12.0, each of the two adds about 4.6, and half the instructions (16 lanes a row for 32) changed nothing.  Rows on their
// way are held in registers, of which one or two rows a group are all that there is room for; by way of shared memory was not tried.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "dependent.h"
#include "gmm_common.h"
#include "norm_common.h"

namespace gmm {
namespace {

constexpr int kMostCtas = 8;    // of a cluster that takes all rows
constexpr int kGradThreads = 256, kGradWarps = kGradThreads / 32;
// Lanes of a row and values of a lane by the number of experts, and the threads of a block of rows, at most: as many as there are registers
// for.
constexpr int lanes_of(int experts) { return experts <= 128 ? 8 : experts <= 256 ? 16 : 32; }
constexpr int values_of(int experts) { return experts <= 64 ? 8 : experts <= 512 ? 16 : 32; }
constexpr int threads_of(int values) { return values <= 8 ? 1024 : values <= 16 ? 512 : 256; }
inline int warps_of(int experts) { return threads_of(values_of(experts)) / 32; }

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
    // workspace of the loss: what a block of rows adds to a sequence is the piece `block + sequence`, which is another one for every block
    // and sequence that meet, since both only grow on the way through the rows
    int chunk, blocks;                  // rows of a block, blocks
    int *ticket;
    int *piece_tokens;                  // [blocks + sequences]
    int *piece_counts;                  // [blocks + sequences, experts]
    float *piece_sums;                  // the same
    int *seq_tokens;                    // [sequences]
    double *seq_dots;                   // the same
};

constexpr float kInf = __builtin_huge_valf();

__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^v and 1 / v to 2 units in the last place; what is below the normal numbers is 0.
__device__ __forceinline__ float exp2_of(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp_of(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// Over groups of G lanes; the maximum passes NaN over.
template <int G>
__device__ __forceinline__ float group_max(float v)
{
    if constexpr (G == 32) {
        asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v));
    } else {
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v)
{
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Rows whose loads a warp has under way: at most four, and no more than there are registers for.
template <typename T, int PER, int V> __host__ __device__ constexpr int rows_ahead(int registers)
{
    const int n = registers * 4 / (PER * (V > 1 ? (int)sizeof(T) : 4));
    return n > 4 ? 4 : n < 1 ? 1 : n;
}

// The expert of the i-th value of a group's lane: V neighbours at a time.
template <int G, int V>
__device__ __forceinline__ int expert_of(int i, int lane) { return (i / V * G + lane) * V + i % V; }

// A row as it is in memory, for the loads of the next one to be under way while this one is worked on; minus infinity where there is no
// expert.  V: values of one 16-byte load, or 1.
template <typename T, int G, int PER, int V>
struct RawRow {
    static constexpr int N = PER / V;
    typename std::conditional<(V > 1), uint4, T>::type raw[N];
    __device__ __forceinline__ RawRow()
    {
        constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (V > 1) raw[i] = make_uint4(none, none, none, none);
            else raw[i] = from_float<T>(-kInf);
        }
    }
    __device__ __forceinline__ void load(const T *row, int experts, int lane)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = expert_of<G, V>(i * V, lane);
            if (e >= experts) continue;
            if constexpr (V > 1) raw[i] = *reinterpret_cast<const uint4 *>(row + e);
            else raw[i] = row[e];
        }
    }
    // Zeros where there is no token, so that nothing in its place is worked on.
    __device__ __forceinline__ void values(bool token, f32x2 (&l)[PER / 2]) const
    {
        if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                uint4 u = raw[i];
                if (!token) u = make_uint4(0, 0, 0, 0);
                unpack<T>(u, l + i * (V / 2));
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; i += 2) l[i / 2] = token ? pair2(to_float<T>(raw[i]), to_float<T>(raw[i + 1])) : 0;
        }
    }
};

// e, of which p = e * inv, of a row's logits, and for the sigmoid's gradient rest = 1 - sigmoid.  An expert whose logit is NaN or minus
// infinity is not there; a row without one is all zeros.
//
// The plain way takes the exponential's argument from one fma (off by a unit of its size, as the difference itself would be; an error that
// the whole row has in common goes out with inv) and passes every infinity through to the right result.  What it cannot do shows in its
// total, and is done again element by element: a logit of NaN, a row whose largest logit is so far out that the fma's constant term is
// off by more than a little, or one whose sigmoids all but vanish, of which p is what softmax makes of it (to 2^-60).  Below sigmoids of
// e^-700, which 64 bits hardly hold, there is nothing.
template <bool SIGMOID, int G, int PER>
__device__ __forceinline__ void scores(const f32x2 (&l)[PER / 2], f32x2 (&e)[PER / 2], f32x2 (&rest)[PER / 2], float &inv)
{
    constexpr float kLog2e = 1.4426950408889634f;
    float top = -kInf;
    f32x2 total2 = 0;
    if constexpr (SIGMOID) {
        const f32x2 scale = pair2(-kLog2e, -kLog2e), one = pair2(1.0f, 1.0f);
#pragma unroll
        for (int i = 0; i < PER / 2; ++i) {
            const float2 x = unpair2(mul2(l[i], scale));
            const f32x2 t = pair2(exp2_of(x.x), exp2_of(x.y));
            const float2 v = unpair2(add2(t, one));
            e[i] = pair2(rcp_of(v.x), rcp_of(v.y));
            const float2 r = unpair2(mul2(t, e[i]));
            rest[i] = pair2(fminf(r.x, 1.0f), fminf(r.y, 1.0f));    // of infinity times 0, too
            total2 = add2(total2, e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER / 2; ++i) {
            const float2 v = unpair2(l[i]);
            top = fmaxf(top, fmaxf(v.x, v.y));
        }
        top = group_max<G>(top);
        const float shift = __fmul_rn(top, -kLog2e);
#pragma unroll
        for (int i = 0; i < PER / 2; ++i) {
            const float2 x = unpair2(fma2(l[i], pair2(kLog2e, kLog2e), pair2(shift, shift)));
            e[i] = pair2(exp2_of(x.x), exp2_of(x.y));
            total2 = add2(total2, e[i]);
        }
    }
    const float2 parts = unpair2(total2);
    float total = group_sum<G>(parts.x + parts.y);
    const bool again = !(total >= 1e-20f) || (!SIGMOID && !(fabsf(top) <= 0x1p20f));
    if (__any_sync(0xffffffffu, again)) {
#pragma unroll
        for (int i = 0; i < PER / 2; ++i) {
            const float2 v = unpair2(l[i]);
            top = fmaxf(top, fmaxf(v.x, v.y));
        }
        top = group_max<G>(top);
        const bool soft = !SIGMOID || (top < -60.0f && top > -700.0f);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER / 2; ++i) {
            const float2 v = unpair2(l[i]);
            float of[2] = {v.x, v.y}, r[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float x = of[j];
                if (soft) {
                    of[j] = x == top ? 1.0f : expf(x - top);
                    r[j] = 1.0f;
                } else {
                    const float t = expf(-fabsf(x)), big = __fdividef(1.0f, 1.0f + t), small = __fmul_rn(t, big);   // of |x| and -|x|
                    of[j] = x >= 0.0f ? big : small;
                    r[j] = x >= 0.0f ? small : big;
                }
                if (!(x > -kInf)) of[j] = r[j] = 0.0f;
                sum += of[j];
            }
            if (again) {
                e[i] = pair2(of[0], of[1]);
                rest[i] = pair2(r[0], r[1]);
            }
        }
        sum = group_sum<G>(sum);
        if (again) total = sum;
    }
    inv = total > 0.0f ? rcp_of(total) : 0.0f;
}

// Rows of sequence s, cut to those that there are.
__device__ __forceinline__ int seq_begin(const BalanceParams &p, int s) { return p.cu ? min(max(p.cu[s], 0), p.rows) : 0; }
__device__ __forceinline__ int seq_end(const BalanceParams &p, int s) { return p.cu ? min(max(p.cu[s + 1], 0), p.rows) : p.rows; }
// The first sequence that ends behind `row`; by a warp, 32 ends at a time.
__device__ __forceinline__ int seq_of(const BalanceParams &p, int row, int lane)
{
    if (!p.cu) return row < p.rows ? 0 : 1;
    int lo = 0, hi = p.sequences;
    while (lo < hi) {
        const int width = (int)(((long long)hi - lo + 31) / 32);
        const long long probe = lo + (lane + 1ll) * width - 1;
        const int before = __popc(__ballot_sync(0xffffffffu, probe < hi && seq_end(p, (int)probe) <= row));
        lo = min(lo + before * width, hi);
        hi = min(hi, lo + width - 1);
    }
    return lo;
}

__device__ __forceinline__ float weight_of(const BalanceParams &p, int tokens, int sequences)
{
    return tokens > 0 ? (float)((double)p.coefficient * p.experts / ((double)p.top_k * tokens * tokens * sequences)) : 0.0f;
}

// The sequence and the block of rows that a piece belongs to: the sequence is the first whose last piece is not before it.
__device__ __forceinline__ int seq_of_piece(const BalanceParams &p, int piece, int lane)
{
    if (!p.cu) return piece < p.blocks ? 0 : 1;
    int lo = 0, hi = p.sequences;
    while (lo < hi) {
        const int width = (hi - lo + 31) / 32, probe = lo + (lane + 1) * width - 1;
        const bool before = probe < hi && probe + max(seq_end(p, probe) - 1, 0) / p.chunk < piece;
        lo = min(lo + __popc(__ballot_sync(0xffffffffu, before)) * width, hi);
        hi = min(hi, lo + width - 1);
    }
    return lo;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync()
{
    __syncwarp();           // a warp's lanes come from branches of their own
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ uint32_t in_first_cta(const void *p)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)));
    return r;
}

// What a block of rows adds to a sequence: one piece, which a CTA makes.  A warp takes a row for each of its groups of G lanes at a time, and
// has the loads of R times as many under way.  ALL: the CTAs, one or a cluster, hold all rows of the only sequence; the first one adds up what
// the others put into its shared memory, and finishes.
template <typename T, bool SIGMOID, int G, int PER, int V, bool ALL>
__global__ void __launch_bounds__(threads_of(PER), 1) balance_rows_kernel(const BalanceParams p)
{
    constexpr int R = rows_ahead<T, PER, V>(PER <= 8 ? 8 : 16), GROUPS = 32 / G;
    extern __shared__ float4 smem[];    // sums [warps][GROUPS][experts], then the counts [experts]
    __shared__ int warp_tokens[32], cta_tokens[kMostCtas];
    __shared__ double warp_dots[32];
    float *sums = reinterpret_cast<float *>(smem);
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5, piece = blockIdx.x;
    const int group = lane / G, mine = lane % G, step = warps * GROUPS;
    int *counts = reinterpret_cast<int *>(sums + step * p.experts);
    for (int e = tid; e < p.experts; e += threads) counts[e] = 0;
    dependent_wait();
    dependent_release();
    if (!ALL && piece == 0 && tid == 0) *p.ticket = 0;
    const int s = ALL ? 0 : seq_of_piece(p, piece, lane);
    if (s >= p.sequences) return;
    const int begin = ALL ? piece * p.chunk : max(seq_begin(p, s), (piece - s) * p.chunk);
    const int end = min(ALL ? p.rows : seq_end(p, s), (piece - s + 1) * p.chunk);
    if (!ALL && begin >= end) return;
    f32x2 sum[PER / 2] = {};
    int tokens = 0;
    RawRow<T, G, PER, V> rows[R];
    int2 ids[R];    // as they are in memory, and the mask too: a look at one would hold up the loads behind it
    int8_t mask[R];
    const auto load_id = [&](int row, int j) {
        const long long i = (long long)row * p.top_k + j;
        return p.ids_i64 ? static_cast<const int2 *>(p.ids)[i] : make_int2(static_cast<const int *>(p.ids)[i], 0);
    };
    const auto count_id = [&](const int2 &v) {
        if ((unsigned)v.x < (unsigned)p.experts && v.y == 0) atomicAdd(counts + v.x, 1);
    };
    const auto fetch = [&](int r, int row) {    // of a row that the mask leaves out, too, so that no load waits for another
        mask[r] = 0;
        if (row >= end) return;
        rows[r].load(static_cast<const T *>(p.logits) + row * p.ld, p.experts, mine);
        if (mine < p.top_k) ids[r] = load_id(row, mine);
        mask[r] = 1;
        if (p.mask) mask[r] = p.mask[row];
    };
#pragma unroll
    for (int r = 0; r < R; ++r) fetch(r, begin + warp * GROUPS + group + r * step);
    __syncthreads();    // the counts are zero
    for (int row0 = begin + warp * GROUPS; row0 < end; row0 += R * step) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = row0 + group + r * step;
            const bool token = mask[r] != 0;
            f32x2 l[PER / 2], e[PER / 2], rest[PER / 2];
            rows[r].values(token, l);
            if (token) {
                tokens += mine == 0;
                if (mine < p.top_k) count_id(ids[r]);
                for (int j = mine + G; j < p.top_k; j += G) count_id(load_id(row, j));
            }
            fetch(r, row + R * step);
            if (!__any_sync(0xffffffffu, token)) continue;
            float inv;
            scores<SIGMOID, G, PER>(l, e, rest, inv);
            if (!token) inv = 0.0f;
#pragma unroll
            for (int i = 0; i < PER / 2; ++i) sum[i] = fma2(e[i], pair2(inv, inv), sum[i]);
        }
    }
    tokens = (int)__reduce_add_sync(0xffffffffu, tokens);
    if (lane == 0) warp_tokens[warp] = tokens;
    float *to = sums + (warp * GROUPS + group) * p.experts;
    if constexpr (V > 1) {
#pragma unroll
        for (int i = 0; i < PER; i += 4) {
            const int e = expert_of<G, V>(i, mine);
            if (e < p.experts) *reinterpret_cast<float4 *>(to + e) = make_float4(element(sum, i), element(sum, i + 1), element(sum, i + 2), element(sum, i + 3));
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = expert_of<G, V>(i, mine);
            if (e < p.experts) to[e] = element(sum, i);
        }
    }
    __syncthreads();
    const auto total_of = [&](int e) {
        float total = 0.0f;
#pragma unroll 8
        for (int w = 0; w < step; ++w) total += sums[w * p.experts + e];
        return total;
    };
    tokens = (int)__reduce_add_sync(0xffffffffu, lane < warps ? warp_tokens[lane] : 0);
    if constexpr (!ALL) {
        for (int e = tid; e < p.experts; e += threads) {
            p.piece_sums[(long long)piece * p.experts + e] = total_of(e);
            p.piece_counts[(long long)piece * p.experts + e] = counts[e];
        }
        if (tid == 0) p.piece_tokens[piece] = tokens;
        return;
    }
    const int ctas = gridDim.x;
    double dot = 0.0;
    if (ctas == 1) {
        for (int e = tid; e < p.experts; e += threads) {
            p.counts[e] = counts[e];
            dot += (double)total_of(e) * counts[e];
        }
    } else {
        constexpr int N = PER / 8;      // experts of a thread, of as many threads as there can be
        float total[N];
#pragma unroll
        for (int i = 0; i < N; ++i) total[i] = tid + i * threads < p.experts ? total_of(tid + i * threads) : 0.0f;
        cluster_sync();     // the first CTA has done with its sums, whose place the parts take
        const uint32_t parts = in_first_cta(sums);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = tid + i * threads;
            if (e < p.experts)
                asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(parts + (uint32_t)(piece * p.experts + e) * 8), "r"(__float_as_uint(total[i])), "r"(counts[e]) : "memory");
        }
        if (tid == 0) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(in_first_cta(cta_tokens + piece)), "r"(tokens) : "memory");
        cluster_sync();
        if (piece != 0) return;
        const uint2 *here = reinterpret_cast<const uint2 *>(sums);
        for (int e = tid; e < p.experts; e += threads) {
            float sum = 0.0f;
            int count = 0;
#pragma unroll 8
            for (int c = 0; c < ctas; ++c) {
                const uint2 v = here[c * p.experts + e];
                sum += __uint_as_float(v.x);
                count += (int)v.y;
            }
            p.counts[e] = count;
            dot += (double)sum * count;
        }
        tokens = (int)__reduce_add_sync(0xffffffffu, lane < ctas ? cta_tokens[lane] : 0);
    }
    dot = warp_sum(dot);
    if (lane == 0) warp_dots[warp] = dot;
    __syncthreads();
    if (warp != 0) return;
    dot = warp_sum(lane < warps ? warp_dots[lane] : 0.0);
    const float weight = weight_of(p, tokens, 1);
    if (lane == 0) p.weight[0] = weight;
    if (lane == 0) *p.loss = (float)(dot * weight);
}

// The sums of a warp's share of a sequence's pieces, for the expert of each lane; N of them under way.
template <int N>
__device__ __forceinline__ void sum_pieces(const BalanceParams &p, int s, int first, int step, int e, float &sum, long long &count, int &tokens)
{
    const int begin = seq_begin(p, s), end = seq_end(p, s);
    if (begin >= end) return;
    const int behind = (end - 1) / p.chunk + 1;
    for (int b = begin / p.chunk + first; b < behind; b += N * step) {
        float some_sum[N];
        int some_count[N], some_tokens[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const long long piece = b + i * step + s;
            const bool there = b + i * step < behind;
            some_sum[i] = there && e < p.experts ? p.piece_sums[piece * p.experts + e] : 0.0f;
            some_count[i] = there && e < p.experts ? p.piece_counts[piece * p.experts + e] : 0;
            some_tokens[i] = there ? p.piece_tokens[piece] : 0;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sum += some_sum[i];
            count += some_count[i];
            tokens += some_tokens[i];
        }
    }
}

// Few sequences: one cluster adds up their pieces, a CTA an eighth of the experts, and its first CTA makes the loss of what they put into
// its shared memory.  (Through memory and a ticket, as below, that last step costs 2.7 us instead of a half.)
constexpr int kFewSequences = 32, kFinishCtas = 8, kMostGroups = 1024 / (32 * kFinishCtas);
__global__ void __launch_bounds__(1024, 1) balance_finish_few_kernel(const BalanceParams p)
{
    __shared__ float sums[32][32];
    __shared__ long long counts[32][32];
    __shared__ int tokens_of[kFewSequences];
    __shared__ double dots[kFewSequences * kMostGroups], all_dots[kFinishCtas][kFewSequences];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x;
    // A CTA's items are a sequence and 32 experts each, for a power of two of warps.
    const int groups = (p.experts + 32 * kFinishCtas - 1) / (32 * kFinishCtas), items = p.sequences * groups;
    int each = 1;
    while (each * 2 * items <= 32) each *= 2;
    const int part = warp & (each - 1);
    cluster_arrive();       // this CTA is there, and can be sent to
    if (tid < kFewSequences) tokens_of[tid] = 0;
    dependent_wait();
    dependent_release();
    for (int item0 = 0; item0 < items; item0 += 32 / each) {
        const int item = item0 + warp / each, s = item / groups, g = item - s * groups, e = (rank * groups + g) * 32 + lane;
        float sum = 0.0f;
        long long count = 0;
        int tokens = 0;
        if (item < items) sum_pieces<5>(p, s, part, each, e, sum, count, tokens);
        sums[warp][lane] = sum;
        counts[warp][lane] = count;
        __syncthreads();
        if (item < items && g == 0 && lane == 0) atomicAdd(tokens_of + s, tokens);
        if (item < items && part == 0) {
            sum = 0.0f;
            count = 0;
#pragma unroll 8
            for (int w = warp; w < warp + each; ++w) {
                sum += sums[w][lane];
                count += counts[w][lane];
            }
            if (e < p.experts) p.counts[(long long)s * p.experts + e] = count;
            const double dot = warp_sum((double)sum * count);
            if (lane == 0) dots[item] = dot;
        }
        __syncthreads();
    }
    cluster_wait();         // until the first CTA is there
    if (tid < p.sequences) {
        double dot = 0.0;
        for (int g = 0; g < groups; ++g) dot += dots[tid * groups + g];
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(in_first_cta(&all_dots[rank][tid])), "d"(dot) : "memory");
    }
    cluster_sync();
    if (rank != 0 || warp != 0) return;
    const int mine = lane < p.sequences ? tokens_of[lane] : 0;
    const float weight = weight_of(p, mine, __popc(__ballot_sync(0xffffffffu, mine > 0)));
    double loss = 0.0;
    if (lane < p.sequences) {
        p.weight[lane] = weight;
#pragma unroll
        for (int r = 0; r < kFinishCtas; ++r) loss += all_dots[r][lane];
    }
    loss = warp_sum(loss * weight);
    if (lane == 0) *p.loss = (float)loss;
}

// Any number of sequences: a CTA adds up the pieces of one, which are few where sequences are many; the one that comes last makes the loss
// of all.
constexpr int kFinishThreads = 256;
__global__ void __launch_bounds__(kFinishThreads) balance_finish_many_kernel(const BalanceParams p)
{
    __shared__ double warp_dots[kFinishThreads / 32];
    __shared__ int last, some;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.x;
    dependent_wait();
    dependent_release();
    int tokens = 0;
    double dot = 0.0;
    for (int e = tid; e < p.experts; e += kFinishThreads) {
        float sum = 0.0f;
        long long count = 0;
        tokens = 0;
        sum_pieces<4>(p, s, 0, 1, e, sum, count, tokens);
        p.counts[(long long)s * p.experts + e] = count;
        dot += (double)sum * count;
    }
    dot = warp_sum(dot);
    if (lane == 0) warp_dots[warp] = dot;
    __syncthreads();
    if (warp == 0) {
        dot = warp_sum(lane < kFinishThreads / 32 ? warp_dots[lane] : 0.0);
        if (lane == 0) {
            p.seq_dots[s] = dot;
            p.seq_tokens[s] = tokens;
            some = 0;
            __threadfence();
            last = atomicAdd(p.ticket, 1) == p.sequences - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double loss = 0.0;
    int mine = 0;
    for (int i = tid; i < p.sequences; i += kFinishThreads) mine += __ldcg(p.seq_tokens + i) > 0;
    if (mine) atomicAdd(&some, mine);
    __syncthreads();
    for (int i = tid; i < p.sequences; i += kFinishThreads) {
        const float weight = weight_of(p, __ldcg(p.seq_tokens + i), some);
        p.weight[i] = weight;
        loss += __ldcg(p.seq_dots + i) * weight;
    }
    loss = warp_sum(loss);
    if (lane == 0) warp_dots[warp] = loss;
    __syncthreads();
    if (warp == 0) {
        loss = warp_sum(lane < kFinishThreads / 32 ? warp_dots[lane] : 0.0);
        if (lane == 0) *p.loss = (float)loss;
    }
}

// A warp holds a row: its loads are the longest part of it, and more warps hide more of them than a row's fewer instructions in fewer lanes
// would gain (4096 x 256 4.0 us, with 16 lanes a row 4.1; 16384 x 256 in fp32 9.2 and 10.4).  Above 512 experts a lane's 32 values do not fit
// its 128 registers, and 0.1 to 0.6 KB a thread go through local memory: 4096 x 512 in bf16 5.0, x 1024 8.7, x 513, on no pack, 9.7.
template <typename T, bool SIGMOID, int PER, int V>
__global__ void __launch_bounds__(kGradThreads, PER <= 8 ? 4 : 2) balance_grad_kernel(const BalanceParams p)
{
    const int lane = threadIdx.x & 31, row0 = (blockIdx.x * kGradWarps + (threadIdx.x >> 5)) * p.chunk, row1 = min(row0 + p.chunk, p.rows);
    dependent_wait();
    dependent_release();
    if (row0 >= row1) return;
    RawRow<T, 32, PER, V> here;
    int8_t mask = 1;
    const auto fetch = [&](int row) {
        here.load(static_cast<const T *>(p.logits) + row * p.ld, p.experts, lane);
        if (p.mask) mask = p.mask[row];
    };
    fetch(row0);
    const float grad_loss = p.grad_loss ? *p.grad_loss : 1.0f;
    int s = seq_of(p, row0, lane), known = -1, begin = 0, end = 0;
    f32x2 load[PER / 2];
    float factor = 0.0f;
    for (int row = row0; row < row1; ++row) {
        while (row >= end && s < p.sequences) {
            begin = seq_begin(p, s);
            end = seq_end(p, s);
            if (row >= end) ++s;
        }
        const bool token = row >= begin && row < end && mask != 0;
        f32x2 l[PER / 2], g[PER / 2] = {};
        here.values(true, l);
        if (row + 1 < row1) fetch(row + 1);
        if (token) {
            if (known != s) {
                // Counts less a whole number near their mean: the difference from the row's mean of them, which is what the gradient is made
                // of, does not lose its places to what they all have in common.
                known = s;
                const long long *counts = p.counts + (long long)s * p.experts;
                factor = __fmul_rn(p.weight[s], grad_loss);
                long long count[PER];
#pragma unroll
                for (int i = 0; i < PER; i += V > 1 ? 2 : 1) {
                    const int e = expert_of<32, V>(i, lane);
                    if constexpr (V > 1) {
                        const longlong2 two = e < p.experts ? *reinterpret_cast<const longlong2 *>(counts + e) : make_longlong2(0, 0);
                        count[i] = two.x;
                        count[i + 1] = two.y;
                    } else {
                        count[i] = e < p.experts ? counts[e] : 0;
                    }
                }
                float total = 0.0f;
#pragma unroll
                for (int i = 0; i < PER; ++i) total += (float)count[i];
                const long long base = (long long)(group_sum<32>(total) / (float)p.experts);
#pragma unroll
                for (int i = 0; i < PER; i += 2) load[i / 2] = pair2((float)(count[i] - base), (float)(count[i + 1] - base));
            }
            f32x2 e[PER / 2], rest[PER / 2], mean2 = 0;
            float inv;
            scores<SIGMOID, 32, PER>(l, e, rest, inv);
#pragma unroll
            for (int i = 0; i < PER / 2; ++i) mean2 = fma2(e[i], load[i], mean2);
            const float2 parts = unpair2(mean2);
            const float mean = -__fmul_rn(group_sum<32>(parts.x + parts.y), inv), scale = __fmul_rn(inv, factor);
#pragma unroll
            for (int i = 0; i < PER / 2; ++i) {
                g[i] = mul2(mul2(e[i], pair2(scale, scale)), add2(load[i], pair2(mean, mean)));
                if (SIGMOID) g[i] = mul2(g[i], rest[i]);
            }
        }
        T *to = static_cast<T *>(p.grad) + row * p.ld_grad;
#pragma unroll
        for (int i = 0; i < PER; i += V) {
            const int e = expert_of<32, V>(i, lane);
            if (e >= p.experts) continue;
            if constexpr (V > 1) *reinterpret_cast<uint4 *>(to + e) = pack<T>(g + i / 2);
            else to[e] = from_float<T>(element(g, i));
        }
    }
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// fn(kernel traits) for the type, the scoring and the way that rows are loaded.
template <int N> struct Int { static constexpr int value = N; };
template <bool B> struct Flag { static constexpr bool value = B; };
template <typename T> struct Type { typedef T type; };

template <typename T, bool SIGMOID, int V, typename Fn>
cudaError_t dispatch_width(int experts, Fn fn)
{
    if (experts <= 64) return fn(Type<T>(), Flag<SIGMOID>(), Int<lanes_of(64)>(), Int<values_of(64)>(), Int<V>());
    if (experts <= 128) return fn(Type<T>(), Flag<SIGMOID>(), Int<lanes_of(128)>(), Int<values_of(128)>(), Int<V>());
    if (experts <= 256) return fn(Type<T>(), Flag<SIGMOID>(), Int<lanes_of(256)>(), Int<values_of(256)>(), Int<V>());
    if (experts <= 512) return fn(Type<T>(), Flag<SIGMOID>(), Int<lanes_of(512)>(), Int<values_of(512)>(), Int<V>());
    return fn(Type<T>(), Flag<SIGMOID>(), Int<lanes_of(1024)>(), Int<values_of(1024)>(), Int<V>());
}
template <typename T, bool SIGMOID, typename Fn>
cudaError_t dispatch_packs(int experts, bool packs, Fn fn)
{
    return packs ? dispatch_width<T, SIGMOID, 16 / (int)sizeof(T)>(experts, fn) : dispatch_width<T, SIGMOID, 1>(experts, fn);
}
template <typename Fn>
cudaError_t dispatch(const BalanceProblem &b, bool packs, Fn fn)
{
    const bool sigmoid = b.scoring == kScoreSigmoid;
    switch (b.dtype) {
        case kF32: return sigmoid ? dispatch_packs<float, true>(b.experts, packs, fn) : dispatch_packs<float, false>(b.experts, packs, fn);
        case kF16: return sigmoid ? dispatch_packs<__half, true>(b.experts, packs, fn) : dispatch_packs<__half, false>(b.experts, packs, fn);
        case kBF16: return sigmoid ? dispatch_packs<__nv_bfloat16, true>(b.experts, packs, fn) : dispatch_packs<__nv_bfloat16, false>(b.experts, packs, fn);
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
    int chunk, blocks, warps;
    explicit Layout(const BalanceProblem &b)
    {
        // One piece for each CTA that there is room for at once, in smaller CTAs where there are many sequences, each of which has a piece
        // that it shares with none; at least a row for each group of lanes.
        const int most = warps_of(b.experts);
        const auto at_once = [&] { return 148 * (most / warps); };
        for (warps = most; warps > 4 && at_once() < 2 * b.sequences;) warps /= 2;
        const int at_least = warps * (32 / lanes_of(b.experts));
        const int64_t wanted = at_once() >= 2 * b.sequences ? at_once() - b.sequences + 1 : at_once() / 2, each = (b.rows + wanted - 1) / wanted;
        chunk = (int)(each < at_least ? at_least : each);
        blocks = (int)((b.rows + chunk - 1) / chunk);
        const size_t pieces = (size_t)blocks + (size_t)b.sequences;
        tokens = 256;
        counts = tokens + align256(pieces * 4);
        sums = counts + align256(pieces * b.experts * 4);
        seq_tokens = sums + align256(pieces * b.experts * 4);
        seq_dots = seq_tokens + align256((size_t)b.sequences * 4);
        bytes = seq_dots + align256((size_t)b.sequences * 8);
    }
};

// CTAs that take all rows by themselves, one up to 12 K scores and a cluster up to 256 K; 0: more of them, and a second kernel behind them.
// (one CTA / a cluster / two kernels, us, bf16: 48 x 256 3.5, 3.5, 6.4; 128 x 256 5.2, 3.7, 6.4; 1024 x 256 24, 6.4, 6.8; 2048 x 256 46, 9.3, 7.1;
// 128 x 64 3.7, 4.1, 6.8; 4096 x 64 27, 6.8, 7.4; 512 x 512 22, 6.6, 6.9; with four CTAs 16 x 1024 3.9, 4.3, 6.5; 128 x 1024 13, 7.1, 7.1)
int ctas_of_all(const BalanceProblem &b)
{
    const int64_t scores = b.rows * (b.experts < 64 ? 64 : b.experts);
    const int most = b.experts <= 512 ? kMostCtas : kMostCtas / 2;      // whose parts fit where the first one's sums were
    return b.cu_seqlens ? 0 : scores <= 12 * 1024 ? 1 : scores <= 32 * 1024 * most ? most : 0;
}

}  // namespace

size_t balance_workspace_bytes(const BalanceProblem &b) { return ctas_of_all(b) ? 0 : Layout(b).bytes; }

cudaError_t balance_launch(const BalanceProblem &b, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    BalanceParams p = params_of(b);
    const int all = ctas_of_all(b);
    const int groups = 32 / lanes_of(b.experts);
    int blocks = 1, warps = warps_of(b.experts);
    if (all) {
        if (all == 1 && warps * groups > b.rows) warps = b.rows <= 4 * groups ? 4 : (int)(b.rows + groups - 1) / groups;
        blocks = all;
        p.chunk = (int)((b.rows + all - 1) / all);
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
        warps = at.warps;
        blocks = at.blocks + (int)b.sequences - (at.blocks > 0);    // no rows: the ticket is cleared all the same
    }
    cudaError_t e = dispatch(b, in_packs(b.logits, b.ld, b), [&](auto type, auto sigmoid, auto lanes, auto per, auto v) {
        typedef typename decltype(type)::type T;
        const auto kernel = all ? balance_rows_kernel<T, decltype(sigmoid)::value, decltype(lanes)::value, decltype(per)::value, decltype(v)::value, true>
                                : balance_rows_kernel<T, decltype(sigmoid)::value, decltype(lanes)::value, decltype(per)::value, decltype(v)::value, false>;
        return launch_dependent(kernel, dim3(blocks), warps * 32, (size_t)(warps * groups + 1) * b.experts * 4, all > 1 ? all : 1, stream, p);
    });
    if (e != cudaSuccess || all) return e;
    if (b.sequences <= kFewSequences) return launch_dependent(balance_finish_few_kernel, dim3(kFinishCtas), 1024, 0, kFinishCtas, stream, p);
    return launch_dependent(balance_finish_many_kernel, dim3((unsigned)b.sequences), kFinishThreads, 0, 1, stream, p);
}

cudaError_t balance_grad_launch(const BalanceProblem &b, cudaStream_t stream)
{
    if (b.rows <= 0) return cudaSuccess;
    BalanceParams p = params_of(b);
    // rows of a warp: as many blocks as an SM holds
    const int64_t warps = (b.experts <= 256 ? 4 : 2) * 148 * kGradWarps;
    p.chunk = (int)((b.rows + warps - 1) / warps);
    const int64_t blocks = (b.rows + (int64_t)p.chunk * kGradWarps - 1) / ((int64_t)p.chunk * kGradWarps);
    return dispatch(b, in_packs(b.logits, b.ld, b) && in_packs(b.grad, b.ld_grad, b) && !((uintptr_t)b.counts & 15), [&](auto type, auto sigmoid, auto lanes, auto per, auto v) {
        typedef typename decltype(type)::type T;
        constexpr int values = decltype(lanes)::value < 32 ? 8 : decltype(per)::value;   // of a lane where a warp holds a row
        return launch_dependent(balance_grad_kernel<T, decltype(sigmoid)::value, values, decltype(v)::value>, dim3((unsigned)blocks),
                                kGradThreads, 0, 1, stream, p);
    });
}

}  // namespace gmm
