// adapter_add: low-rank adapters of many requests on top of a projection that they share.
//
//   out[t] = base[t] + scaling[i] * (x[t] a[i]^T) b[i]^T,  i = ids[t]
//
// The tokens of one adapter are gathered into tiles, and two kernels run over them:
//   shrink - v[t] = scaling * x[t] a[i]^T in fp32, K split over CTAs, one partial sum each (workspace)
//   expand - out[t] = base[t] + v[t] b[i]^T: the partial sums are added in a fixed order, the result is rounded once
// Both products run on the tensor cores (tcgen05, fp32 accumulators in tensor memory) although few operations come with every byte:
// they then cost no issue slots beside the loads.  The tokens are rows of the first product and columns of the second, so that tiles of
// 16 tokens (few tokens) and of 64 share the code and the channels of a result row lie in neighbouring lanes.
// v enters the second product as two 16-bit parts, v = hi + lo: one alone would add an error of 2^-9 (bf16) of v, as large as the
// rounding of the result.  fp16 has no range to spare, so there every token's v is scaled by a power of two to below 2.
// The operands are fetched with 16-byte asynchronous copies (8, 4 or 2 bytes where rows start on no such boundary), straight into the
// 128-byte-swizzled layout that the tensor cores read; a row's tail is zero filled.
//
// Which tokens share an adapter is found on the device.  Up to kSelfPlan tokens every CTA ranks the tokens among those of their
// adapter itself, beside its first loads; beyond, a one-CTA kernel counts and sorts them.  The order within an adapter does not matter:
// every row's arithmetic is its own.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "gmm_common.h"

namespace gmm {
namespace {

constexpr int kBlockK = 128;         // elements of a row per K block: two swizzled rows of 128 bytes
constexpr int kChunkN = 128;         // channels per step of the second product
constexpr int kSelfPlan = 256;       // most tokens for which every CTA finds its tile itself
constexpr int kPlanThreads = 1024;
constexpr int kShrinkThreads = 256, kExpandThreads = 256;
constexpr int kShrinkStages = 3, kExpandStages = 2;
constexpr long long kWaitLimitCycles = 1ll << 31;   // about a second

struct AdapterParams {
    const void *base, *x, *a, *b;
    const float *x_scale, *scaling;
    const int *ids;
    void *out;
    long long ld_base, ld_x, ld_out;
    int rows, k, n, adapters, rank;
    int rank_pad;                   // rank, rounded up to the tensor cores' K step of 16
    int grain_x, grain_a, grain_b, grain_base, grain_out;   // bytes of a copy
    int ksplit, nsplit;
    int *status;                    // [4]
    int *n_tiles;
    int4 *tiles;                    // adapter (-1: none), first entry in `order`, tokens
    int *order;                     // [rows] tokens grouped by adapter
    float *v;                       // [ksplit, rows, rank_pad]
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait for the tensor cores.  When it runs out the status says so and later waits of the CTA return at once.
__device__ __noinline__ void mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int *gave_up, int *status, int role)
{
    const long long t0 = clock64();
    while (!mbar_try(bar, parity)) {
        if (*gave_up) return;
        if (clock64() - t0 > kWaitLimitCycles) {
            *gave_up = 1;
            if (atomicCAS(status, kStatusOk, kStatusWaitTimeout) == kStatusOk) {
                status[1] = (int)(blockIdx.y * gridDim.x + blockIdx.x);
                status[2] = role;
                status[3] = (int)parity;
            }
            return;
        }
    }
}
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, volatile int *gave_up, int *status, int role)
{
    if (!mbar_try(bar, parity)) mbar_wait_slow(bar, parity, gave_up, status, role);
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t *dst, uint32_t cols)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t cols)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// K-major operand in rows of 128 bytes with the 128-byte swizzle, 8 rows (1024 bytes) a group.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr)
{
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | (uint64_t)2 << 61;
}
// fp32 accumulators, both operands K-major and of type T, M = 128.
template <typename T>
__device__ __forceinline__ uint32_t instr_desc(int n)
{
    constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return 1u << 4 | type << 7 | type << 10 | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, int valid)
{
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(valid), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One copy of GRAIN bytes, of which `valid` are read and the rest is zero.
template <int GRAIN>
__device__ __forceinline__ void copy_grain(uint32_t dst, const char *src, int valid)
{
    if (GRAIN >= 4) {
        cp_async<GRAIN>(dst, src, valid);
    } else if (GRAIN == 2) {
        const uint16_t v = valid > 0 ? *reinterpret_cast<const uint16_t *>(src) : (uint16_t)0;
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst), "h"(v) : "memory");
    } else {
        const uint16_t v = valid > 0 ? *reinterpret_cast<const uint8_t *>(src) : (uint16_t)0;
        asm volatile("st.shared.u8 [%0], %1;" ::"r"(dst), "h"(v) : "memory");
    }
}

// Offset of byte `b` of row `r` in a tile of 128-byte rows with the 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int r, int b) { return (uint32_t)(r * 128 + ((((b >> 4) ^ r) & 7) << 4) + (b & 15)); }

// Rows of `width` bytes (a power of two up to 256) into shared memory, `valid` bytes of each read; row r comes from src(r).
// SWIZZLE: into 128-byte swizzled rows (width <= 128), else rows `width` bytes apart.
template <int GRAIN, bool SWIZZLE, int THREADS, typename Src>
__device__ __forceinline__ void copy_rows_grain(uint32_t dst, int rows, int width, int valid, Src src)
{
    const int shift = 31 - __clz(width / GRAIN);
    for (int i = threadIdx.x; i < rows << shift; i += THREADS) {
        const int r = i >> shift, b = (i & ((1 << shift) - 1)) * GRAIN;
        const int have = min(max(valid - b, 0), GRAIN);
        const char *row = src(r);
        copy_grain<GRAIN>(dst + (SWIZZLE ? swizzled(r, b) : (uint32_t)(r * width + b)), have > 0 ? row + b : row, have);
    }
}
template <bool SWIZZLE, int THREADS, typename Src>
__device__ __forceinline__ void copy_rows(int grain, uint32_t dst, int rows, int width, int valid, Src src)
{
    if (grain == 16) copy_rows_grain<16, SWIZZLE, THREADS>(dst, rows, width, valid, src);
    else if (grain == 8) copy_rows_grain<8, SWIZZLE, THREADS>(dst, rows, width, valid, src);
    else if (grain == 4) copy_rows_grain<4, SWIZZLE, THREADS>(dst, rows, width, valid, src);
    else if (grain == 2) copy_rows_grain<2, SWIZZLE, THREADS>(dst, rows, width, valid, src);
    else copy_rows_grain<1, SWIZZLE, THREADS>(dst, rows, width, valid, src);
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    const T lo = from_float<T>(a), hi = from_float<T>(b);
    return (uint32_t)*reinterpret_cast<const uint16_t *>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t *>(&hi) << 16;
}

// The int8 elements that this thread copied to `raw` (rows of kBlockK), as T in the swizzled tiles, `next` bytes apart: exact in both
// types.
template <typename T, int GRAIN, int THREADS>
__device__ __forceinline__ void widen_rows_grain(uint32_t raw, uint32_t dst, uint32_t next, int rows)
{
    constexpr int PER_ROW = kBlockK / GRAIN;
    for (int i = threadIdx.x; i < rows * PER_ROW; i += THREADS) {
        const int r = i / PER_ROW, c = (i % PER_ROW) * GRAIN;
        if (GRAIN == 1) {
            uint16_t q;
            asm volatile("ld.shared.u8 %0, [%1];" : "=h"(q) : "r"(raw + r * kBlockK + c) : "memory");
            const T f = from_float<T>((float)(int8_t)q);
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + c / 64 * next + swizzled(r, 2 * c % 128)), "h"(*reinterpret_cast<const uint16_t *>(&f)) : "memory");
        } else {
#pragma unroll
            for (int e = 0; e < GRAIN; e += 4) {
                int q;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(q) : "r"(raw + r * kBlockK + c + e) : "memory");
                const uint32_t lo = pack2<T>((float)(int8_t)q, (float)(int8_t)(q >> 8));
                const uint32_t hi = pack2<T>((float)(int8_t)(q >> 16), (float)(q >> 24));
                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst + c / 64 * next + swizzled(r, 2 * (c + e) % 128)), "r"(lo), "r"(hi) : "memory");
            }
        }
    }
}
template <typename T, int THREADS>
__device__ __forceinline__ void widen_rows(int grain, uint32_t raw, uint32_t dst, uint32_t next, int rows)
{
    if (grain == 16) widen_rows_grain<T, 16, THREADS>(raw, dst, next, rows);
    else if (grain == 8) widen_rows_grain<T, 8, THREADS>(raw, dst, next, rows);
    else if (grain == 4) widen_rows_grain<T, 4, THREADS>(raw, dst, next, rows);
    else widen_rows_grain<T, 1, THREADS>(raw, dst, next, rows);
}

// ---------------------------------------------------------------------------------------------------------
// Which tokens make a tile
// ---------------------------------------------------------------------------------------------------------

struct Tile {
    int adapter, count;   // adapter -1: tokens without one; count 0: there is no such tile
};

__device__ __forceinline__ int adapter_of(const AdapterParams &p, int t)
{
    const int i = __ldg(p.ids + t);
    return i >= 0 && i < p.adapters ? i : -1;
}

// Tile number blockIdx.x of at most TN tokens each, found by every CTA for itself; rows[slot] = token.  A token whose rank among the
// tokens of its adapter is a multiple of TN begins a tile, and tiles are numbered by their first tokens.
struct SelfPlan {
    int ids[kSelfPlan];
    int leaders[kSelfPlan / 32];
    int adapter, from, count;
};
template <int TN, int THREADS>
__device__ __forceinline__ Tile self_plan(const AdapterParams &p, SelfPlan &s, int *rows)
{
    constexpr int PER = kSelfPlan / THREADS;
    const int tid = threadIdx.x;
    for (int t = tid; t < kSelfPlan; t += THREADS) s.ids[t] = t < p.rows ? adapter_of(p, t) : -2;
    if (tid == 0) { s.count = 0; s.from = -1; s.adapter = -1; }
    __syncthreads();
    int rank[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = j * THREADS + tid, id = s.ids[t];
        int r = 0;
        for (int o = 0; j * THREADS < p.rows && o < p.rows; o += 4) {
            const int4 q = *reinterpret_cast<const int4 *>(&s.ids[o]);
            r += (q.x == id && o < t) + (q.y == id && o + 1 < t) + (q.z == id && o + 2 < t) + (q.w == id && o + 3 < t);
        }
        rank[j] = r;
        const unsigned b = __ballot_sync(0xffffffffu, id != -2 && r % TN == 0);
        if ((tid & 31) == 0) s.leaders[t >> 5] = (int)b;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = j * THREADS + tid;
        int before = 0;
        for (int w = 0; w < (t >> 5); ++w) before += __popc(s.leaders[w]);
        const unsigned mine = (unsigned)s.leaders[t >> 5];
        before += __popc(mine & ((1u << (t & 31)) - 1u));
        if ((mine >> (t & 31) & 1u) && before == (int)blockIdx.x) { s.adapter = s.ids[t]; s.from = rank[j]; }
    }
    __syncthreads();
    if (s.from < 0) return Tile{-1, 0};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = j * THREADS + tid;
        if (s.ids[t] == s.adapter && rank[j] >= s.from && rank[j] < s.from + TN) {
            rows[rank[j] - s.from] = t;
            atomicAdd(&s.count, 1);
        }
    }
    __syncthreads();
    return Tile{s.adapter, s.count};
}

// The same from the plan in the workspace.
__device__ __forceinline__ Tile read_plan(const AdapterParams &p, int threads, int *rows)
{
    if ((int)blockIdx.x >= __ldcg(p.n_tiles)) return Tile{-1, 0};
    const int4 t = __ldcg(p.tiles + blockIdx.x);
    for (int i = threadIdx.x; i < t.z; i += threads) rows[i] = __ldcg(p.order + t.y + i);
    __syncthreads();
    return Tile{t.x, t.z};
}

// One CTA: counts the tokens of every adapter (the last counter: none), lays the tiles out and sorts the tokens.
__global__ void __launch_bounds__(kPlanThreads) adapter_plan_kernel(const AdapterParams p, int tile_tokens)
{
    extern __shared__ int counts[];          // [adapters + 1] tokens, then the next place in `order`
    __shared__ int2 carry, warp_sum[32];
    const int tid = threadIdx.x, lane = tid & 31, n = p.adapters + 1;
    pdl_release();
    for (int i = tid; i < n; i += kPlanThreads) counts[i] = 0;
    if (tid == 0) carry = make_int2(0, 0);
    if (tid < 4) p.status[tid] = 0;
    __syncthreads();
    // the first tokens' adapters stay in registers between the two passes; all loads of a batch are under way together
    constexpr int KEEP = 8;
    int ids[KEEP];
    const auto fetch = [&](int t0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int t = t0 + j * kPlanThreads + tid;
            ids[j] = t < p.rows ? adapter_of(p, t) : -2;
        }
    };
    for (int t0 = 0; t0 < p.rows; t0 += KEEP * kPlanThreads) {
        fetch(t0);
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            if (t0 + j * kPlanThreads >= p.rows) break;
            const unsigned same = __match_any_sync(0xffffffffu, ids[j]);
            if (ids[j] != -2 && lane == __ffs(same) - 1) atomicAdd(&counts[ids[j] < 0 ? p.adapters : ids[j]], __popc(same));
        }
    }
    __syncthreads();
    // running totals of tokens and tiles over the adapters
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + tid, c = i < n ? counts[i] : 0, tiles = (c + tile_tokens - 1) / tile_tokens;
        int2 s = make_int2(c, tiles);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
            if (lane >= o) { s.x += a; s.y += b; }
        }
        if (lane == 31) warp_sum[tid >> 5] = s;
        __syncthreads();
        if (tid < 32) {
            int2 w = warp_sum[tid];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, w.x, o), b = __shfl_up_sync(0xffffffffu, w.y, o);
                if (lane >= o) { w.x += a; w.y += b; }
            }
            warp_sum[tid] = w;
        }
        __syncthreads();
        const int2 before = tid >= 32 ? warp_sum[(tid >> 5) - 1] : make_int2(0, 0);
        const int start = carry.x + before.x + s.x - c, first = carry.y + before.y + s.y - tiles;
        if (i < n) {
            counts[i] = start;
            for (int q = 0; q < tiles; ++q)
                p.tiles[first + q] = make_int4(i < p.adapters ? i : -1, start + q * tile_tokens, min(tile_tokens, c - q * tile_tokens), 0);
        }
        __syncthreads();
        if (tid == kPlanThreads - 1) carry = make_int2(carry.x + warp_sum[31].x, carry.y + warp_sum[31].y);
        __syncthreads();
    }
    if (tid == 0) *p.n_tiles = carry.y;
    for (int t0 = 0; t0 < p.rows; t0 += KEEP * kPlanThreads) {
        if (p.rows > KEEP * kPlanThreads) fetch(t0);
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            if (t0 + j * kPlanThreads >= p.rows) break;
            const int id = ids[j];
            const unsigned same = __match_any_sync(0xffffffffu, id);
            const int leader = __ffs(same) - 1;
            int at = 0;
            if (id != -2 && lane == leader) at = atomicAdd(&counts[id < 0 ? p.adapters : id], __popc(same));
            at = __shfl_sync(0xffffffffu, at, leader);
            if (id != -2) p.order[at + __popc(same & ((1u << lane) - 1u))] = t0 + j * kPlanThreads + tid;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// v = scaling * x a^T
// ---------------------------------------------------------------------------------------------------------

__host__ __device__ constexpr int align_up(int v, int a) { return (v + a - 1) / a * a; }
__host__ __device__ inline int tmem_cols(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }
// Bytes of a stage: two tiles of the tokens' rows, two of the weights' (and the int8 rows as they come).
__host__ __device__ inline int shrink_stage(int tn, int rank_pad, bool i8) { return (tn + rank_pad) * 256 + (i8 ? tn * kBlockK : 0); }
// The first product reads 128 rows from the start of a tile of tokens, however few there are: what lies behind it decides nothing but
// results that are not read.  The last stage's second tile may need some room behind it.
inline int shrink_smem(int tn, int rank_pad, bool i8)
{
    const int stage = align_up(shrink_stage(tn, rank_pad, i8), 1024), last = tn * 128 + 128 * 128;
    return 1024 + (kShrinkStages - 1) * stage + (stage > last ? stage : last);
}

// Grid: (tiles, ksplit).  CTA y takes the K blocks [y * blocks / ksplit, (y + 1) * blocks / ksplit).
// FAST: rows of x and a start on 16-byte boundaries.  A thread then copies the same 16 bytes of every K block, whose addresses it works
// out once; with the addresses of every copy worked out anew the kernel was bound by its instructions.
template <typename T, bool I8, int TN, bool SELF, bool FAST>
__global__ void __launch_bounds__(kShrinkThreads) adapter_shrink_kernel(const AdapterParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(16) SelfPlan plan;
    __shared__ alignas(8) uint64_t bars[kShrinkStages];
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ int rows[TN];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t cols = tmem_cols(p.rank_pad);
    if (warp == 0) tmem_alloc(&tmem_base, cols);
    if (tid == 0) {
        for (int i = 0; i < kShrinkStages; ++i) mbar_init(smem_u32(&bars[i]), 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (SELF && blockIdx.x == 0 && blockIdx.y == 0)   // long before a wait can run out and record it
            for (int i = 0; i < 4; ++i) p.status[i] = 0;
    }
    tc_fence_before();
    if (!SELF) pdl_wait();
    // Only now: the next kernel's CTAs wait for this grid with tensor memory in their hands, so every CTA of this one has its own first.
    __syncthreads();
    pdl_release();
    tc_fence_after();
    const Tile tile = SELF ? self_plan<TN, kShrinkThreads>(p, plan, rows) : read_plan(p, kShrinkThreads, rows);
    const int blocks = (p.k + kBlockK - 1) / kBlockK;
    const int kb0 = (int)((long long)blockIdx.y * blocks / p.ksplit), kb1 = (int)((long long)(blockIdx.y + 1) * blocks / p.ksplit);
    if (tile.count > 0 && tile.adapter >= 0 && kb0 < kb1) {
        const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
        const uint32_t stage_bytes = align_up(shrink_stage(TN, p.rank_pad, I8), 1024);
        constexpr int XB = I8 ? 1 : 2;
        const char *x = reinterpret_cast<const char *>(p.x);
        const char *a = reinterpret_cast<const char *>(p.a) + (long long)tile.adapter * p.rank * p.k * 2;
        const uint32_t a_tile = TN * 256, raw_tile = (uint32_t)(TN + p.rank_pad) * 256;
        // copies per token row of a K block, and rows apart of a thread's copies: a multiple of 8, so their places differ by that many rows
        constexpr int XC = kBlockK * XB / 16, X_ROWS = kShrinkThreads / XC, AC = kBlockK * 2 / 16, A_ROWS = kShrinkThreads / AC;
        static_assert(X_ROWS % 8 == 0 && A_ROWS % 8 == 0, "whole groups of swizzled rows");
        constexpr int NX = (TN + X_ROWS - 1) / X_ROWS, NA = 128 / A_ROWS;
        const char *x_at[NX];
        const int xc = tid % XC, xr = tid / XC, ac = tid % AC, ar = tid / AC;
        const uint32_t x_to = I8 ? raw_tile + (uint32_t)(xr * kBlockK + xc * 16) : (uint32_t)(xc / 8 * TN * 128) + swizzled(xr, xc % 8 * 16);
        const uint32_t a_to = a_tile + (uint32_t)(ac / 8 * p.rank_pad * 128) + swizzled(ar, ac % 8 * 16);
        const char *a_at = a + (long long)ar * p.k * 2 + ac * 16;
        const long long a_step = (long long)A_ROWS * p.k * 2;
        const int na = FAST ? (p.rank - ar + A_ROWS - 1) / A_ROWS : 0;
        if (FAST) {
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                const int r = xr + i * X_ROWS;
                x_at[i] = r < tile.count ? x + (long long)rows[r] * p.ld_x * XB + xc * 16 : nullptr;
            }
        }
        const auto load = [&](int kb) {
            const uint32_t s = smem0 + (uint32_t)((kb - kb0) % kShrinkStages) * stage_bytes;
            const int have = min(kBlockK, p.k - kb * kBlockK);
            if (FAST) {
                const int ax = min(max(have * XB - xc * 16, 0), 16), aa = min(max(have * 2 - ac * 16, 0), 16);
                // a copy of no bytes names the row's start: its own place may lie beyond the tensor
                const long long xo = ax > 0 ? (long long)kb * kBlockK * XB : -(long long)xc * 16;
                const char *from = a_at + (aa > 0 ? (long long)kb * kBlockK * 2 : -(long long)ac * 16);
#pragma unroll
                for (int i = 0; i < NX; ++i)
                    if (x_at[i]) cp_async<16>(s + x_to + i * X_ROWS * (I8 ? kBlockK : 128), x_at[i] + xo, ax);
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    if (i < na) cp_async<16>(s + a_to + i * A_ROWS * 128, from, aa);
                    from += a_step;
                }
                return;
            }
            for (int at = 0; at < 2; ++at) {
                const long long k0 = (long long)kb * kBlockK + at * 64;
                if (at * 64 >= (have + 15) / 16 * 16) break;   // no K step reaches the second tile
                copy_rows<true, kShrinkThreads>(p.grain_a, s + a_tile + (uint32_t)(at * p.rank_pad * 128), p.rank, 128, (have - at * 64) * 2,
                                                [&](int r) { return a + ((long long)r * p.k + k0) * 2; });
                if (!I8)
                    copy_rows<true, kShrinkThreads>(p.grain_x, s + (uint32_t)(at * TN * 128), tile.count, 128, (have - at * 64) * 2,
                                                    [&](int r) { return x + ((long long)rows[r] * p.ld_x + k0) * XB; });
            }
            if (I8)
                copy_rows<false, kShrinkThreads>(p.grain_x, s + raw_tile, tile.count, kBlockK, have,
                                                 [&](int r) { return x + (long long)rows[r] * p.ld_x + (long long)kb * kBlockK; });
        };
        for (int i = 0; i < kShrinkStages - 1; ++i) {
            if (kb0 + i < kb1) load(kb0 + i);
            cp_commit();
        }
        const uint32_t idesc = instr_desc<T>(p.rank_pad);
        for (int kb = kb0; kb < kb1; ++kb) {
            const int i = kb - kb0, stage = i % kShrinkStages;
            const uint32_t s = smem0 + (uint32_t)stage * stage_bytes;
            cp_wait<kShrinkStages - 2>();
            if (I8 && FAST) widen_rows_grain<T, 16, kShrinkThreads>(s + raw_tile, s, TN * 128, tile.count);
            else if (I8) widen_rows<T, kShrinkThreads>(p.grain_x, s + raw_tile, s, TN * 128, tile.count);
            fence_async_proxy();
            __syncthreads();
            if (tid == 0) {
                tc_fence_after();
                const uint64_t xd = operand_desc(s), ad = operand_desc(s + a_tile);
                const int steps = (min(kBlockK, p.k - kb * kBlockK) + 15) / 16;
                for (int j = 0; j < steps; ++j)
                    umma_f16(tmem_base, xd + j / 4 * (TN * 128 / 16) + j % 4 * 2, ad + j / 4 * (p.rank_pad * 128 / 16) + j % 4 * 2, idesc, (i | j) != 0);
                umma_commit(smem_u32(&bars[stage]));
            }
            // the stage that the block before this one was read from takes the next block
            if (kb + kShrinkStages - 1 < kb1) {
                if (i > 0) mbar_wait(smem_u32(&bars[(i - 1) % kShrinkStages]), ((i - 1) / kShrinkStages) & 1, &gave_up, p.status, 900);
                load(kb + kShrinkStages - 1);
            }
            cp_commit();
        }
        const int last = kb1 - 1 - kb0;
        mbar_wait(smem_u32(&bars[last % kShrinkStages]), (last / kShrinkStages) & 1, &gave_up, p.status, 901);
        tc_fence_after();
        const int slot = warp * 32 + lane;
        if (warp * 32 < TN) {
            const bool live = slot < tile.count;
            const int row = live ? rows[slot] : 0;
            float f = p.scaling ? __ldg(p.scaling + tile.adapter) : 1.0f;
            if (I8 && live) f = __fmul_rn(f, __ldg(p.x_scale + row));
            float4 *v = reinterpret_cast<float4 *>(p.v + ((long long)blockIdx.y * p.rows + row) * p.rank_pad);
            for (int c = 0; c < p.rank_pad; c += 16) {
                uint32_t d[16];
                tmem_ld16(tmem_base + ((uint32_t)(warp * 32) << 16) + (uint32_t)c, d);
                tmem_ld_wait();
                if (live) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        v[(c + e) / 4] = make_float4(__fmul_rn(__uint_as_float(d[e]), f), __fmul_rn(__uint_as_float(d[e + 1]), f),
                                                     __fmul_rn(__uint_as_float(d[e + 2]), f), __fmul_rn(__uint_as_float(d[e + 3]), f));
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem_base, cols);
}

// ---------------------------------------------------------------------------------------------------------
// out = base + v b^T
// ---------------------------------------------------------------------------------------------------------

__host__ __device__ inline int rank_atoms(int rank_pad) { return rank_pad > 64 ? 2 : 1; }
__host__ __device__ inline int expand_stage(int tn, int rank_pad) { return rank_atoms(rank_pad) * kChunkN * 128 + tn * kChunkN * 2; }
inline int expand_smem(int tn, int rank_pad) { return 1024 + rank_atoms(rank_pad) * tn * 256 + kExpandStages * expand_stage(tn, rank_pad); }

// Grid: (tiles, nsplit).  CTA y takes the channel chunks [y * chunks / nsplit, (y + 1) * chunks / nsplit).
// GB: 16 or 8 bytes of b a copy, with rows of base and out on 16-byte boundaries; addresses are worked out once, and results go back
// through the chunk's base rows in shared memory, from which they are stored 16 bytes at a time.  0: any strides.
template <typename T, int TN, bool SELF, int GB>
__global__ void __launch_bounds__(kExpandThreads) adapter_expand_kernel(const AdapterParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(16) SelfPlan plan;
    __shared__ alignas(8) uint64_t bar;
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ int rows[TN];
    __shared__ float unscale[TN];          // fp16: the power of two that v was divided by
    constexpr bool F16 = std::is_same<T, __half>::value;
    constexpr uint32_t COLS = TN <= 32 ? 32 : TN;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (warp == 0) tmem_alloc(&tmem_base, COLS);
    if (tid == 0) {
        mbar_init(smem_u32(&bar), 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const Tile tile = SELF ? self_plan<TN, kExpandThreads>(p, plan, rows) : read_plan(p, kExpandThreads, rows);
    const int chunks = (p.n + kChunkN - 1) / kChunkN;
    const int c0 = (int)((long long)blockIdx.y * chunks / p.nsplit), c1 = (int)((long long)(blockIdx.y + 1) * chunks / p.nsplit);
    const T *base = reinterpret_cast<const T *>(p.base);
    T *out = reinterpret_cast<T *>(p.out);
    if (tile.count > 0 && tile.adapter < 0) {
        if (p.out != p.base) {
            pdl_wait();
            const int n0 = c0 * kChunkN, width = min(c1 * kChunkN, p.n) - n0;
            constexpr int V = GB ? 8 : 1, AHEAD = 4;     // elements a copy, copies in flight
            using Copy = typename std::conditional<GB != 0, uint4, uint16_t>::type;
            const int across = (width + V - 1) / V, total = across * tile.count;   // at most 64 rows of 65535
            for (int i0 = tid; i0 < total; i0 += kExpandThreads * AHEAD) {
                Copy v[AHEAD];
                T *to[AHEAD];
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const int i = i0 + j * kExpandThreads, r = i / across, c = n0 + (i - r * across) * V;
                    to[j] = nullptr;
                    if (i < total) {
                        v[j] = *reinterpret_cast<const Copy *>(base + (long long)rows[r] * p.ld_base + c);
                        to[j] = out + (long long)rows[r] * p.ld_out + c;
                    }
                }
#pragma unroll
                for (int j = 0; j < AHEAD; ++j)
                    if (to[j]) *reinterpret_cast<Copy *>(to[j]) = v[j];
            }
        }
    } else if (tile.count > 0 && c0 < c1) {
        const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
        const int atoms = rank_atoms(p.rank_pad);
        const uint32_t v_hi = smem0, v_lo = v_hi + (uint32_t)(atoms * TN * 128), stage0 = v_lo + (uint32_t)(atoms * TN * 128);
        const uint32_t stage_bytes = expand_stage(TN, p.rank_pad), base_at = (uint32_t)(atoms * kChunkN * 128);
        const char *b = reinterpret_cast<const char *>(p.b) + (long long)tile.adapter * p.n * p.rank * 2;
        // b: the copies of a chunk, offset in its rows << 8 | bytes, and place in the tile
        constexpr int NB = GB ? 256 / (2 * GB) : 1, NR = TN * 16 / kExpandThreads;
        const int per_row = GB ? p.rank_pad * 2 / (GB ? GB : 1) : 1, nb = per_row * kChunkN / kExpandThreads;
        uint32_t b_from[NB], b_to[NB];
        long long base_at_row[NR], out_at_row[NR];
        const int rc = (tid % 16) * 8;
        if (GB) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int idx = tid + i * kExpandThreads, r = idx / per_row, byte = (idx - r * per_row) * GB;
                const int valid = min(max(p.rank * 2 - byte, 0), GB);
                b_from[i] = (uint32_t)(r * p.rank * 2 + (valid ? byte : 0)) << 8 | (uint32_t)valid;
                b_to[i] = (uint32_t)(byte / 128 * kChunkN * 128) + swizzled(r, byte % 128);
            }
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int r = tid / 16 + i * 16;
                base_at_row[i] = r < tile.count ? (long long)rows[r] * p.ld_base + rc : -1;
                out_at_row[i] = r < tile.count ? (long long)rows[r] * p.ld_out + rc : -1;
            }
        }
        const auto load = [&](int c) {
            const uint32_t s = stage0 + (uint32_t)((c - c0) % kExpandStages) * stage_bytes;
            const int n0 = c * kChunkN, channels = min(kChunkN, p.n - n0);
            if (GB) {
                const char *from = b + (long long)n0 * p.rank * 2;
                const uint32_t end = (uint32_t)(channels * p.rank * 2);
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    if (i >= nb) break;
                    if (b_from[i] >> 8 < end) cp_async<GB ? GB : 16>(s + b_to[i], from + (b_from[i] >> 8), (int)(b_from[i] & 255u));
                }
#pragma unroll
                for (int i = 0; i < NR; ++i)
                    if (base_at_row[i] >= 0 && rc < channels)
                        cp_async<16>(s + base_at + (uint32_t)((tid + i * kExpandThreads) * 16), base + base_at_row[i] + n0, 16);
                return;
            }
            for (int at = 0; at < atoms; ++at) {
                const int left = p.rank_pad - at * 64;                       // a whole number of K steps, zero beyond the rank
                const int width = left > 32 ? 128 : left > 16 ? 64 : 32;
                copy_rows<true, kExpandThreads>(p.grain_b, s + (uint32_t)at * kChunkN * 128, channels, width, (p.rank - at * 64) * 2,
                                                [&](int r) { return b + ((long long)(n0 + r) * p.rank + at * 64) * 2; });
            }
            copy_rows<false, kExpandThreads>(p.grain_base, s + base_at, tile.count, kChunkN * 2, channels * 2,
                                             [&](int r) { return reinterpret_cast<const char *>(base + (long long)rows[r] * p.ld_base + n0); });
        };
        for (int i = 0; i < kExpandStages; ++i) {
            if (c0 + i < c1) load(c0 + i);
            cp_commit();
        }
        pdl_wait();   // the partial sums are complete
        {
            constexpr int LANES = kExpandThreads / TN;    // per token
            const int slot = tid / LANES, part = tid % LANES;
            const bool live = slot < tile.count;
            const int row = live ? rows[slot] : 0;
            constexpr int CH = 16 / LANES;                // 8 components of v each, LANES apart
            float f[CH][8];
#pragma unroll
            for (int h = 0; h < CH; ++h)
#pragma unroll
                for (int e = 0; e < 8; ++e) f[h][e] = 0.0f;
            const float4 *v = reinterpret_cast<const float4 *>(p.v + (long long)row * p.rank_pad);
            const long long split = (long long)p.rows * p.rank_pad / 4;
            if (live) {
                constexpr int AHEAD = CH == 1 ? 8 : 4;    // partial sums that are fetched together
                for (int s0 = 0; s0 < p.ksplit; s0 += AHEAD) {
#pragma unroll
                    for (int h = 0; h < CH; ++h) {
                        const int j = (part + h * LANES) * 8;
                        if (j >= p.rank_pad) break;
                        float4 q[AHEAD][2];
#pragma unroll
                        for (int s = 0; s < AHEAD; ++s) {
                            const bool there = s0 + s < p.ksplit;
                            q[s][0] = there ? __ldcg(v + (s0 + s) * split + j / 4) : make_float4(0, 0, 0, 0);
                            q[s][1] = there ? __ldcg(v + (s0 + s) * split + j / 4 + 1) : make_float4(0, 0, 0, 0);
                        }
#pragma unroll
                        for (int s = 0; s < AHEAD; ++s) {
                            f[h][0] += q[s][0].x; f[h][1] += q[s][0].y; f[h][2] += q[s][0].z; f[h][3] += q[s][0].w;
                            f[h][4] += q[s][1].x; f[h][5] += q[s][1].y; f[h][6] += q[s][1].z; f[h][7] += q[s][1].w;
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < CH; ++h)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((part + h * LANES) * 8 + e >= p.rank) f[h][e] = 0.0f;
            }
            float down = 1.0f;
            if (F16) {
                uint32_t m = 0;
#pragma unroll
                for (int h = 0; h < CH; ++h)
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(f[h][e]) & 0x7fffffffu);
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                // 2^-e for a largest value in [2^e, 2^(e+1)); none for zero, for what no power of two can help, and at the ends of fp32
                const int e = (int)(m >> 23) - 127;
                const bool shift = m != 0 && e > -120 && e < 120;
                down = shift ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.0f;
                if (part == 0) unscale[slot] = shift ? __uint_as_float((uint32_t)(127 + e) << 23) : 1.0f;
            }
#pragma unroll
            for (int h = 0; h < CH; ++h) {
                const int j = (part + h * LANES) * 8;
                if (j >= p.rank_pad) break;
                float g[8];
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f[h][e] = __fmul_rn(f[h][e], down);
                    g[e] = __fsub_rn(f[h][e], to_float(from_float<T>(f[h][e])));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[e] = pack2<T>(f[h][2 * e], f[h][2 * e + 1]);
                    lo[e] = pack2<T>(g[2 * e], g[2 * e + 1]);
                }
                const uint32_t at = (uint32_t)(j / 64 * TN * 128) + swizzled(slot, (j % 64) * 2);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(v_hi + at), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(v_lo + at), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
            }
        }
        const uint32_t idesc = instr_desc<T>(TN);
        const auto multiply = [&](int c) {   // by one thread
            const uint32_t s = stage0 + (uint32_t)((c - c0) % kExpandStages) * stage_bytes;
            tc_fence_after();
            uint32_t more = 0;
            for (int j = 0; j < p.rank_pad / 16; ++j) {
                const uint64_t bd = operand_desc(s + (uint32_t)(j / 4) * kChunkN * 128) + (j % 4) * 2;
                umma_f16(tmem_base, bd, operand_desc(v_hi + (uint32_t)(j / 4) * TN * 128) + (j % 4) * 2, idesc, more);
                more = 1;
                umma_f16(tmem_base, bd, operand_desc(v_lo + (uint32_t)(j / 4) * TN * 128) + (j % 4) * 2, idesc, more);
            }
            umma_commit(smem_u32(&bar));
        };
        cp_wait<kExpandStages - 1>();
        fence_async_proxy();
        __syncthreads();
        if (tid == 0) multiply(c0);
        // warp w: channels 32 (w % 4) + lane, half of the tokens
        constexpr int HALF = TN / 2;
        const int q = warp & 3, ch = q * 32 + lane, first = (warp >> 2) * HALF;
        for (int c = c0; c < c1; ++c) {
            const int i = c - c0, n = c * kChunkN + ch;
            const uint32_t s = stage0 + (uint32_t)(i % kExpandStages) * stage_bytes;
            mbar_wait(smem_u32(&bar), i & 1, &gave_up, p.status, 910);
            tc_fence_after();
            uint32_t d[HALF];
            if (first < tile.count) {
#pragma unroll
                for (int t0 = 0; t0 < HALF; t0 += 8) tmem_ld8(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(first + t0), d + t0);
                tmem_ld_wait();
                const uint32_t at = s + base_at + (uint32_t)(first * kChunkN * 2 + ch * 2);
#pragma unroll
                for (int t0 = 0; t0 < HALF; t0 += 8) {
                    if (first + t0 >= tile.count) break;
                    uint16_t raw[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) asm volatile("ld.shared.u16 %0, [%1];" : "=h"(raw[e]) : "r"(at + (t0 + e) * kChunkN * 2) : "memory");
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int slot = first + t0 + e;   // beyond the tile's tokens: values of no meaning that are not stored
                        float f = __uint_as_float(d[t0 + e]);
                        if (F16) f = __fmul_rn(f, unscale[slot]);
                        const T o = from_float<T>(__fadd_rn(to_float(*reinterpret_cast<const T *>(&raw[e])), f));
                        if (GB) asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + (t0 + e) * kChunkN * 2), "h"(*reinterpret_cast<const uint16_t *>(&o)) : "memory");
                        else if (slot < tile.count && n < p.n) out[(long long)rows[slot] * p.ld_out + n] = o;
                    }
                }
            }
            tc_fence_before();
            cp_wait<0>();           // the next chunk, for which a whole round was time
            fence_async_proxy();
            __syncthreads();        // this chunk's results are in place, its accumulators read, the next chunk there
            if (tid == 0 && c + 1 < c1) multiply(c + 1);
            if (GB) {   // a thread stores the 16 bytes whose place it then fills again
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    if (out_at_row[i] >= 0 && c * kChunkN + rc < p.n) {
                        uint4 o;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(o.x), "=r"(o.y), "=r"(o.z), "=r"(o.w)
                                     : "r"(s + base_at + (uint32_t)((tid + i * kExpandThreads) * 16)) : "memory");
                        *reinterpret_cast<uint4 *>(out + out_at_row[i] + c * kChunkN) = o;
                    }
                }
            }
            if (c + kExpandStages < c1) load(c + kExpandStages);
            cp_commit();
        }
        cp_wait<0>();
    }
    pdl_wait();   // this grid must not end before the kernels in front of it: the stream goes on behind it alone
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem_base, COLS);
}

// ---------------------------------------------------------------------------------------------------------

template <typename... KArgs>
cudaError_t launch_kernel(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t stream, bool dependent, KArgs... args)
{
    if (smem > 44 * 1024) {   // with what the kernel has of its own it may pass 48 KB
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

constexpr size_t align256(size_t v) { return (v + 255) / 256 * 256; }

struct Shape {
    int tile_tokens, tiles, ksplit, nsplit, rank_pad;
    bool self;
};

// Tiles of 16 tokens while every CTA plans for itself, of 64 beyond.  `tiles` is the most there can be: full ones, and one that is not for
// every adapter and for none.  K and N are split so that the CTAs find a place on the SMs together (about five of the small ones fit an SM,
// two of the large), but no CTA gets less than two K blocks.
Shape shape_of(const AdapterProblem &p)
{
    Shape s;
    s.self = p.rows <= kSelfPlan;
    s.tile_tokens = s.self ? 16 : 64;
    const long long partial = p.adapters + 1 < p.rows ? p.adapters + 1 : p.rows;
    s.tiles = (int)(p.rows / s.tile_tokens + partial);
    if (s.tiles > p.rows) s.tiles = (int)p.rows;
    s.rank_pad = align_up((int)p.rank, 16);
    const int want = (s.self ? 4 : 2) * 148 / s.tiles;
    const int blocks = (int)((p.k + kBlockK - 1) / kBlockK), chunks = (int)((p.n + kChunkN - 1) / kChunkN);
    s.ksplit = want < blocks / 2 ? want : blocks / 2;
    if (s.ksplit > 16) s.ksplit = 16;
    if (s.ksplit < 1) s.ksplit = 1;
    s.nsplit = want < chunks ? want : chunks;
    if (s.nsplit < 1) s.nsplit = 1;
    return s;
}

int grain_of(const void *base, long long pitch_bytes, int smallest)
{
    const uintptr_t v = (uintptr_t)base | (uintptr_t)pitch_bytes;
    return v % 16 == 0 ? 16 : v % 8 == 0 ? 8 : v % 4 == 0 ? 4 : smallest;
}

template <typename T, bool I8, int TN, bool SELF>
cudaError_t launch_tiles(const AdapterParams &p, const Shape &s, cudaStream_t stream)
{
    cudaError_t e = cudaSuccess;
    if (!SELF) {
        e = launch_kernel(adapter_plan_kernel, dim3(1), kPlanThreads, (p.adapters + 1) * 4, stream, false, p, s.tile_tokens);
        if (e != cudaSuccess) return e;
    }
    const auto shrink = p.grain_x == 16 && p.grain_a == 16 ? adapter_shrink_kernel<T, I8, TN, SELF, true> : adapter_shrink_kernel<T, I8, TN, SELF, false>;
    e = launch_kernel(shrink, dim3((unsigned)s.tiles, (unsigned)s.ksplit), kShrinkThreads, shrink_smem(TN, s.rank_pad, I8), stream, !SELF, p);
    if (e != cudaSuccess) return e;
    const bool rows16 = p.grain_base == 16 && p.grain_out == 16 && p.n % 8 == 0;
    const auto expand = rows16 && p.grain_b == 16 ? adapter_expand_kernel<T, TN, SELF, 16>
                        : rows16 && p.grain_b == 8 ? adapter_expand_kernel<T, TN, SELF, 8> : adapter_expand_kernel<T, TN, SELF, 0>;
    return launch_kernel(expand, dim3((unsigned)s.tiles, (unsigned)s.nsplit), kExpandThreads, expand_smem(TN, s.rank_pad), stream, true, p);
}

template <typename T, bool I8>
cudaError_t launch_typed(const AdapterParams &p, const Shape &s, cudaStream_t stream)
{
    return s.self ? launch_tiles<T, I8, 16, true>(p, s, stream) : launch_tiles<T, I8, 64, false>(p, s, stream);
}

}  // namespace

size_t adapter_workspace_bytes(const AdapterProblem &p)
{
    const Shape s = shape_of(p);
    return 256 + (s.self ? 0 : 256 + align256((size_t)s.tiles * sizeof(int4)) + align256((size_t)p.rows * 4)) +
           align256((size_t)s.ksplit * (size_t)p.rows * (size_t)s.rank_pad * 4);
}

cudaError_t adapter_launch(const AdapterProblem &a, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (a.rows <= 0) return cudaSuccess;
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < adapter_workspace_bytes(a)) return cudaErrorInvalidValue;
    const Shape s = shape_of(a);
    AdapterParams p;
    p.base = a.base; p.x = a.x; p.a = a.a; p.b = a.b;
    p.x_scale = a.x_scale; p.scaling = a.scaling; p.ids = a.ids; p.out = a.out;
    p.ld_base = a.ld_base; p.ld_x = a.ld_x; p.ld_out = a.ld_out;
    p.rows = (int)a.rows; p.k = (int)a.k; p.n = (int)a.n; p.adapters = (int)a.adapters; p.rank = (int)a.rank;
    p.rank_pad = s.rank_pad;
    const int xb = a.x_i8 ? 1 : 2;
    p.grain_x = grain_of(a.x, a.ld_x * xb, xb);
    p.grain_a = grain_of(a.a, a.k * 2, 2);
    p.grain_b = grain_of(a.b, a.rank * 2, 2);
    p.grain_base = grain_of(a.base, a.ld_base * 2, 2);
    p.grain_out = grain_of(a.out, a.ld_out * 2, 2);
    p.ksplit = s.ksplit; p.nsplit = s.nsplit;
    char *ws = static_cast<char *>(workspace);
    p.status = reinterpret_cast<int *>(ws);
    ws += 256;
    p.n_tiles = nullptr; p.tiles = nullptr; p.order = nullptr;
    if (!s.self) {
        p.n_tiles = reinterpret_cast<int *>(ws); ws += 256;
        p.tiles = reinterpret_cast<int4 *>(ws); ws += align256((size_t)s.tiles * sizeof(int4));
        p.order = reinterpret_cast<int *>(ws); ws += align256((size_t)a.rows * 4);
    }
    p.v = reinterpret_cast<float *>(ws);
    if (a.dtype == kF16) return a.x_i8 ? launch_typed<__half, true>(p, s, stream) : launch_typed<__half, false>(p, s, stream);
    return a.x_i8 ? launch_typed<__nv_bfloat16, true>(p, s, stream) : launch_typed<__nv_bfloat16, false>(p, s, stream);
}

}  // namespace gmm
