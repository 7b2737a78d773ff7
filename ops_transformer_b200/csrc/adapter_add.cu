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
// v enters the second product as three 16-bit parts, each the rounded rest of v less the ones before: all 24 bits of it, so the sums are
// those of fp32 throughout.  fp16 has no range to spare, so there every token's v is scaled by a power of two to just below 2^15: parts
// end at 2^-24, which is 2^-39 of the token's largest component.
// The operands are fetched with 16-byte asynchronous copies (8, 4 or 2 bytes where rows start on no such boundary), straight into the
// 128-byte-swizzled layout that the tensor cores read; a row's tail is zero filled.
//
// Which tokens share an adapter is found on the device by a one-CTA kernel that counts and sorts them.  The order within an adapter does
// not matter: every row's arithmetic is its own.  A few tokens take two kernels on the CUDA cores instead, whose CTAs find their tiles
// themselves.
//
// 4096 tokens of 8 adapters, 7168 -> 4096, rank 64, bf16: 50 us for 137 MB, which take 21 at the rate of a copy: the plan 5, the first
// product 17 (its operands come at about 55 bytes per ns and SM, weights included, which every tile reads anew), the second some 22 (3 for
// the partial sums, then 4 TB/s; with two parts of v the three kernels took 48).  611 tokens of 13, 1424 -> 2976, rank 12: 16 us, the three kernels' latencies (3, 5 and 5).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "gmm_common.h"

namespace gmm {
namespace {

constexpr int kBlockK = 128;         // elements of a row per K block
constexpr int kBlockTiles = kBlockK / 64;   // swizzled rows of 128 bytes that these make
constexpr int kChunkN = 128;         // channels per step of the second product
constexpr int kSelfPlan = 256;       // most tokens for which every CTA finds its tile itself, a thread for each
constexpr int kPlanThreads = 1024;
constexpr int kWorkers = 256;        // threads of the first kernel that copy; one warp more issues the products
__host__ __device__ constexpr int expand_workers(int tn) { return tn == 64 ? 512 : 256; }
constexpr int kMaxStages = 6, kShrinkAhead = 2, kExpandStages = 2;
constexpr long long kWaitLimitCycles = 1ll << 31;   // of a call that names no other: about a second

struct AdapterParams {
    const void *base, *x, *a, *b;
    const float *x_scale, *scaling;
    const int *ids;
    void *out;
    long long ld_base, ld_x, ld_out;
    int rows, k, n, adapters, rank;
    int rank_pad;                   // rank, rounded up to the tensor cores' K step of 16
    int grain_x, grain_a, grain_b, grain_base, grain_out;   // bytes of a copy
    int ksplit, nsplit, stages;
    int parts;                      // tiles of the second kernel in one of the first
    int skip_blocks;                // test only: K blocks of every tile whose arrival the first kernel leaves out
    long long wait_limit;           // cycles
    int *status;                    // [4]
    int *n_tiles;
    int2 *tiles;                    // adapter (-1: none), tokens
    int *order;                     // [tiles, tile_tokens] the tokens of every tile
    float *v;                       // [ksplit, rows, rank_pad] partial sums
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
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// An arrival at `bar` once this thread's copies so far have landed.
__device__ __forceinline__ void mbar_arrive_copies(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
template <int THREADS>
__device__ __forceinline__ void worker_sync() { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); }
// Bounded wait for the tensor cores, or for the copies that they wait for.  When it runs out the status says so and later waits of the CTA
// return at once, except those that LAST stands for: behind one, nothing that the CTA has under way may be left.
template <bool LAST>
__device__ __noinline__ void mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int *gave_up, int *status, long long limit, int role)
{
    const long long t0 = clock64();
    while (!mbar_try(bar, parity)) {
        if (!LAST && *gave_up) return;
        if (clock64() - t0 > limit) {
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
template <bool LAST = false>
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, volatile int *gave_up, const AdapterParams &p, int role)
{
    if (!mbar_try(bar, parity)) mbar_wait_slow<LAST>(bar, parity, gave_up, p.status, p.wait_limit, role);
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

// The tile of at most TN tokens that begins with token blockIdx.x, found by every CTA for itself; rows[slot] = token.  A token begins one if
// a multiple of TN tokens of its adapter come before it; the CTAs of the others have nothing to do.
struct SelfPlan {
    unsigned same[kSelfPlan / 32];   // the tokens of the first token's adapter
};
template <int TN>
__device__ __forceinline__ Tile self_plan(const AdapterParams &p, SelfPlan &s, int *rows)
{
    const int tid = threadIdx.x, x = blockIdx.x, id = adapter_of(p, x);
    bool same = false;
    if (tid < kSelfPlan) {
        same = tid < p.rows && adapter_of(p, tid) == id;
        const unsigned b = __ballot_sync(0xffffffffu, same);
        if ((tid & 31) == 0) s.same[tid >> 5] = b;
    }
    __syncthreads();
    int before = 0, all = 0, mine = 0;
#pragma unroll
    for (int w = 0; w < kSelfPlan / 32; ++w) {
        const unsigned b = s.same[w];
        const auto below = [&](int t) { return __popc(t >= w * 32 + 32 ? b : t <= w * 32 ? 0u : b & ((1u << (t - w * 32)) - 1u)); };
        all += __popc(b);
        before += below(x);
        mine += below(tid);
    }
    if (before % TN != 0) return Tile{-1, 0};
    if (same && mine >= before && mine < before + TN) rows[mine - before] = tid;
    __syncthreads();
    return Tile{id, min(TN, all - before)};
}

// The same from the plan in the workspace, whose tiles hold `parts` of them: number `place`.
template <int TN>
__device__ __forceinline__ Tile read_plan(const AdapterParams &p, int place, int parts, int threads, int *rows)
{
    const int tiles = __ldcg(p.n_tiles), at = place / parts, part = place % parts;
    const int2 t = __ldcg(p.tiles + at);   // with the rows, whose places do not hang on it, in one go
    for (int i = threadIdx.x; i < TN; i += threads) rows[i] = __ldcg(p.order + (long long)place * TN + i);
    __syncthreads();
    return at < tiles ? Tile{t.x, max(0, min(TN, t.y - part * TN))} : Tile{-1, 0};
}

// One CTA: counts the tokens of every adapter (the last counter: none), lays the tiles out and sorts the tokens.
__global__ void __launch_bounds__(kPlanThreads) adapter_plan_kernel(const AdapterParams p, int tile_tokens)
{
    extern __shared__ int counts[];          // [adapters + 1] tokens, then the next place in `order`, whose tiles are not packed
    __shared__ int carry, warp_sum[32];
    const int tid = threadIdx.x, lane = tid & 31, n = p.adapters + 1;
    pdl_release();
    for (int i = tid; i < n; i += kPlanThreads) counts[i] = 0;
    if (tid == 0) carry = 0;
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
    // running totals of the tiles over the adapters
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + tid, c = i < n ? counts[i] : 0, tiles = (c + tile_tokens - 1) / tile_tokens;
        int s = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += t;
        }
        if (lane == 31) warp_sum[tid >> 5] = s;
        __syncthreads();
        if (tid < 32) {
            int w = warp_sum[tid];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += t;
            }
            warp_sum[tid] = w;
        }
        __syncthreads();
        const int first = carry + (tid >= 32 ? warp_sum[(tid >> 5) - 1] : 0) + s - tiles;
        if (i < n) {
            counts[i] = first * tile_tokens;
            for (int q = 0; q < tiles; ++q) p.tiles[first + q] = make_int2(i < p.adapters ? i : -1, min(tile_tokens, c - q * tile_tokens));
        }
        __syncthreads();
        if (tid == kPlanThreads - 1) carry += warp_sum[31];
        __syncthreads();
    }
    if (tid == 0) *p.n_tiles = carry;
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

// Channels [n0, n1) of rows without an adapter, V elements a copy.
template <typename T, int V, int THREADS>
__device__ __forceinline__ void copy_base(const AdapterParams &p, const int *rows, int count, int n0, int n1)
{
    using Copy = typename std::conditional<V == 8, uint4, uint16_t>::type;
    static_assert(V == 8 || V == 1, "");
    constexpr int AHEAD = 4;   // copies in flight
    const T *base = reinterpret_cast<const T *>(p.base);
    T *out = reinterpret_cast<T *>(p.out);
    const int across = (n1 - n0 + V - 1) / V, total = across * count;   // at most 64 rows of 65535
    for (int i0 = threadIdx.x; i0 < total; i0 += THREADS * AHEAD) {
        Copy v[AHEAD];
        T *to[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j * THREADS, r = i / across, c = n0 + (i - r * across) * V;
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

// ---------------------------------------------------------------------------------------------------------
// A few tokens per adapter: streams of weights, on the CUDA cores
// ---------------------------------------------------------------------------------------------------------
//
// With up to four tokens a tile each weight takes part in four products at most, which costs fewer instructions than bringing it to the
// tensor cores; the weights go straight from memory to registers, 16 bytes a lane, and every CTA finds its own tile, so there are two
// kernels and nothing in front of them.  One token, 2048 -> 4096, rank 16: 4.3 us, the two kernels' latency; 128 tokens of 64 adapters,
// 2048 -> 7168, rank 32, int8: 19.3 us (28 on the tensor cores) for 42 MB.  Neither the memory (at 6.4 us for these) nor the issue slots (46 % of
// them used) bound that: with 74 and 107 registers a thread an SM has 20 and 14 warps at work on average, whose longest stall is for loads.

constexpr int kFew = 4;
constexpr int kFewThreads = 256;
constexpr int kFewExpandCtas = 2;   // that fit an SM by their registers

template <typename T> __device__ __forceinline__ void unpack8(const uint4 &u, f32x2 (&f)[4]);
template <> __device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4 &u, f32x2 (&f)[4])
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pair2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <> __device__ __forceinline__ void unpack8<__half>(const uint4 &u, f32x2 (&f)[4])
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[i] = pair2(t.x, t.y);
    }
}
// Eight int8: a byte plus 128 in the low bits of 2^23 is the float 2^23 + 128 + q.
__device__ __forceinline__ void unpack8(const uint2 &u, f32x2 (&f)[4])
{
    const uint32_t w[2] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = __uint_as_float(__byte_perm(w[i / 2], 0x4b000000u, i % 2 ? 0x7652 : 0x7650));
        const float b = __uint_as_float(__byte_perm(w[i / 2], 0x4b000000u, i % 2 ? 0x7653 : 0x7651));
        f[i] = pair2(__fsub_rn(a, 8388736.0f), __fsub_rn(b, 8388736.0f));
    }
}

// 16 bytes at `at`, on any boundary of a 16-bit element, of which the first `valid` count and the others are zero: out of the two aligned
// packs that hold them, where these lie in [begin, end), else element by element.
__device__ __forceinline__ uint4 load_any(const char *at, int valid, const char *begin, const char *end)
{
    if (valid <= 0) return make_uint4(0, 0, 0, 0);
    const int shift = (int)((uintptr_t)at & 15);
    const bool two = shift + valid > 16;
    const char *from = at - shift;
    uint32_t out[4] = {};
    if (from >= begin && from + (two ? 32 : 16) <= end) {
        const uint4 lo = __ldg(reinterpret_cast<const uint4 *>(from));
        const uint4 hi = two ? __ldg(reinterpret_cast<const uint4 *>(from) + 1) : make_uint4(0, 0, 0, 0);
        uint32_t w[9] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w, 0};
#pragma unroll
        for (int by = 2; by > 0; by >>= 1)
            if (shift & by * 4) {
#pragma unroll
                for (int i = 0; i + by < 9; ++i) w[i] = w[i + by];
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int keep = valid - i * 4;
            out[i] = __funnelshift_r(w[i], w[i + 1], shift % 4 * 8) & (keep >= 4 ? ~0u : keep <= 0 ? 0u : 0xffffu);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e * 2 < valid) out[e / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(at) + e) << (e % 2 * 16);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// fn(integral constant) for a tile of 1 to kFew tokens: with the count known to the compiler nothing stands between the loads, and all of
// a step are under way together.
template <typename Fn>
__device__ __forceinline__ void for_count(int count, Fn fn)
{
    static_assert(kFew == 4, "");
    if (count == 1) fn(std::integral_constant<int, 1>());
    else if (count == 2) fn(std::integral_constant<int, 2>());
    else if (count == 3) fn(std::integral_constant<int, 3>());
    else fn(std::integral_constant<int, 4>());
}

// Grid: (tiles, ceil(rank / 8)); a warp takes one component of v, its lanes 8 elements of K each in turn.
template <typename T, bool I8>
__global__ void __launch_bounds__(kFewThreads) adapter_few_shrink_kernel(const AdapterParams p)
{
    __shared__ alignas(16) SelfPlan plan;
    __shared__ int rows[kFew];
    const int tid = threadIdx.x, lane = tid & 31, j = (int)blockIdx.y * (kFewThreads / 32) + (tid >> 5);
    pdl_release();
    if (tid < 4 && blockIdx.x == 0 && blockIdx.y == 0) p.status[tid] = 0;
    const Tile tile = self_plan<kFew>(p, plan, rows);
    if (tile.count == 0 || tile.adapter < 0) return;
    if (j >= p.rank) {   // the components that the next kernel reads with the last ones
        if (lane < tile.count) p.v[(long long)rows[lane] * p.rank_pad + j] = 0.0f;
        return;
    }
    const uint4 *a = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(p.a) + ((long long)tile.adapter * p.rank + j) * p.k);
    for_count(tile.count, [&](auto tokens) {
        constexpr int C = decltype(tokens)::value, AHEAD = 4;
        using Pack = typename std::conditional<I8, uint2, uint4>::type;
        const Pack *x[C];
        f32x2 sum[C];
#pragma unroll
        for (int t = 0; t < C; ++t) {
            x[t] = reinterpret_cast<const Pack *>(reinterpret_cast<const char *>(p.x) + (long long)rows[t] * p.ld_x * (I8 ? 1 : 2));
            sum[t] = 0;
        }
        const int packs = p.k / 8;
        for (int c0 = lane; c0 < packs; c0 += 32 * AHEAD) {
            uint4 w[AHEAD];
            Pack xs[AHEAD][C];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {   // beyond the end: zeros
                const bool there = c0 + u * 32 < packs;
                w[u] = there ? __ldg(a + c0 + u * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int t = 0; t < C; ++t) xs[u][t] = there ? __ldg(x[t] + c0 + u * 32) : Pack{};
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (c0 + u * 32 >= packs) break;
                f32x2 f[4], g[4];
                unpack8<T>(w[u], f);
#pragma unroll
                for (int t = 0; t < C; ++t) {
                    if constexpr (I8) unpack8(xs[u][t], g);
                    else unpack8<T>(xs[u][t], g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[t] = fma2(f[e], g[e], sum[t]);
                }
            }
        }
        float v[C];
#pragma unroll
        for (int t = 0; t < C; ++t) {
            const float2 both = unpair2(sum[t]);
            v[t] = both.x + both.y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int t = 0; t < C; ++t) v[t] += __shfl_xor_sync(0xffffffffu, v[t], o);
        float mine = v[0];
#pragma unroll
        for (int t = 1; t < C; ++t) mine = lane == t ? v[t] : mine;
        if (lane < C) {
            const float by = p.scaling ? __ldg(p.scaling + tile.adapter) : 1.0f;
            p.v[(long long)rows[lane] * p.rank_pad + j] = __fmul_rn(mine, I8 ? __fmul_rn(by, __ldg(p.x_scale + rows[lane])) : by);
        }
    });
}

// Grid: (tiles, nsplit), channels in units of kFewChannels.  LANES neighbouring lanes (the power of two that holds rank / 8) share a
// channel's row of b, 8 components each, and add their sums up; of the tokens' results each then stores its share.  ANY: rows of b on any
// boundary.
constexpr int kFewChannels = 256;
template <typename T, int LANES, bool ANY>
__global__ void __launch_bounds__(kFewThreads) adapter_few_expand_kernel(const AdapterParams p)
{
    __shared__ alignas(16) SelfPlan plan;
    __shared__ int rows[kFew];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Tile tile = self_plan<kFew>(p, plan, rows);
    const int units = (p.n + kFewChannels - 1) / kFewChannels;
    const int n0 = (int)((long long)blockIdx.y * units / p.nsplit) * kFewChannels;
    const int n1 = min((int)((long long)(blockIdx.y + 1) * units / p.nsplit) * kFewChannels, p.n);
    if (tile.count == 0 || tile.adapter < 0) {
        if (tile.count > 0 && p.out != p.base) {
            if (p.grain_base == 16 && p.grain_out == 16 && p.n % 8 == 0) copy_base<T, 8, kFewThreads>(p, rows, tile.count, n0, n1);
            else copy_base<T, 1, kFewThreads>(p, rows, tile.count, n0, n1);
        }
        if (tile.count > 0) pdl_wait();   // as every CTA with a tile: the grid must not end before the one in front of it
        return;
    }
    constexpr int AHEAD = 4, ACROSS = 32 / LANES, STRIDE = kFewThreads / 32 * ACROSS;   // channels of a warp's step, of the CTA's
    const int part = lane % LANES;
    const bool mine = part * 8 < p.rank;
    const T *b = reinterpret_cast<const T *>(p.b) + (long long)tile.adapter * p.n * p.rank + part * 8;
    const T *base = reinterpret_cast<const T *>(p.base);
    T *out = reinterpret_cast<T *>(p.out);
    const char *b0 = reinterpret_cast<const char *>(p.b), *b1 = b0 + (long long)p.adapters * p.n * p.rank * 2;
    const int have = min(16, (p.rank - part * 8) * 2);   // bytes of a channel's row
    const auto at = [&](int c) { return reinterpret_cast<const char *>(b + (long long)c * p.rank); };
    int c = n0 + warp * ACROSS + lane / LANES;
    uint4 w[AHEAD];
    const auto fetch = [&](int u, int c) {
        if (ANY) w[u] = load_any(at(c), mine && c < n1 ? have : 0, b0, b1);
        else w[u] = mine && c < n1 ? __ldg(reinterpret_cast<const uint4 *>(at(c))) : make_uint4(0, 0, 0, 0);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) fetch(u, c + u * STRIDE);
    pdl_wait();   // v is complete
    for_count(tile.count, [&](auto tokens) {
        constexpr int C = decltype(tokens)::value, OWN = (C + LANES - 1) / LANES;   // tokens that a lane stores: part, part + LANES, ...
        f32x2 v[C][4];
#pragma unroll
        for (int t = 0; t < C; ++t) {
            const float4 *from = reinterpret_cast<const float4 *>(p.v + (long long)rows[t] * p.rank_pad + part * 8);
            const float4 q = mine ? __ldcg(from) : make_float4(0, 0, 0, 0), r = mine ? __ldcg(from + 1) : make_float4(0, 0, 0, 0);
            v[t][0] = pair2(q.x, q.y); v[t][1] = pair2(q.z, q.w); v[t][2] = pair2(r.x, r.y); v[t][3] = pair2(r.z, r.w);
        }
        long long base_row[OWN], out_row[OWN];
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            const int t = part + i * LANES;
            base_row[i] = t < C ? (long long)rows[t] * p.ld_base : -1;
            out_row[i] = t < C ? (long long)rows[t] * p.ld_out : -1;
        }
        T add[AHEAD][OWN];   // base, fetched a step ahead like b
        const auto fetch_base = [&](int c) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int i = 0; i < OWN; ++i)
                    if (base_row[i] >= 0 && c + u * STRIDE < n1) add[u][i] = base[base_row[i] + c + u * STRIDE];
        };
        fetch_base(c);
        for (; c - lane / LANES < n1; c += AHEAD * STRIDE) {   // the same for all lanes of a warp
            float to_add[AHEAD][OWN], sum[AHEAD][C];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int i = 0; i < OWN; ++i) to_add[u][i] = to_float(add[u][i]);
            fetch_base(c + AHEAD * STRIDE);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                f32x2 f[4];
                unpack8<T>(w[u], f);
                fetch(u, c + (u + AHEAD) * STRIDE);
#pragma unroll
                for (int t = 0; t < C; ++t) {
                    f32x2 s2 = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) s2 = fma2(f[e], v[t][e], s2);
                    const float2 both = unpair2(s2);
                    sum[u][t] = both.x + both.y;
                }
            }
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                    for (int t = 0; t < C; ++t) sum[u][t] += __shfl_xor_sync(0xffffffffu, sum[u][t], o);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
                for (int i = 0; i < OWN; ++i) {
                    float s = sum[u][i * LANES];
#pragma unroll
                    for (int t = i * LANES + 1; t < C && t < (i + 1) * LANES; ++t) s = part == t - i * LANES ? sum[u][t] : s;
                    if (out_row[i] >= 0 && c + u * STRIDE < n1) out[out_row[i] + c + u * STRIDE] = from_float<T>(__fadd_rn(to_add[u][i], s));
                }
            }
        }
    });
}

// ---------------------------------------------------------------------------------------------------------
// v = scaling * x a^T
// ---------------------------------------------------------------------------------------------------------

__host__ __device__ constexpr int align_up(int v, int a) { return (v + a - 1) / a * a; }
__host__ __device__ inline int tmem_cols(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }
// Bytes of a stage: the tokens' rows, the weights' (and the int8 rows as they come).
__host__ __device__ inline int shrink_stage(int tn, int rank_pad, bool i8) { return (tn + rank_pad) * kBlockK * 2 + (i8 ? tn * kBlockK : 0); }
// As many stages as fit a CTA of the large tiles alone on an SM, or one of two.
inline int shrink_stages(int tn, int rank_pad, bool i8)
{
    const int n = (tn > 64 ? 216 : 108) * 1024 / align_up(shrink_stage(tn, rank_pad, i8), 1024);
    return n < 3 ? 3 : n > kMaxStages ? kMaxStages : n;   // one that is read and kShrinkAhead under way
}
// The first product reads 128 rows from the start of a tile of tokens, however few there are: what lies behind it decides nothing but
// results that are not read.  The last stage's last tile may need some room behind it.
inline int shrink_smem(int tn, int rank_pad, bool i8)
{
    const int stage = align_up(shrink_stage(tn, rank_pad, i8), 1024), last = (kBlockTiles - 1) * tn * 128 + 128 * 128;
    return 1024 + (shrink_stages(tn, rank_pad, i8) - 1) * stage + (stage > last ? stage : last);
}

// Grid: tiles * ksplit, a tile's CTAs in a row: those of the places that no tile takes come last, so that they keep nobody waiting.  CTA s
// of a tile takes the K blocks [s * blocks / ksplit, (s + 1) * blocks / ksplit).
// FAST: rows of x and a start on 16-byte boundaries.  A thread then copies the same 16 bytes of every K block, whose addresses it works
// out once; with the addresses of every copy worked out anew the kernel was bound by its instructions.
// The products are issued by a warp of their own, which also orders them behind the copies (fence.proxy.async).  What bounds the kernel
// is that thread: a product of 128 x 64 x 16 costs it 0.05 us, a block's barriers and fence 0.27; so blocks are 128 deep.
template <typename T, bool I8, int TN, bool FAST>
__global__ void __launch_bounds__(kWorkers + 32) adapter_shrink_kernel(const AdapterParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(8) uint64_t full[kMaxStages], empty[kMaxStages], done;
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ int rows[TN];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool issuer = tid >= kWorkers;
    const uint32_t cols = tmem_cols(p.rank_pad);
    if (issuer) tmem_alloc(&tmem_base, cols);
    if (tid == 0) {
        for (int i = 0; i < kMaxStages; ++i) {
            mbar_init(smem_u32(&full[i]), kWorkers / 32);
            mbar_init(smem_u32(&empty[i]), 1);
        }
        mbar_init(smem_u32(&done), 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    pdl_wait();
    // Only now: the next kernel's CTAs wait for this grid with tensor memory in their hands, so every CTA of this one has its own first.
    __syncthreads();
    pdl_release();
    tc_fence_after();
    const int split = (int)(blockIdx.x % (unsigned)p.ksplit);
    const Tile tile = read_plan<TN>(p, (int)(blockIdx.x / (unsigned)p.ksplit), 1, kWorkers + 32, rows);
    const int blocks = (p.k + kBlockK - 1) / kBlockK;
    const int kb0 = (int)((long long)split * blocks / p.ksplit), kb1 = (int)((long long)(split + 1) * blocks / p.ksplit);
    const bool work = tile.count > 0 && tile.adapter >= 0;   // kb0 < kb1, since ksplit is at most blocks
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t stage_bytes = align_up(shrink_stage(TN, p.rank_pad, I8), 1024), a_tile = TN * kBlockK * 2;
    if (work && issuer) {
        const uint32_t idesc = instr_desc<T>(p.rank_pad);
        int stage = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            const uint32_t s = smem0 + (uint32_t)stage * stage_bytes;
            mbar_wait(smem_u32(&full[stage]), phase, &gave_up, p, 900);
            fence_async_proxy();
            tc_fence_after();
            if (lane == 0) {
                const uint64_t xd = operand_desc(s), ad = operand_desc(s + a_tile);
                const uint32_t x_next = TN * 128 / 16, a_next = (uint32_t)p.rank_pad * 128 / 16;
                if (p.k - kb * kBlockK >= kBlockK) {
#pragma unroll
                    for (int j = 0; j < kBlockK / 16; ++j)
                        umma_f16(tmem_base, xd + (j / 4 * x_next + j % 4 * 2), ad + (j / 4 * a_next + j % 4 * 2), idesc, j > 0 || kb > kb0);
                } else {
                    const int steps = (p.k - kb * kBlockK + 15) / 16;
                    for (int j = 0; j < steps; ++j)
                        umma_f16(tmem_base, xd + (j / 4 * x_next + j % 4 * 2), ad + (j / 4 * a_next + j % 4 * 2), idesc, j > 0 || kb > kb0);
                }
                umma_commit(smem_u32(&empty[stage]));
                if (kb == kb1 - 1) umma_commit(smem_u32(&done));
            }
            __syncwarp();
            if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
    } else if (work) {
        constexpr int XB = I8 ? 1 : 2;
        const char *x = reinterpret_cast<const char *>(p.x);
        const char *a = reinterpret_cast<const char *>(p.a) + (long long)tile.adapter * p.rank * p.k * 2;
        const uint32_t raw_tile = (uint32_t)(TN + p.rank_pad) * kBlockK * 2;
        // copies per token row of a K block, and rows apart of a thread's copies: a multiple of 8, so their places differ by that many rows
        constexpr int XC = kBlockK * XB / 16, X_ROWS = kWorkers / XC, AC = kBlockK * 2 / 16, A_ROWS = kWorkers / AC;
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
        const auto load = [&](int kb, int stage) {
            const uint32_t s = smem0 + (uint32_t)stage * stage_bytes;
            const int have = min(kBlockK, p.k - kb * kBlockK);
            if constexpr (FAST) {
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
            } else {
                for (int at = 0; at < kBlockTiles; ++at) {
                    const long long k0 = (long long)kb * kBlockK + at * 64;
                    if (at * 64 >= (have + 15) / 16 * 16) break;   // no K step reaches the tile
                    copy_rows<true, kWorkers>(p.grain_a, s + a_tile + (uint32_t)(at * p.rank_pad * 128), p.rank, 128, (have - at * 64) * 2,
                                              [&](int r) { return a + ((long long)r * p.k + k0) * 2; });
                    if (!I8)
                        copy_rows<true, kWorkers>(p.grain_x, s + (uint32_t)(at * TN * 128), tile.count, 128, (have - at * 64) * 2,
                                                  [&](int r) { return x + ((long long)rows[r] * p.ld_x + k0) * XB; });
                }
                if (I8)
                    copy_rows<false, kWorkers>(p.grain_x, s + raw_tile, tile.count, kBlockK, have,
                                               [&](int r) { return x + (long long)rows[r] * p.ld_x + (long long)kb * kBlockK; });
            }
        };
        // A warp's copies of block i have landed when those of the kShrinkAhead blocks behind it are all that its threads have under way;
        // one lane says so.
        const auto landed = [&](int stage, bool say) {
            const uint32_t s = smem0 + (uint32_t)stage * stage_bytes;
            if (I8 && FAST) widen_rows_grain<T, 16, kWorkers>(s + raw_tile, s, TN * 128, tile.count);
            else if (I8) widen_rows<T, kWorkers>(p.grain_x, s + raw_tile, s, TN * 128, tile.count);
            __syncwarp();
            if (lane == 0 && say) mbar_arrive(smem_u32(&full[stage]));
        };
        const int n = kb1 - kb0;
        int stage = 0, behind = 0;
        uint32_t phase = 1;   // a stage is free at first
        for (int i = 0; i < n + kShrinkAhead; ++i) {
            if (i < n) {
                mbar_wait(smem_u32(&empty[stage]), phase, &gave_up, p, 901);
                load(kb0 + i, stage);
                if (++stage == p.stages) { stage = 0; phase ^= 1; }
            }
            cp_commit();
            if (i >= kShrinkAhead) {
                cp_wait<kShrinkAhead>();
                landed(behind, i - kShrinkAhead < n - p.skip_blocks);
                if (++behind == p.stages) behind = 0;
            }
        }
    }
    if (work) {
        mbar_wait<true>(smem_u32(&done), 0, &gave_up, p, 902);
        tc_fence_after();
        const int quarter = warp % 4, half = p.rank_pad / 2, slot = quarter * 32 + lane;
        if (!issuer && quarter * 32 < TN) {   // warp w: 32 tokens (w % 4) and half of the columns (w / 4)
            const bool live = slot < tile.count;
            const int row = live ? rows[slot] : 0;
            float f = p.scaling ? __ldg(p.scaling + tile.adapter) : 1.0f;
            if (I8 && live) f = __fmul_rn(f, __ldg(p.x_scale + row));
            float4 *v = reinterpret_cast<float4 *>(p.v + ((long long)split * p.rows + row) * p.rank_pad);
            for (int c = warp / 4 * half; c < (warp / 4 + 1) * half; c += 8) {
                uint32_t d[8];
                tmem_ld8(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c, d);
                tmem_ld_wait();
                if (live) {
#pragma unroll
                    for (int e = 0; e < 8; e += 4)
                        v[(c + e) / 4] = make_float4(__fmul_rn(__uint_as_float(d[e]), f), __fmul_rn(__uint_as_float(d[e + 1]), f),
                                                     __fmul_rn(__uint_as_float(d[e + 2]), f), __fmul_rn(__uint_as_float(d[e + 3]), f));
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (issuer) {
        tc_fence_after();
        tmem_dealloc(tmem_base, cols);
    }
}

// ---------------------------------------------------------------------------------------------------------
// out = base + v b^T
// ---------------------------------------------------------------------------------------------------------

constexpr int kParts = 3;   // 16-bit parts of a component of v
__host__ __device__ inline int rank_atoms(int rank_pad) { return rank_pad > 64 ? 2 : 1; }
__host__ __device__ inline int expand_stage(int tn, int rank_pad) { return rank_atoms(rank_pad) * kChunkN * 128 + tn * kChunkN * 2; }
inline int expand_smem(int tn, int rank_pad) { return 1024 + kParts * rank_atoms(rank_pad) * tn * 128 + kExpandStages * expand_stage(tn, rank_pad); }

// Grid: tiles * nsplit, as above.  CTA s of a tile takes the channel chunks [s * chunks / nsplit, (s + 1) * chunks / nsplit).
// GB 16: rows of b, base and out on 16-byte boundaries; addresses are worked out once, and results go back through the chunk's base rows in
// shared memory, from which they are stored 16 bytes at a time.  2: the same with rows of b on any boundary, by way of registers (rank 61
// beside 64, 3000 tokens: 44 us and 35; element by element, as with 0, 64).  0: any strides.
template <typename T, int TN, int GB>
__global__ void __launch_bounds__(expand_workers(TN) + 32, TN == 64 ? 2 : 1) adapter_expand_kernel(const AdapterParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(8) uint64_t full[kExpandStages], acc_full[2], acc_empty[2], v_full;
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ int rows[TN];
    __shared__ float unscale[TN];          // fp16: the power of two that v was divided by
    constexpr bool F16 = std::is_same<T, __half>::value;
    constexpr uint32_t COLS = 2 * TN <= 32 ? 32 : 2 * TN;   // two buffers of accumulators
    constexpr int WORKERS = expand_workers(TN), THREADS = WORKERS + 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool issuer = tid >= WORKERS;
    if (issuer) tmem_alloc(&tmem_base, COLS);
    if (tid == 0) {
        for (int i = 0; i < kExpandStages; ++i) mbar_init(smem_u32(&full[i]), GB == 2 ? 2 * WORKERS : WORKERS);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), WORKERS / 32);
        }
        mbar_init(smem_u32(&v_full), WORKERS / 32);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int split = (int)(blockIdx.x % (unsigned)p.nsplit);
    const Tile tile = read_plan<TN>(p, (int)(blockIdx.x / (unsigned)p.nsplit), p.parts, THREADS, rows);
    const int chunks = (p.n + kChunkN - 1) / kChunkN;
    const int c0 = (int)((long long)split * chunks / p.nsplit), c1 = (int)((long long)(split + 1) * chunks / p.nsplit);
    const T *base = reinterpret_cast<const T *>(p.base);
    T *out = reinterpret_cast<T *>(p.out);
    if (tile.count > 0 && tile.adapter < 0) {
        if (p.out != p.base) {
            pdl_wait();
            copy_base<T, GB ? 8 : 1, THREADS>(p, rows, tile.count, c0 * kChunkN, min(c1 * kChunkN, p.n));
        }
    } else if (tile.count > 0 && c0 < c1) {
        const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
        const int atoms = rank_atoms(p.rank_pad);
        const uint32_t v_part = (uint32_t)(atoms * TN * 128), stage0 = smem0 + kParts * v_part;   // the parts of v, one behind the other
        const uint32_t stage_bytes = expand_stage(TN, p.rank_pad), base_at = (uint32_t)(atoms * kChunkN * 128);
        const char *b = reinterpret_cast<const char *>(p.b) + (long long)tile.adapter * p.n * p.rank * 2;
        // b: the copies of a chunk, offset in its rows << 8 | bytes, and place in the tile
        constexpr int NB = 16 * kChunkN / WORKERS, NR = TN * 16 / WORKERS;
        const int per_row = p.rank_pad / 8, nb = (per_row * kChunkN + WORKERS - 1) / WORKERS;
        uint32_t b_from[NB], b_to[NB];
        long long base_at_row[NR], out_at_row[NR];
        const int rc = (tid % 16) * 8;
        if (GB && !issuer) {
            const float across = 1.0f / (float)per_row;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                if (i >= nb) break;
                const int idx = tid + i * WORKERS, r = (int)(((float)idx + 0.5f) * across), byte = (idx - r * per_row) * 16;   // exact for idx < 2^12
                const int valid = min(max(p.rank * 2 - byte, 0), 16);
                // one too many lies behind every chunk's end
                b_from[i] = idx < per_row * kChunkN ? (uint32_t)(r * p.rank * 2 + (valid ? byte : 0)) << 8 | (uint32_t)valid : ~0u;
                b_to[i] = (uint32_t)(byte / 128 * kChunkN * 128) + swizzled(r, byte % 128);
            }
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int r = tid / 16 + i * (WORKERS / 16);
                base_at_row[i] = r < tile.count ? (long long)rows[r] * p.ld_base + rc : -1;
                out_at_row[i] = r < tile.count ? (long long)rows[r] * p.ld_out + rc : -1;
            }
        }
        const auto load = [&](int c) {
            const uint32_t s = stage0 + (uint32_t)((c - c0) % kExpandStages) * stage_bytes;
            const int n0 = c * kChunkN, channels = min(kChunkN, p.n - n0);
            if constexpr (GB != 0) {
                const char *from = b + (long long)n0 * p.rank * 2;
                const uint32_t end = (uint32_t)(channels * p.rank * 2);
                const char *b0 = reinterpret_cast<const char *>(p.b), *b1 = b0 + (long long)p.adapters * p.n * p.rank * 2;
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    if (i >= nb) break;
                    if (b_from[i] >> 8 >= end) continue;
                    if constexpr (GB == 2) {
                        const uint4 w = load_any(from + (b_from[i] >> 8), (int)(b_from[i] & 255u), b0, b1);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(s + b_to[i]), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
                    } else cp_async<16>(s + b_to[i], from + (b_from[i] >> 8), (int)(b_from[i] & 255u));
                }
#pragma unroll
                for (int i = 0; i < NR; ++i)
                    if (base_at_row[i] >= 0 && rc < channels)
                        cp_async<16>(s + base_at + (uint32_t)((tid + i * WORKERS) * 16), base + base_at_row[i] + n0, 16);
            } else {
                for (int at = 0; at < atoms; ++at) {
                    const int left = p.rank_pad - at * 64;                       // a whole number of K steps, zero beyond the rank
                    const int width = left > 32 ? 128 : left > 16 ? 64 : 32;
                    copy_rows<true, WORKERS>(p.grain_b, s + (uint32_t)at * kChunkN * 128, channels, width, (p.rank - at * 64) * 2,
                                                    [&](int r) { return b + ((long long)(n0 + r) * p.rank + at * 64) * 2; });
                }
                copy_rows<false, WORKERS>(p.grain_base, s + base_at, tile.count, kChunkN * 2, channels * 2,
                                                 [&](int r) { return reinterpret_cast<const char *>(base + (long long)rows[r] * p.ld_base + n0); });
            }
        };
        if (issuer) {
            pdl_wait();
            const uint32_t idesc = instr_desc<T>(TN);
            mbar_wait(smem_u32(&v_full), 0, &gave_up, p, 910);
            for (int c = c0; c < c1; ++c) {
                const int i = c - c0, buf = i & 1;
                const uint32_t s = stage0 + (uint32_t)(i % kExpandStages) * stage_bytes, d = tmem_base + (uint32_t)(buf * TN);
                mbar_wait(smem_u32(&full[i % kExpandStages]), (i / kExpandStages) & 1, &gave_up, p, 911);
                if (i >= 2) mbar_wait(smem_u32(&acc_empty[buf]), (i / 2 - 1) & 1, &gave_up, p, 912);
                fence_async_proxy();
                tc_fence_after();
                if (lane == 0) {
                    uint32_t more = 0;
                    for (int j = 0; j < p.rank_pad / 16; ++j) {
                        const uint64_t bd = operand_desc(s + (uint32_t)(j / 4) * kChunkN * 128) + (j % 4) * 2;
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            umma_f16(d, bd, operand_desc(smem0 + part * v_part + (uint32_t)(j / 4) * TN * 128) + (j % 4) * 2, idesc, more);
                            more = 1;
                        }
                    }
                    umma_commit(smem_u32(&acc_full[buf]));
                }
                __syncwarp();
            }
            // all products are done, also where the others have given up
            mbar_wait<true>(smem_u32(&acc_full[(c1 - 1 - c0) & 1]), ((c1 - 1 - c0) / 2) & 1, &gave_up, p, 915);
        } else {
            // Copies through shared memory by whole 16 bytes announce themselves; others are waited for, a chunk ahead.
            const auto announce = [&](int c) {
                if (GB) mbar_arrive_copies(smem_u32(&full[(c - c0) % kExpandStages]));
                if (GB == 2) mbar_arrive(smem_u32(&full[(c - c0) % kExpandStages]));
            };
            const auto landed = [&](int c) {
                if (GB) return;
                cp_wait<0>();
                mbar_arrive(smem_u32(&full[(c - c0) % kExpandStages]));
            };
            load(c0);
            announce(c0);
            if (GB && c0 + 1 < c1) {
                load(c0 + 1);
                announce(c0 + 1);
            }
            pdl_wait();   // v is complete
            {
                constexpr int LANES = WORKERS / TN, CH = 16 / LANES;   // threads of a token, and groups of 8 components of each
                const int slot = tid / LANES, part = tid % LANES;
                const bool live = slot < tile.count;
                const int row = live ? rows[slot] : 0;
                float f[CH][8];
#pragma unroll
                for (int h = 0; h < CH; ++h)
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[h][e] = 0.0f;
                const float4 *v = reinterpret_cast<const float4 *>(p.v + (long long)row * p.rank_pad);
                const long long split = (long long)p.rows * p.rank_pad / 4;
                if (live) {
                    constexpr int AT_ONCE = 4;   // partial sums that are fetched together; they are added in the order of the splits
                    for (int s0 = 0; s0 < p.ksplit; s0 += AT_ONCE) {
#pragma unroll
                        for (int h = 0; h < CH; ++h) {
                            const int j = (part + h * LANES) * 8;
                            if (j >= p.rank_pad) break;
                            float4 q[AT_ONCE][2];
#pragma unroll
                            for (int s = 0; s < AT_ONCE; ++s) {
                                const bool there = s0 + s < p.ksplit;
                                q[s][0] = there ? __ldcg(v + (s0 + s) * split + j / 4) : make_float4(0, 0, 0, 0);
                                q[s][1] = there ? __ldcg(v + (s0 + s) * split + j / 4 + 1) : make_float4(0, 0, 0, 0);
                            }
#pragma unroll
                            for (int s = 0; s < AT_ONCE; ++s) {
                                f[h][0] += q[s][0].x; f[h][1] += q[s][0].y; f[h][2] += q[s][0].z; f[h][3] += q[s][0].w;
                                f[h][4] += q[s][1].x; f[h][5] += q[s][1].y; f[h][6] += q[s][1].z; f[h][7] += q[s][1].w;
                            }
                        }
                    }
#pragma unroll
                    for (int h = 0; h < CH; ++h)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if ((part + h * LANES) * 8 + e >= p.rank) f[h][e] = 0.0f;   // the K steps end in zeros
                }
                float down = 1.0f;
                if (F16) {
                    uint32_t m = 0;
#pragma unroll
                    for (int h = 0; h < CH; ++h)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t mag = __float_as_uint(f[h][e]) & 0x7fffffffu;
                            m = max(m, mag < 0x7f800000u ? mag : 0u);   // infinities and NaN stay what they are
                        }
#pragma unroll
                    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                    // 2^(14 - e) for a largest value in [2^e, 2^(e+1)); none where all are so small that no result sees them
                    const int e = (int)(m >> 23) - 127;
                    const bool shift = e > -112;
                    down = shift ? __uint_as_float((uint32_t)(127 + 14 - e) << 23) : 1.0f;
                    if (part == 0) unscale[slot] = shift ? __uint_as_float((uint32_t)(127 - 14 + e) << 23) : 1.0f;
                }
#pragma unroll
                for (int h = 0; h < CH; ++h) {
                    const int j = (part + h * LANES) * 8;
                    if (j >= p.rank_pad) break;
                    if (F16) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[h][e] = __fmul_rn(f[h][e], down);
                    }
                    uint32_t at = smem0 + (uint32_t)(j / 64 * TN * 128) + swizzled(slot, (j % 64) * 2);
#pragma unroll
                    for (int q = 0; q < kParts; ++q, at += v_part) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = pack2<T>(f[h][2 * e], f[h][2 * e + 1]);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
#pragma unroll
                        for (int e = 0; e < 8; ++e) {   // the rest, which is exact; an infinity less itself is none
                            const float taken = to_float(from_float<T>(f[h][e]));
                            f[h][e] = isinf(taken) ? 0.0f : __fsub_rn(f[h][e], taken);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&v_full));
                if (F16) worker_sync<WORKERS>();   // unscale
            }
            cp_commit();
            landed(c0);
            if (!GB && c0 + 1 < c1) {
                load(c0 + 1);
                cp_commit();
            }
            // warp w: channels 32 (w % 4) + lane, its share of the tokens
            constexpr int SHARE = TN * 128 / WORKERS;
            const int q = warp & 3, ch = q * 32 + lane, first = (warp >> 2) * SHARE;
            for (int c = c0; c < c1; ++c) {
                const int i = c - c0, buf = i & 1, n = c * kChunkN + ch;
                const uint32_t s = stage0 + (uint32_t)(i % kExpandStages) * stage_bytes;
                if (c + 1 < c1) landed(c + 1);
                mbar_wait(smem_u32(&full[i % kExpandStages]), (i / kExpandStages) & 1, &gave_up, p, 913);   // base, copied by others
                mbar_wait(smem_u32(&acc_full[buf]), (i / 2) & 1, &gave_up, p, 914);
                tc_fence_after();
                uint32_t d[SHARE];
                if (first < tile.count) {
#pragma unroll
                    for (int t0 = 0; t0 < SHARE; t0 += 8) tmem_ld8(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * TN + first + t0), d + t0);
                    tmem_ld_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&acc_empty[buf]));
                const uint32_t at = s + base_at + (uint32_t)(first * kChunkN * 2 + ch * 2);
#pragma unroll
                for (int t0 = 0; t0 < SHARE; t0 += 8) {
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
                worker_sync<WORKERS>();   // this chunk's results are in place, and its base rows have been read
                if (GB) {   // a thread stores the 16 bytes whose place it then fills again
#pragma unroll
                    for (int j = 0; j < NR; ++j) {
                        if (out_at_row[j] >= 0 && c * kChunkN + rc < p.n) {
                            uint4 o;
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(o.x), "=r"(o.y), "=r"(o.z), "=r"(o.w)
                                         : "r"(s + base_at + (uint32_t)((tid + j * WORKERS) * 16)) : "memory");
                            *reinterpret_cast<uint4 *>(out + out_at_row[j] + c * kChunkN) = o;
                        }
                    }
                }
                if (c + kExpandStages < c1) {
                    load(c + kExpandStages);
                    announce(c + kExpandStages);
                    cp_commit();
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");   // none is left unless a wait ran out
        }
    }
    // This grid must not end before the kernels in front of it: the stream goes on behind it alone.  The CTAs without a tile leave their
    // places at once, to those that found none yet.
    if (tile.count > 0) pdl_wait();
    __syncthreads();
    if (issuer) tmem_dealloc(tmem_base, COLS);
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
    cfg.attrs = attr;
    if (dependent) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

constexpr size_t align256(size_t v) { return (v + 255) / 256 * 256; }

int grain_of(const void *base, long long pitch_bytes, int smallest)
{
    const uintptr_t v = (uintptr_t)base | (uintptr_t)pitch_bytes;
    return v % 16 == 0 ? 16 : v % 8 == 0 ? 8 : v % 4 == 0 ? 4 : smallest;
}

struct Shape {
    int tile_tokens, tiles, ksplit, nsplit, rank_pad;
    bool few;
};

// On the CUDA cores, in tiles of 4 tokens: up to kSelfPlan tokens while all tiles together read no more than `limit` elements of weights,
// if rows of x and a start on packs (others, with two loads and a shift a pack: 200 tokens, 1500 -> 4096, 22 us, 16 on the tensor cores).
// They read them anew for every tile, at about 10 us per 10 million elements beyond the first 5; the tensor cores' way reads them once,
// but takes a third kernel and some 0.3 us per adapter.  2048 -> 2048, rank 16: 16 tokens of 4 adapters 6.5 us and 10.6, 128 of 128 8.7
// and 21; 4096 -> 4096, rank 64: 32 of 8 12.9 and 16.3, 64 of 8 18.0 and 17.9, 128 of 8 27 and 19, 128 of 128 40 and 40.
//
// Else tiles of 16 tokens, of 64 where adapters have more than 16 on average (2000 of 4 adapters 21 us, 31 with tiles of 16; 128 of 64 29,
// 36 with tiles of 64) or, where they have 128 and there are enough tiles for the SMs, of 128 (4096 of 8 49.7, 51.9 with tiles of 64; up to
// rank 64, for the sake of three stages): the first product reads 128 rows of the tokens' tile whether they are tokens or not.  `tiles` is
// the most there can be: full ones, and one that is not for every adapter and for none; a tile on the CUDA cores may begin with any token.
// K and N are split for four of the first kernel's small CTAs on an SM, two of the next size, one large, and two of the second kernel's.  By
// their shared memory three small ones fit at rank 16, two at higher ranks (one with int8 rows of rank 128); of the next size two up to rank
// 80 (48 with int8 rows), then one; of the second kernel's two up to rank 64, then one with tiles of 64.  What does not fit comes in a second
// turn.  Rows that are not copied 16 bytes at a time take longer, so K is split further there (300 tokens, 1001 -> 3001: 22 us, 29 with four
// splits).  The tensor cores' figures here were taken with two parts of v; the third adds 1 to 4 % to all of them.
Shape shape_of(const AdapterProblem &p, bool may_be_few)
{
    Shape s;
    const long long groups = p.adapters < p.rows ? p.adapters : p.rows, partial = p.adapters + 1 < p.rows ? p.adapters + 1 : p.rows;
    const long long fours = p.rows / kFew + groups / 2 < p.rows ? p.rows / kFew + groups / 2 : p.rows;   // tiles of four, about
    const long long limit = 5000000 + 400000 * groups < 35000000 ? 5000000 + 400000 * groups : 35000000;
    s.few = may_be_few && p.rows <= kSelfPlan && fours * p.rank * (p.k + p.n) <= limit;
    s.tile_tokens = s.few ? kFew : p.rows >= 2048 && p.rows >= 128 * groups && p.rank <= 64 ? 128 : p.rows > 16 * groups ? 64 : 16;
    s.tiles = (int)(p.rows / s.tile_tokens + partial);
    if (s.few || s.tiles > p.rows) s.tiles = (int)p.rows;
    s.rank_pad = align_up((int)p.rank, 16);
    const int per_sm = s.tile_tokens == 16 ? 4 : s.tile_tokens == 64 ? 2 : 1;
    const int likely = (int)(p.rows / s.tile_tokens + partial / 2) > 0 ? (int)(p.rows / s.tile_tokens + partial / 2) : 1;
    const int blocks = (int)((p.k + kBlockK - 1) / kBlockK), chunks = (int)((p.n + kChunkN - 1) / kChunkN);
    s.ksplit = 1;
    while (s.ksplit < (p.k % 8 ? 8 : 4) && 2 * s.ksplit * likely <= per_sm * 148 && 2 * s.ksplit <= blocks) s.ksplit *= 2;
    const int want = 2 * 148 / (s.tile_tokens == 128 ? 2 * likely : likely);
    const int per = want > 0 ? (chunks + want - 1) / want : chunks;
    s.nsplit = (chunks + per - 1) / per;   // no more CTAs than the most chunks of one make necessary
    if (s.few) {
        const int units = (int)((p.n + kFewChannels - 1) / kFewChannels), places = kFewExpandCtas * 148 / (int)(fours > 0 ? fours : 1);
        s.ksplit = 1;
        s.nsplit = places < units ? places : units;   // one wave: every CTA looks for its tile first
    }
    if (s.nsplit < 1) s.nsplit = 1;
    return s;
}

template <typename T, bool I8, int TN>   // TN: tokens of the first kernel's tiles; the second one's have at most 64
cudaError_t launch_tiles(const AdapterParams &p, const Shape &s, cudaStream_t stream)
{
    cudaError_t e = launch_kernel(adapter_plan_kernel, dim3(1), kPlanThreads, (p.adapters + 1) * 4, stream, false, p, s.tile_tokens);
    if (e != cudaSuccess) return e;
    const auto shrink = p.grain_x == 16 && p.grain_a == 16 ? adapter_shrink_kernel<T, I8, TN, true> : adapter_shrink_kernel<T, I8, TN, false>;
    e = launch_kernel(shrink, dim3((unsigned)s.tiles * (unsigned)s.ksplit), kWorkers + 32, shrink_smem(TN, s.rank_pad, I8), stream, true, p);
    if (e != cudaSuccess) return e;
    const bool rows16 = p.grain_base == 16 && p.grain_out == 16 && p.n % 8 == 0;
    constexpr int EN = TN < 64 ? TN : 64;
    const auto expand = rows16 && p.grain_b == 16 ? adapter_expand_kernel<T, EN, 16>
                        : rows16 ? adapter_expand_kernel<T, EN, 2> : adapter_expand_kernel<T, EN, 0>;
    return launch_kernel(expand, dim3((unsigned)(s.tiles * p.parts) * (unsigned)s.nsplit), expand_workers(EN) + 32, expand_smem(EN, s.rank_pad), stream, true, p);
}

template <typename T, bool ANY>
cudaError_t launch_few_expand(const AdapterParams &p, const Shape &s, cudaStream_t stream)
{
    const auto expand = p.rank <= 8 ? adapter_few_expand_kernel<T, 1, ANY> : p.rank <= 16 ? adapter_few_expand_kernel<T, 2, ANY>
                        : p.rank <= 32 ? adapter_few_expand_kernel<T, 4, ANY> : p.rank <= 64 ? adapter_few_expand_kernel<T, 8, ANY> : adapter_few_expand_kernel<T, 16, ANY>;
    return launch_kernel(expand, dim3((unsigned)s.tiles, (unsigned)s.nsplit), kFewThreads, 0, stream, true, p);
}

template <typename T, bool I8>
cudaError_t launch_typed(const AdapterParams &p, const Shape &s, cudaStream_t stream)
{
    if (s.few) {
        const cudaError_t e = launch_kernel(adapter_few_shrink_kernel<T, I8>, dim3((unsigned)s.tiles, (unsigned)((p.rank + 7) / 8)), kFewThreads, 0, stream, false, p);
        if (e != cudaSuccess) return e;
        return p.grain_b == 16 ? launch_few_expand<T, false>(p, s, stream) : launch_few_expand<T, true>(p, s, stream);
    }
    return s.tile_tokens == 16 ? launch_tiles<T, I8, 16>(p, s, stream)
           : s.tile_tokens == 64 ? launch_tiles<T, I8, 64>(p, s, stream) : launch_tiles<T, I8, 128>(p, s, stream);
}

}  // namespace

size_t adapter_workspace_bytes(const AdapterProblem &p)
{
    // which kernels take the call hangs on the addresses that it is run with
    size_t most = 0;
    for (const bool few : {false, true}) {
        const Shape s = shape_of(p, few);
        const size_t bytes = 256 + (s.few ? 0 : 256 + align256((size_t)s.tiles * sizeof(int2)) + align256((size_t)s.tiles * s.tile_tokens * 4)) +
                             align256((size_t)s.ksplit * (size_t)p.rows * (size_t)s.rank_pad * 4);
        if (bytes > most) most = bytes;
    }
    return most;
}

cudaError_t adapter_launch(const AdapterProblem &a, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (a.rows <= 0) return cudaSuccess;
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < adapter_workspace_bytes(a)) return cudaErrorInvalidValue;
    const Shape s = shape_of(a, grain_of(a.x, a.ld_x * (a.x_i8 ? 1 : 2), 1) >= (a.x_i8 ? 8 : 16) && grain_of(a.a, a.k * 2, 1) == 16);
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
    p.wait_limit = a.opt.wait_limit_cycles > 0 ? a.opt.wait_limit_cycles : kWaitLimitCycles;
    p.skip_blocks = a.opt.test_skip_k_blocks;
    p.ksplit = s.ksplit; p.nsplit = s.nsplit; p.parts = s.tile_tokens > 64 ? s.tile_tokens / 64 : 1;
    char *ws = static_cast<char *>(workspace);
    p.status = reinterpret_cast<int *>(ws);
    ws += 256;
    p.n_tiles = nullptr; p.tiles = nullptr; p.order = nullptr;
    if (!s.few) {
        p.n_tiles = reinterpret_cast<int *>(ws); ws += 256;
        p.tiles = reinterpret_cast<int2 *>(ws); ws += align256((size_t)s.tiles * sizeof(int2));
        p.order = reinterpret_cast<int *>(ws); ws += align256((size_t)s.tiles * s.tile_tokens * 4);
    }
    p.v = reinterpret_cast<float *>(ws);
    p.stages = shrink_stages(s.tile_tokens, s.rank_pad, a.x_i8);
    if (a.dtype == kF16) return a.x_i8 ? launch_typed<__half, true>(p, s, stream) : launch_typed<__half, false>(p, s, stream);
    return a.x_i8 ? launch_typed<__nv_bfloat16, true>(p, s, stream) : launch_typed<__nv_bfloat16, false>(p, s, stream);
}

}  // namespace gmm
