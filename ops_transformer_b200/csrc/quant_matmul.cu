// quant_matmul: y = ((x w) * scale) * per_token_scale + bias of int8 matrices, without groups.
//
// Orientation as in gmm_sm100.cu: weight channels are the M side of the MMA (128 per CTA, a TMEM lane each), tokens its N side, up to 256.
// What a few tokens cost is the weights' way from memory, so K is split over the CTAs of a cluster until all SMs read: each accumulates its
// part of K in TMEM and finishes an equal share of the tile's tokens, for which the others send it their int32 sums, into its shared memory:
// word by word as they leave TMEM where a tile has few tokens, else as one copy each from where the rows of sums were laid down.  Integer
// sums are exact in any order, so there is nothing to put in sequence and no workspace for it.
//
// Measured, us: 16 x 768 -> 2048 3.7, 16 x 7168 -> 4096 9.7 (29 MB, 3.0 TB/s: a third of it is the launch, the first bytes' way and the
// sums'), 128 tokens of it 11.4, 256 13.8, 1024 26.0, 1024 x 2048 -> 2048 8.8, 611 x 1424 -> 2976 8.4.  A CTA has one tile, so that the first
// bytes' way, the K blocks and the end follow one another: with 100 to 600 tokens memory or the tensor cores would take a fifth to three
// fifths of these times.  From about 2000 tokens of 7168 on the persistent kernel of the grouped product (two SMs a tile,
// epilogue beside the next tile's MMAs) is faster, and takes the call: 4096 tokens 78 against 95, of the 77 that the tensor cores take at
// twice the 16-bit rate.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "dependent.h"
#include "gmm_common.h"

namespace gmm {
namespace {

constexpr int kChannels = 128, kBlockK = 128, kMaxTokens = 256;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxStages = 10, kMaxSplit = 8, kSms = 148;
constexpr uint32_t kWeightStage = kChannels * kBlockK, kTokenBytes = kChannels * 4;   // of a K block's weights, of a token's sums
template <int N> struct Int { static constexpr int value = N; };
template <bool B> struct Flag { static constexpr bool value = B; };
constexpr long long kWaitLimitCycles = 1ll << 31, kDrainLimitCycles = 1ll << 24;   // about a second, a few milliseconds

struct MatmulParams {
    const void *scale, *bias;
    int scale_dtype, bias_dtype;
    const float *token_scale;
    void *y;
    long long ld_y;
    int m, k, n;
    int tile_tokens, token_tiles;   // tokens of a tile, a multiple of 32; tiles along them
    int split, stages;
    uint32_t parts_at;              // sums of the cluster's other CTAs: behind the ring, or in its place behind this CTA's own
    bool apart;                     // behind the ring, this CTA's own among them
    bool packs;                     // four results of a row can be stored at once
    long long wait_limit;
    int skip_blocks;                // test only: K blocks that the producer leaves out
    int *status;
    bool clear_status;              // else it has been, before the launch
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t *bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// CLUSTER: for what other CTAs have sent.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_try(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    if (CLUSTER) asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    else asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait; false when it ran out, which the status says, or when another one of the CTA has.
template <bool CLUSTER>
__device__ __noinline__ bool mbar_wait_slow(uint64_t *bar, uint32_t parity, volatile int *gave_up, const MatmulParams &p, int role)
{
    const long long t0 = clock64();
    while (!mbar_try<CLUSTER>(bar, parity)) {
        if (*gave_up) return false;
        if (clock64() - t0 > p.wait_limit) {
            *gave_up = 1;
            if (atomicCAS(p.status, kStatusOk, kStatusWaitTimeout) == kStatusOk) {
                p.status[1] = (int)blockIdx.x;
                p.status[2] = role;
                p.status[3] = (int)parity;
            }
            return false;
        }
    }
    return true;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, volatile int *gave_up, const MatmulParams &p, int role)
{
    return mbar_try<CLUSTER>(bar, parity) || mbar_wait_slow<CLUSTER>(bar, parity, gave_up, p, role);
}
// Behind a wait that ran out: what is under way has to land before this CTA's memory is another's.
__device__ __forceinline__ void drain(uint64_t *bar, uint32_t parity)
{
    const long long begin = clock64();
    while (!mbar_try(bar, parity) && clock64() - begin < kDrainLimitCycles) {}
}
// One lane of a converged warp: copies and MMAs issued under this predicate cost a few cycles each, in a branch that one thread enters 150.
__device__ __forceinline__ bool elect_one()
{
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
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
// Operand descriptors, 128-byte swizzle: rows of 128 K-bytes in groups of 8 (tokens, weights stored [n, k]), or 128 channels of one K row,
// 8 K rows 1024 bytes on (weights stored [k, n]).
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, uint32_t lbo_bytes)
{
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(lbo_bytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// The cluster's barrier in two parts, and bytes from this CTA's shared memory into another's, whose barrier counts them.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_cta(uint32_t saddr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void copy_to_cta(uint32_t to, uint32_t from, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "r"(from), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void st_async(uint32_t to, uint32_t v, uint32_t bar)
{
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to), "r"(v), "r"(bar) : "memory");
}
template <bool TOGETHER>   // four neighbours, or every 32nd
__device__ __forceinline__ int4 ld_shared(uint32_t saddr)
{
    int4 v;
    if (TOGETHER) {
        asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(saddr) : "memory");
    } else {
        asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v.x) : "r"(saddr) : "memory");
        asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v.y) : "r"(saddr + 128) : "memory");
        asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v.z) : "r"(saddr + 256) : "memory");
        asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v.w) : "r"(saddr + 384) : "memory");
    }
    return v;
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float load_as_float(const void *p, int dtype, long long i)
{
    if (dtype == kF32) return static_cast<const float *>(p)[i];
    if (dtype == kF16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
template <typename Y> __device__ __forceinline__ Y from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void store4(float *y, const float (&v)[4]) { *reinterpret_cast<float4 *>(y) = make_float4(v[0], v[1], v[2], v[3]); }
template <typename Y>
__device__ __forceinline__ void store4(Y *y, const float (&v)[4])
{
    Y h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = from_float<Y>(v[i]);
    *reinterpret_cast<uint2 *>(y) = *reinterpret_cast<const uint2 *>(h);
}

// NK: the weight is stored [n, k].
template <bool NK, typename Y>
__global__ void __launch_bounds__(kThreads) quant_matmul_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                               const MatmulParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(8) uint64_t full[kMaxStages], empty[kMaxStages], done, received;
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ alignas(16) float token_scales[kMaxTokens], scales[kChannels], biases[kChannels];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int rank = (int)(blockIdx.x % (unsigned)p.split), tile = (int)(blockIdx.x / (unsigned)p.split);
    const int t0 = tile % p.token_tiles * p.tile_tokens, c0 = tile / p.token_tiles * kChannels;
    const int blocks = (p.k + kBlockK - 1) / kBlockK;
    const int kb0 = (int)((long long)rank * blocks / p.split), kb1 = (int)((long long)(rank + 1) * blocks / p.split);
    const int per = p.tile_tokens / p.split;   // tokens whose sums a CTA of the cluster makes
    uint32_t cols = 32;
    while (cols < (uint32_t)p.tile_tokens) cols *= 2;
    const uint32_t stage_bytes = kWeightStage + (uint32_t)p.tile_tokens * kBlockK;
    const int copies = max(kb1 - kb0 - p.skip_blocks, 0);
    int issued = min(copies, p.stages);        // by warp 0
    const auto copy_block = [&](int i, int stage) {
        const uint32_t s = smem0 + (uint32_t)stage * stage_bytes;
        mbar_arrive_expect_tx(&full[stage], stage_bytes);
        if (NK) tma_load(s, &map_w, (kb0 + i) * kBlockK, c0, &full[stage]);
        else tma_load(s, &map_w, c0, (kb0 + i) * kBlockK, &full[stage]);
        tma_load(s + kWeightStage, &map_x, (kb0 + i) * kBlockK, t0, &full[stage]);
    };
    if (warp == 0 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_x) : "memory");
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(&done, 1);
        mbar_init(&received, 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (p.split > 1) mbar_arrive_expect_tx(&received, (uint32_t)(p.apart ? p.split : p.split - 1) * per * kTokenBytes);
    }
    dependent_wait();
    if (warp == 0) {
        // the ring is filled before anything else: what follows runs beside the copies' way
        __syncwarp();
        const bool leader = elect_one();
        for (int i = 0; i < issued; ++i) {
            if (leader) copy_block(i, i);
            __syncwarp();
        }
    }
    // What the sums are multiplied with is fetched beside the product and stored behind the barrier; behind the product, its way from memory
    // would be waited for.
    float mine[2] = {0.0f, 0.0f};
    if (warp >= 4) {
        const int i = tid - 128;
        if (c0 + i < p.n) {
            mine[0] = load_as_float(p.scale, p.scale_dtype, c0 + i);
            if (p.bias) mine[1] = load_as_float(p.bias, p.bias_dtype, c0 + i);
        }
    }
    // Block 0 is among the first to start, and a wait of the default limit runs out about a second after.
    if (p.clear_status && blockIdx.x == 0 && warp == 2 && lane < 4) p.status[lane] = 0;
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    dependent_release();   // tensor memory is in hand: the next kernel's CTAs may come and wait
    tc_fence_after();
    const uint32_t taddr = tmem_base;
    if (p.apart) cluster_arrive();   // this CTA can be sent to

    if (warp == 0) {
        const bool leader = elect_one();
        int stage = 0;
        uint32_t phase = 0;
        for (; issued < copies; ++issued) {
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase, &gave_up, p, 100 + stage))) break;
            if (leader) copy_block(issued, stage);
            __syncwarp();
            if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        // D = S32 (2 at bit 4), A = B = signed 8 bits (1 at bits 7 and 10), the major of A (the weights) at bit 15, N >> 3 at bit 17, M >> 4 at 24
        const uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (NK ? 0u : 1u) << 15 | (uint32_t)p.tile_tokens >> 3 << 17 | (kChannels >> 4) << 24;
        const uint64_t w0 = operand_desc(smem0, NK ? 16 : kWeightStage), x0 = operand_desc(smem0 + kWeightStage, 16);
        constexpr uint32_t kStepW = (NK ? 32 : 32 * kChannels) >> 4, kStepX = 32 >> 4;
        const bool leader = elect_one();
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, &gave_up, p, 200 + stage));
            if (!ok) break;
            tc_fence_after();
            if (leader) {
                const uint32_t off = (uint32_t)stage * stage_bytes >> 4;
#pragma unroll
                for (int i = 0; i < kBlockK / 32; ++i)
                    umma_i8(taddr, w0 + off + i * kStepW, x0 + off + i * kStepX, idesc, kb > kb0 || i > 0);
                umma_commit(&empty[stage]);
                if (kb + 1 == kb1) umma_commit(&done);
            }
            __syncwarp();
            if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        }
        if (!ok && leader) umma_commit(&done);   // of the MMAs that were issued
        __syncwarp();
    }
    if (warp >= 4) {
        scales[tid - 128] = mine[0];
        biases[tid - 128] = mine[1];
    } else if (warp >= 2) {
        for (int t = tid - 64; t < p.tile_tokens; t += 64) token_scales[t] = p.token_scale && t0 + t < p.m ? p.token_scale[t0 + t] : 1.0f;
    }
    // The sums: TMEM lane = channel, column = token.  They go into shared memory by rows, at the ring's place (every copy has been read by an
    // MMA and every MMA is done), and those that another CTA finishes from there in one piece; few go straight to it instead.
    const int quarter = warp & 3, half = warp >> 2;
    bool ok = __all_sync(0xffffffffu, mbar_wait(&done, 0, &gave_up, p, 300 + warp) && !*(volatile int *)&gave_up);
    if (!ok) drain(&done, 0);   // MMAs write to TMEM, which is given back below, and read the ring
    tc_fence_after();
    const uint32_t piece = (uint32_t)per * kTokenBytes, parts = smem0 + p.parts_at;
    if (p.apart) cluster_wait();
    const int begin = half * (p.tile_tokens / 2), end = ok ? begin + p.tile_tokens / 2 : begin;
    for (int t = begin; t < end; t += 16) {
        uint32_t v[16];
        tmem_ld16(taddr + ((uint32_t)quarter << 21) + (uint32_t)t, v);
        tmem_ld_wait();
        const uint32_t to = (uint32_t)(quarter * 32 + lane) * 4;
        if (!p.apart) {
#pragma unroll
            for (int i = 0; i < 16; ++i) asm volatile("st.shared.b32 [%0], %1;" ::"r"(smem0 + to + (uint32_t)(t + i) * kTokenBytes), "r"(v[i]) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const uint32_t owner = (uint32_t)((t + i) / per), at = parts + to + (uint32_t)(rank * per + (t + i) % per) * kTokenBytes;
                const uint32_t there = in_cta(at, owner), bar = in_cta(smem_u32(&received), owner);
#pragma unroll
                for (int j = 0; j < 4; ++j) st_async(there + j * kTokenBytes, v[i + j], bar);
            }
        }
    }
    tc_fence_before();
    if (p.split > 1 && !p.apart) {
        fence_async_proxy();
        cluster_arrive();   // what comes from the others stands in the ring's place, which every CTA of the cluster is done with then
        cluster_wait();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
    }
    if (p.split > 1) {
        if (warp == 2 && ok && !p.apart) {
            const bool leader = elect_one();
            for (int i = 1; i < p.split; ++i) {
                const int owner = (rank + i) % p.split;   // it has a place for every other CTA
                if (leader)
                    copy_to_cta(in_cta(parts + (uint32_t)(rank - (rank > owner)) * piece, owner), smem0 + (uint32_t)owner * piece, piece,
                                in_cta(smem_u32(&received), owner));
                __syncwarp();
            }
        }
        const bool all = __all_sync(0xffffffffu, mbar_wait<true>(&received, 0, &gave_up, p, 400 + warp));
        if (!all) drain(&received, 0);
        ok = ok && all;
        __syncwarp();
        cluster_arrive();
    }
    // A warp takes a token, a lane four channels: neighbours that are stored at once, or where rows of y are on no such boundary every 32nd.
    const int first = rank * per, tokens = ok ? min(per, p.m - t0 - first) : 0;
    const auto finish = [&](auto together, auto packed) {
        constexpr int kTokens = decltype(together)::value;
        constexpr bool PACKS = decltype(packed)::value;
        const auto channel = [&](int i) { return PACKS ? lane * 4 + i : lane + 32 * i; };
        float scale[4], bias[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            scale[i] = scales[channel(i)];
            bias[i] = biases[channel(i)];
        }
        for (int begin = warp; begin < tokens; begin += kTokens * kWarps) {
            int acc[kTokens][4] = {};
            for (int r = 0; r < p.split; ++r) {
                const uint32_t part = p.apart ? parts + (uint32_t)r * piece : r == rank ? smem0 + (uint32_t)r * piece : parts + (uint32_t)(r - (r > rank)) * piece;
                int4 v[kTokens];
#pragma unroll
                for (int j = 0; j < kTokens; ++j) v[j] = ld_shared<PACKS>(part + (uint32_t)min(begin + j * kWarps, tokens - 1) * kTokenBytes + (uint32_t)channel(0) * 4);
#pragma unroll
                for (int j = 0; j < kTokens; ++j) {
                    acc[j][0] += v[j].x; acc[j][1] += v[j].y; acc[j][2] += v[j].z; acc[j][3] += v[j].w;
                }
            }
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                const int t = begin + j * kWarps;
                if (t >= tokens) break;
                const float token = token_scales[first + t];
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = __fmul_rn(__fmul_rn(__int2float_rn(acc[j][i]), scale[i]), token);
                    if (p.bias) v[i] = __fadd_rn(v[i], bias[i]);
                }
                Y *y = static_cast<Y *>(p.y) + (long long)(t0 + first + t) * p.ld_y + c0;
                if (PACKS && c0 + channel(3) < p.n) {
                    store4(y + channel(0), v);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c0 + channel(i) < p.n) y[channel(i)] = from_float<Y>(v[i]);
                }
            }
        }
    };
    if (!p.packs) finish(Int<4>(), Flag<false>());
    else if (tokens <= kWarps) finish(Int<1>(), Flag<true>());
    else if (p.split == 1) finish(Int<8>(), Flag<true>());
    else finish(Int<4>(), Flag<true>());
    // A wait that ran out may have left copies in flight, which must not land in shared memory that is no longer this CTA's.
    if (warp == 0 && *(volatile int *)&gave_up) {
        for (int i = max(issued - p.stages, 0); i < issued; ++i) drain(&full[i % p.stages], (uint32_t)(i / p.stages) & 1u);
    }
    // No CTA leaves before all of them have received, and so before what it has sent is read.
    __syncwarp();
    if (p.split > 1) cluster_wait();
}

// 16 bytes from byte `shift` of two packs on.
__device__ __forceinline__ uint4 shifted(const uint4 &lo, const uint4 &hi, int shift)
{
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (shift & 8) { w[0] = w[2]; w[1] = w[3]; w[2] = w[4]; w[3] = w[5]; w[4] = w[6]; w[5] = w[7]; }
    if (shift & 4) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = w[4]; w[4] = w[5]; }
    const uint32_t bits = (uint32_t)(shift & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}
__device__ __forceinline__ uint4 first_bytes(const uint4 &v, int valid)
{
    uint32_t r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = valid - 4 * j;
        if (n < 4) r[j] = n <= 0 ? 0u : r[j] & ((1u << 8 * n) - 1u);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Rows on no 16-byte boundary, which no tensor map can describe, copied onto one, with zeros up to the next: a warp takes 2 KB of a row.
// 7168 x 4095 bytes take 8 us, 59 MB read and written.  (Rows shifted into place by the product's own idle warps, which a copy of the weights
// as they lie in memory ran ahead of: 16 x 7168 -> 4095 15.5 us, 17.6 with the copy; 256 x 767 -> 2049 9.5 and 6.8, since every tile shifts its
// weights anew at 0.8 us a K block.  Not kept: 160 lines for the few sizes where it wins.)
struct PackParams {
    const int8_t *src[2];
    int8_t *dst[2];
    long long ld[2], units[2];          // distance of rows; pieces of 2 KB
    int width[2], pitch[2], pieces[2];  // bytes of a row, of its copy; its pieces
};
__global__ void __launch_bounds__(256) quant_matmul_pack_kernel(const PackParams p)
{
    dependent_wait();
    dependent_release();
    long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int o = unit >= p.units[0];
    if (o) unit -= p.units[0];
    if (unit >= p.units[o]) return;
    const int width = o ? p.width[1] : p.width[0], pitch = o ? p.pitch[1] : p.pitch[0], pieces = o ? p.pieces[1] : p.pieces[0];
    const long long row = pieces == 1 ? unit : unit / pieces;
    const int first = (int)(unit - row * pieces) * 128 + (threadIdx.x & 31);
    const int8_t *src = (o ? p.src[1] : p.src[0]) + row * (o ? p.ld[1] : p.ld[0]);
    int8_t *dst = (o ? p.dst[1] : p.dst[0]) + row * pitch;
    const int shift = (int)((uintptr_t)src & 15);
    const uint4 *packs = reinterpret_cast<const uint4 *>((uintptr_t)src & ~(uintptr_t)15);
    uint4 v[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = first + 32 * i;
        v[i][0] = 16 * c < width ? packs[c] : make_uint4(0, 0, 0, 0);
        v[i][1] = 16 * (c + 1) - shift < width ? packs[c + 1] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = first + 32 * i;
        if (16 * c < width) *reinterpret_cast<uint4 *>(dst + 16 * c) = first_bytes(shifted(v[i][0], v[i][1], shift), width - 16 * c);
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn()
{
    static EncodeTiledFn fn = []() -> EncodeTiledFn {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    return fn;
}
bool encode(CUtensorMap *map, const void *base, long long inner, long long rows, long long pitch, int box_rows)
{
    const EncodeTiledFn fn = encode_fn();
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, ones[2] = {1, 1};
    return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a tensor map can describe: rows on packs that do not overlap.  A single row has no distance to the next one.
bool on_packs(const void *p, long long ld, long long width, long long rows) { return ((uintptr_t)p & 15) == 0 && (rows <= 1 || (ld % 16 == 0 && ld >= width)); }
size_t round16(long long v) { return (size_t)(v + 15) / 16 * 16; }
size_t align256(size_t v) { return (v + 255) / 256 * 256; }
long long weight_rows(const QuantMatmulProblem &q) { return q.w_nk ? q.n : q.k; }
long long weight_width(const QuantMatmulProblem &q) { return q.w_nk ? q.k : q.n; }

// Tiles and the split of K.
struct Shape {
    int tile_tokens, token_tiles, channel_tiles, split, stages;
    bool apart;
    size_t parts_at, smem;
    double us;                          // about what the kernel takes
};

// Between the values at 32, 64, 128 and 256 tokens.
double at_tokens(const double (&v)[4], int tokens)
{
    const int i = tokens <= 64 ? 0 : tokens <= 128 ? 1 : 2;
    return v[i] + (v[i + 1] - v[i]) * (tokens - (32 << i)) / (32 << i);
}

// Smaller tiles and K splits bring more CTAs to the weights, larger tiles read them less often, and a split has its sums sent around.  What
// is best is where the estimate below is least: its parts were fitted to times of all ways over 165 sizes (1 to 4096 tokens, K and N of 256
// to 8192; in replayed graphs, with as many sets of operands in turn as make 300 MB and twelve at most, so that weights of more than 10 MB
// come from memory and smaller ones from L2), where the way that it picks takes 1 % longer than the best one on average and 14 % at most.
// It ranks ways and is no forecast: one memory rate for both places and no share of the launch make it up to a quarter too low (16 x 7168
// -> 4096 with 32/4 7.0 for 9.4).  A K block takes 0.16 us at 32 tokens and 0.40 at 256 (what an SM gets from L2, 110 bytes per ns, bounds
// both), the end of a tile 0.4 to 2.9 us, a split 1.4 to 2.6.
// Some of the measured times (us), tile tokens / split: 16 x 7168 -> 4096 32/1 14.1, 32/2 11.0, 32/4 9.4; 16 x 2048 -> 7168 32/1 6.5, 32/4
// 7.2; 256 x 7168 -> 4096 256/2 17.8, 128/1 17.4, 128/2 13.3; 1024 x 2048 -> 2048 256/1 11.2, 128/1 8.5, 64/1 9.2, 128/2 16.2.
Shape shape_with(const QuantMatmulProblem &q, int most_tokens, int split)
{
    static constexpr double kBlock[4] = {0.16, 0.22, 0.23, 0.40}, kEnd[4] = {0.42, 0.62, 1.16, 2.9}, kSplit[4] = {2.2, 1.4, 2.6, 2.5};
    constexpr double kStart = 1.8, kSharedSm = 1.25, kSharedEnd = 0.55, kSharedSplit = 1.6, kBytesPerUs = 9.4e6;
    Shape s;
    s.token_tiles = (int)((q.m + most_tokens - 1) / most_tokens);
    s.tile_tokens = (int)(((q.m + s.token_tiles - 1) / s.token_tiles + 31) / 32 * 32);
    s.channel_tiles = (int)((q.n + kChannels - 1) / kChannels);
    s.split = split;
    const int blocks = (int)((q.k + kBlockK - 1) / kBlockK), each = (blocks + split - 1) / split;
    const double ctas = (double)s.token_tiles * s.channel_tiles * split;
    // room for two CTAs on an SM where tiles are small, or of medium size and more than the SMs.  Small ones leave it where the grid is smaller
    // than the SMs, too, since calls in a row overlap in it (32 tokens, 7168 -> 4096, 32/4 9.6 us, with a ring over all of the memory 10.1; 4096
    // -> 4096 7.7 and 8.3; over 368 such pairs of times the two are equal on average).
    const bool two = s.tile_tokens <= 64 || (s.tile_tokens <= 128 && ctas > kSms);
    const size_t stage = kWeightStage + (size_t)s.tile_tokens * kBlockK, room = (two ? 109 : 220) * 1024;
    const size_t sums = (size_t)s.tile_tokens * kTokenBytes, parts = sums / split * (split - 1);
    s.apart = split > 1 && s.tile_tokens == 32;   // few sums go straight to their place, more (64 tokens: 10.4 us, 13.4 so) in one copy
    s.stages = (int)((room - (s.apart ? sums : 0)) / stage);
    if (s.stages > kMaxStages) s.stages = kMaxStages;
    if (s.stages > each) s.stages = each;
    const size_t ring = s.stages * stage, all = s.apart ? ring + sums : split > 1 ? sums + parts : sums;
    s.parts_at = s.apart ? ring : sums;
    s.smem = 1024 + (all > ring ? all : ring);
    const double turns = std::ceil(ctas / kSms), shared = two && turns > 1 ? turns : 1;   // CTAs of the SM that has most
    const double tile = two ? each * at_tokens(kBlock, s.tile_tokens) * (turns > 1 ? kSharedSm * turns : 1) : each * at_tokens(kBlock, s.tile_tokens) * turns;
    const double end = at_tokens(kEnd, s.tile_tokens) * (two ? 1 + kSharedEnd * (shared - 1) : turns);
    const double memory = ((double)q.m * q.k + (double)q.n * q.k + 2.0 * q.m * q.n) / kBytesPerUs + at_tokens(kEnd, s.tile_tokens);
    s.us = kStart + (tile + end > memory ? tile + end : memory);
    if (split > 1) s.us += at_tokens(kSplit, s.tile_tokens) * (split - 1) / split * (turns > 1 ? kSharedSplit : 1);
    if (each * split >= blocks + split || split > blocks || all > room) s.us = HUGE_VAL;   // an empty part, or too little memory
    return s;
}
Shape shape_of(const QuantMatmulProblem &q)
{
    Shape best = shape_with(q, kMaxTokens, 1);
    for (int tokens = kMaxTokens; tokens >= 32; tokens /= 2) {
        if (tokens > 32 && tokens / 2 >= q.m) continue;   // the same tile as the next one's
        for (int split = 1; split <= kMaxSplit; split *= 2) {
            const Shape s = shape_with(q, tokens, split);
            if (s.us < best.us) best = s;
        }
    }
    return best;
}

// The persistent kernel of the grouped products takes large calls (4096 x 7168 -> 4096 78 us, 95 here): its CTA pairs have 256 channels for
// the tokens that they read, and end a tile beside the next one's products.  About 9 us and, for every round of tiles over its units, a tile's
// K blocks or its end (fitted to the same measurements); half a round at least for a last one that is not full.
double grouped_us(const QuantMatmulProblem &q)
{
    const bool pairs = q.m > 128 && q.k >= 1536;
    const double tiles = std::ceil(q.n / (pairs ? 256.0 : 128.0)) * std::ceil(q.m / 256.0), units = pairs ? kSms / 2 : kSms;
    double rounds = tiles / units;
    const double part = rounds - std::floor(rounds);
    if (rounds < 1) rounds = 1;
    else if (part > 0 && part < 0.5) rounds += 0.5 - part;
    const double tile = std::ceil(q.k / 128.0) * 0.37 + 0.7;
    return 9 + rounds * (tile > 3.4 ? tile : 3.4);
}
// The way that a call takes: the kernel above or the grouped one, and what is copied on 16-byte boundaries before.
struct Way {
    bool pack_x, pack_w, grouped;
    Shape shape;
    size_t off_w, bytes;                // workspace: status, copies
    explicit Way(const QuantMatmulProblem &q)
    {
        pack_x = !on_packs(q.x, q.ld_x, q.k, q.m);
        pack_w = !on_packs(q.w, q.ld_w, weight_width(q), weight_rows(q));
        off_w = 256 + (pack_x ? align256((size_t)q.m * round16(q.k)) : 0);
        bytes = off_w + (pack_w ? align256((size_t)weight_rows(q) * round16(weight_width(q))) : 0);
        shape = shape_of(q);
        const auto at4 = [](const void *p) { return ((uintptr_t)p & 3) == 0; };
        grouped = q.y_dtype != kF32 && q.n % 16 == 0 && ((uintptr_t)q.y & 15) == 0 && (q.m == 1 || q.ld_y == q.n) && at4(q.scale) && at4(q.bias) &&
                  grouped_us(q) < shape.us;
    }
};

template <typename Y>
cudaError_t launch_typed(bool nk, const CUtensorMap &map_x, const CUtensorMap &map_w, const MatmulParams &p, const Shape &s, cudaStream_t stream)
{
    const auto kernel = nk ? quant_matmul_kernel<true, Y> : quant_matmul_kernel<false, Y>;
    static unsigned long long done_masks[2] = {0, 0};   // once per device; the attribute is idempotent, so a race only repeats the call
    unsigned long long &done_mask = done_masks[nk];
    int dev = 0;
    cudaGetDevice(&dev);
    if (!((done_mask >> (dev & 63)) & 1ull)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
        if (e != cudaSuccess) return e;
        done_mask |= 1ull << (dev & 63);
    }
    return launch_dependent(kernel, (unsigned)((long long)s.token_tiles * s.channel_tiles * s.split), kThreads, s.smem, s.split, stream, map_x, map_w, p);
}
cudaError_t launch_grouped(const QuantMatmulProblem &q, char *ws, cudaStream_t stream)
{
    Problem g;
    g.x = q.x; g.w = q.w; g.w_scale = q.scale; g.w_scale_dtype = q.scale_dtype; g.x_scale = q.token_scale;
    g.bias = q.bias; g.bias_dtype = q.bias ? q.bias_dtype : kNone;
    g.gl_len = 1; g.M = q.m; g.K = q.k; g.N = q.n; g.E = 1;
    g.ld_x = q.ld_x; g.ld_w = q.ld_w;
    g.w_layout = q.w_nk ? 1 : 0;
    g.out_f16 = q.y_dtype == kF16; g.out0 = q.y;
    g.opt = q.opt;
    g.opt.max_ctas = 0;   // which the kernels above could not follow
    Plan plan;
    make_plan(g, &plan);
    if (plan.path != kPathSm100 || plan.ws_bytes > 256) return cudaErrorInvalidValue;
    return launch(g, plan, ws, 256, stream);
}

}  // namespace

size_t quant_matmul_workspace_bytes(const QuantMatmulProblem &q) { return Way(q).bytes; }

cudaError_t quant_matmul_launch(const QuantMatmulProblem &given, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (given.m <= 0) return cudaSuccess;
    const Way way(given);
    if (!workspace || workspace_bytes < way.bytes) return cudaErrorInvalidValue;
    char *ws = static_cast<char *>(workspace);
    QuantMatmulProblem q = given;
    // A caller's limit may be short: nothing but the stream orders another block's record behind the clearing then.
    const bool clear_status = q.opt.wait_limit_cycles <= 0;
    if (!clear_status && !way.grouped) {
        const cudaError_t e = cudaMemsetAsync(ws, 0, 16, stream);
        if (e != cudaSuccess) return e;
    }
    // a single row may name any distance to the next one
    if (q.m == 1) q.ld_x = (int64_t)round16(q.k);
    if (weight_rows(q) == 1) q.ld_w = (int64_t)round16(weight_width(q));
    if (way.pack_x || way.pack_w) {
        PackParams p = {};
        int n = 0;
        const auto add = [&](const int8_t *&from, int64_t &ld, size_t off, long long rows, long long width) {
            p.src[n] = from; p.dst[n] = reinterpret_cast<int8_t *>(ws + off);
            p.ld[n] = ld; p.width[n] = (int)width; p.pitch[n] = (int)round16(width);
            p.pieces[n] = (int)((width + 2047) / 2048); p.units[n] = rows * p.pieces[n];
            from = p.dst[n];
            ld = p.pitch[n++];
        };
        if (way.pack_x) add(q.x, q.ld_x, 256, q.m, q.k);
        if (way.pack_w) add(q.w, q.ld_w, way.off_w, weight_rows(q), weight_width(q));
        const cudaError_t e = launch_dependent(quant_matmul_pack_kernel, (unsigned)((p.units[0] + p.units[1] + 7) / 8), 256, 0, 1, stream, p);
        if (e != cudaSuccess) return e;
    }
    if (way.grouped) return launch_grouped(q, ws, stream);
    const Shape &s = way.shape;
    CUtensorMap map_x, map_w;
    if (!encode(&map_x, q.x, q.k, q.m, q.ld_x, s.tile_tokens) || !encode(&map_w, q.w, weight_width(q), weight_rows(q), q.ld_w, 128)) return cudaErrorInvalidValue;
    MatmulParams p;
    p.scale = q.scale; p.bias = q.bias; p.scale_dtype = q.scale_dtype; p.bias_dtype = q.bias_dtype;
    p.token_scale = q.token_scale; p.y = q.y; p.ld_y = q.ld_y;
    p.m = (int)q.m; p.k = (int)q.k; p.n = (int)q.n;
    p.tile_tokens = s.tile_tokens; p.token_tiles = s.token_tiles; p.split = s.split; p.stages = s.stages;
    p.parts_at = (uint32_t)s.parts_at; p.apart = s.apart;
    const int y_bytes = q.y_dtype == kF32 ? 4 : 2;
    p.packs = (uintptr_t)q.y % (4 * y_bytes) == 0 && (q.m == 1 || q.ld_y % 4 == 0);
    p.wait_limit = q.opt.wait_limit_cycles > 0 ? q.opt.wait_limit_cycles : kWaitLimitCycles;
    p.skip_blocks = q.opt.test_skip_k_blocks;
    p.status = reinterpret_cast<int *>(ws);
    p.clear_status = clear_status;
    if (q.opt.ev_start) cudaEventRecord(q.opt.ev_start, stream);
    const cudaError_t e = q.y_dtype == kF32 ? launch_typed<float>(q.w_nk, map_x, map_w, p, s, stream)
                        : q.y_dtype == kF16 ? launch_typed<__half>(q.w_nk, map_x, map_w, p, s, stream)
                                            : launch_typed<__nv_bfloat16>(q.w_nk, map_x, map_w, p, s, stream);
    if (q.opt.ev_stop) cudaEventRecord(q.opt.ev_stop, stream);
    return e;
}

}  // namespace gmm
