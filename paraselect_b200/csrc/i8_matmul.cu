// Products of rows of 8-bit codes with a scale for each row on both sides:
//   out[i][j] = x_scale[i] w_scale[j] sum_k x[i][k] w[j][k].
// The sum is exact (int32 on the tensor cores, tcgen05 kind::i8), the scaling is three fp32 roundings, the output's type one more.
//
// The rows of w (channels, stored rows) take the tensor cores' M side, 128 to a block, and the rows of x (tokens, queries) the N side, up to
// 256: a thread of the epilogue then holds one channel for all tokens, a warp 32 neighbouring channels, and its stores of a token's outputs
// lie side by side without a pass through shared memory.
//
// k runs through shared memory in slabs of 128 codes (one 128-byte swizzle row), loaded by TMA into a ring; codes behind the end of a row and
// rows behind the last are the TMA's zeros.  Few tiles are split along k over a cluster of up to 8 blocks, which hold their partial sums in
// shared memory and add them there: integers, so the order does not matter.
//
// Waits on the device are bounded.  A block one of whose waits gave up, whichever role's, waits for the products and copies that it has issued, frees
// its tensor memory and forms its outputs with dp4a instead, so that the results are the same.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace psb {

namespace {

namespace cg = cooperative_groups;

constexpr int kSlab = 128;                 // codes of a row in a slab: one swizzle row
constexpr int kChannels = 128;             // rows of w a block
constexpr int kMaxTokens = 256;            // rows of x a tile
constexpr int kEpilogue = 8;               // epilogue warps: two to each quarter of the tensor memory's lanes
constexpr int kThreads = 32 * kEpilogue + 64;   // one warp loads, one issues products
constexpr int kMaxStages = 12;
constexpr int kMaxParts = 8;               // blocks that share a tile
constexpr int kRing = 200 * 1024;
// More than half of an SM's shared memory, so that no two blocks of these kernels share an SM: blocks of a cluster hold their tensor memory while they wait for
// one another, and two clusters, each with a block that waits for the tensor memory that the other's holds, would wait for good.
constexpr size_t kAlone = 116 * 1024;
constexpr int kWaitPolls = 1 << 22;
constexpr long long kAllTiles = 0x7fffffffffffffffll;

struct MatmulArgs {
    const signed char* x;
    const signed char* w;
    const float* x_scales;
    const float* w_scales;
    void* out;
    long long x_stride, w_stride, out_stride;
    int m, n, k;                           // tokens, channels, codes a row
    int tokens;                            // rows of x a tile: a multiple of 16
    int stages, slabs;
    int channel_tiles, tiles;
    long long issued;                      // tiles that get their products (all but in tests)
    int polls;
};

// kind::i8 instruction descriptor: D int32, A and B signed, both K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__host__ __device__ inline int tmem_columns(int tokens, int buffers) {
    int c = 32;
    while (c < tokens * buffers) c <<= 1;
    return c;
}

// The dot product of two rows of codes, four at a time (rows begin at multiples of 16 bytes).
__device__ int dot_codes(const signed char* a, const signed char* b, int k) {
    int s = 0, i = 0;
    for (; i + 4 <= k; i += 4) s = __dp4a(*reinterpret_cast<const int*>(a + i), *reinterpret_cast<const int*>(b + i), s);
    for (; i < k; ++i) s += (int)a[i] * (int)b[i];
    return s;
}

// The scales that a thread of the epilogue needs for a tile: its channel's and one token's.  They are read a tile ahead: a tile of one slab took 0.95 us, most of
// which was the way of its scales from memory (8 x 500,000 x 128: 27 us).
struct Scales { float w, x; };
__device__ __forceinline__ Scales scales_of(const MatmulArgs& a, bool there, int c, int t0, int token) {
    return Scales{there && c < a.n ? __ldg(a.w_scales + c) : 0.f, there && token < a.tokens && t0 + token < a.m ? __ldg(a.x_scales + t0 + token) : 0.f};
}

// The end of a wait, for all lanes of a warp alike: where one gave up, all did.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int polls) { return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, polls)); }

// A named barrier of whole warps; true where every thread says so.
__device__ __forceinline__ bool all_of(bool ok, int barrier, int threads) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "bar.red.and.pred p, %2, %3, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)ok), "r"(barrier), "r"(threads)
        : "memory");
    return r != 0;
}

// An epilogue warp's columns of a tile, 32 channels: channel c in this thread, tokens from t0.  SOLO: the four warps of this half of the epilogue have the tile
// to themselves (its tokens are 32 at most), otherwise each half takes every other 16 tokens; all warps that share the tile call it, whether their wait
// for it ended well (`ready`) or not: where one's did not, none stores and all leave, so that no warp is waited for that has left.
// `scales`: the other of the two buffers still serves slower warps' last tile.
template <typename T, bool SOLO>
__device__ __forceinline__ bool store_tile(const MatmulArgs& a, bool ready, float* scales, const Scales& own, uint32_t from, int c, int t0, int warp, int lane) {
    const int half = SOLO ? 0 : warp >> 2, every = SOLO ? 16 : 32;
    if (SOLO) scales += warp >> 2 << 7;
    scales[(SOLO ? warp & 3 : warp) * 32 + lane] = own.x;
    const bool here = c < a.n;
    const float ws = own.w;
    if (!all_of(ready, SOLO ? 1 + (warp >> 2) : 1, SOLO ? 16 * kEpilogue : 32 * kEpilogue)) return false;
    T* out = static_cast<T*>(a.out) + (long long)(t0 + half * 16) * a.out_stride + c;
    const int live = min(a.tokens, a.m - t0);
    for (int t = half * 16; t < live; t += every, out += every * a.out_stride) {
        uint32_t v[16];
        tmem_ld16(from + t, v);
        float by[16];
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(by + i) = *reinterpret_cast<const float4*>(scales + t + i);
        tc::tmem_ld_wait();
        if (here) {
            T* to = out;
            if (t + 16 <= live) {
#pragma unroll
                for (int i = 0; i < 16; ++i, to += a.out_stride) *to = rounded<T>((float)(int)v[i] * by[i] * ws);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i, to += a.out_stride)
                    if (t + i < live) *to = rounded<T>((float)(int)v[i] * by[i] * ws);
            }
        }
    }
    return true;
}

// Where a block gave up, the copies that are under way to its ring land before it ends.  For one thread.  (They land whatever the call's own limit is.)
__device__ __forceinline__ void await_loads(uint64_t* full, int loads, int stages) {
    for (int i = max(0, loads - stages); i < loads; ++i) tc::mbar_wait(&full[i % stages], (i / stages) & 1);
}

// SPLIT: the blocks of a cluster share a tile, each with its share of the slabs.  Otherwise a block takes every gridDim.x-th tile, its
// accumulators in two buffers, so that the epilogue of one tile lies beside the products of the next.
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) k_i8_matmul(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const MatmulArgs a) {
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], ready[2], drained[2], last;
    __shared__ uint32_t tmem_at;
    __shared__ int gave_up, loads;
    __shared__ __align__(16) float s_scales[2][kMaxTokens];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = SPLIT ? (int)cg::this_cluster().num_blocks() : 1;
    const int part = SPLIT ? (int)cg::this_cluster().block_rank() : 0;
    const int first = SPLIT ? (int)blockIdx.x / parts : (int)blockIdx.x;
    const int step = SPLIT ? a.tiles : (int)gridDim.x;         // a split tile is its cluster's only one
    const int slab0 = a.slabs * part / parts, slab1 = a.slabs * (part + 1) / parts;
    const int stage_bytes = (kChannels + a.tokens) * kSlab;
    constexpr int kBuffers = SPLIT ? 1 : 2;
    // Tiles of few tokens go to the two halves of the epilogue in turn: what a tile takes is then the way from barrier to barrier, not its stores
    // (8 x 500,000 x 128: 24.6 us with both at each tile).
    const bool solo = !SPLIT && a.tokens <= 32;
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) { tc::mbar_init(&full[i], 1); tc::mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { tc::mbar_init(&ready[i], 1); tc::mbar_init(&drained[i], solo ? kEpilogue / 2 : kEpilogue); }
        tc::mbar_init(&last, 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpilogue) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
        }
    } else if (warp == kEpilogue + 1) {
        tc::tmem_alloc(&tmem_at, tmem_columns(a.tokens, kBuffers));
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = tmem_at;

    if (warp == kEpilogue) {
        if (tc::elect_one()) {
            int at = 0;
            bool ok = true;
            for (int tile = first; ok && tile < a.tiles; tile += step) {
                const int c0 = tile % a.channel_tiles * kChannels, t0 = tile / a.channel_tiles * a.tokens;
                for (int slab = slab0; slab < slab1; ++slab, ++at) {
                    const int st = at % a.stages;
                    if (at >= a.stages && !tc::mbar_wait(&empty[st], (at / a.stages - 1) & 1, a.polls)) { ok = false; break; }
                    tc::mbar_expect_tx(&full[st], stage_bytes);
                    unsigned char* to = ring + st * stage_bytes;
                    tc::tma_load_2d(to, &map_w, slab * kSlab, c0, &full[st]);
                    tc::tma_load_2d(to + kChannels * kSlab, &map_x, slab * kSlab, t0, &full[st]);
                }
            }
            loads = at;
            if (!ok) gave_up = 1;
        }
        __syncwarp();
    } else if (warp == kEpilogue + 1) {
        if (tc::elect_one()) {
            const uint32_t idesc = idesc_i8(kChannels, a.tokens);
            int at = 0, count = 0;
            bool ok = true;
            for (int tile = first; ok && tile < a.tiles; tile += step, ++count) {
                const int buf = count % kBuffers;
                if (count >= kBuffers && !tc::mbar_wait(&drained[buf], (count / kBuffers - 1) & 1, a.polls)) { ok = false; break; }
                if (tile >= a.issued) { ok = false; break; }
                tc::tc_fence_after();
                for (int slab = slab0; slab < slab1; ++slab, ++at) {
                    const int st = at % a.stages;
                    if (!tc::mbar_wait(&full[st], (at / a.stages) & 1, a.polls)) { ok = false; break; }
                    tc::tc_fence_after();
                    const uint32_t w_at = tc::smem_u32(ring + st * stage_bytes);
                    const uint64_t dw = tc::make_sw128_desc(w_at), dx = tc::make_sw128_desc(w_at + kChannels * kSlab);
#pragma unroll
                    for (int q = 0; q < kSlab / 32; ++q) umma_i8(tmem + buf * a.tokens, dw + 2 * q, dx + 2 * q, idesc, slab > slab0 || q > 0);
                    tc::umma_commit(&empty[st]);
                }
                if (ok) tc::umma_commit(&ready[buf]);
            }
            if (!ok) gave_up = 1;
        }
        __syncwarp();
    } else {
        int count = 0;
        const int turns = solo ? 2 : 1;
        auto scales = [&](int tile) {
            return scales_of(a, !SPLIT && tile < a.tiles, tile % a.channel_tiles * kChannels + (warp & 3) * 32 + lane, tile / a.channel_tiles * a.tokens, (solo ? warp & 3 : warp) * 32 + lane);
        };
        if (solo) count = warp >> 2;
        int tile = first + count * step;
        Scales next = scales(tile);
        for (; tile < a.tiles; tile += turns * step, count += turns) {
            const int buf = count % kBuffers;
            const int c0 = tile % a.channel_tiles * kChannels, t0 = tile / a.channel_tiles * a.tokens;
            const Scales own = next;
            next = scales(tile + turns * step);
            const bool ok = warp_wait(&ready[buf], (count / kBuffers) & 1, a.polls);
            tc::tc_fence_after();
            const int quarter = warp & 3, half = warp >> 2;
            const uint32_t from = tmem + buf * a.tokens + ((uint32_t)(quarter * 32) << 16);
            const int c = quarter * 32 + lane;
            if constexpr (SPLIT) {   // all products have ended: the ring is free for the partial sums, [token][channel]
                if (!ok) { gave_up = 1; break; }
                int* partial = reinterpret_cast<int*>(ring);
                for (int t = half * 16; t < a.tokens; t += 32) {
                    uint32_t v[16];
                    tmem_ld16(from + t, v);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) partial[(t + i) * kChannels + c] = (int)v[i];
                }
            } else {
                const bool stored = solo ? store_tile<T, true>(a, ok, s_scales[count / 2 & 1], own, from, c0 + c, t0, warp, lane)
                                         : store_tile<T, false>(a, ok, s_scales[count & 1], own, from, c0 + c, t0, warp, lane);
                if (!stored) { gave_up = 1; break; }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(&drained[buf])) : "memory");
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (gave_up) {   // whichever role did: the products and copies under way end before the tensor memory is freed and the ring left
        if (warp == kEpilogue + 1) {
            if (tc::elect_one()) {   // the thread that issued them
                tc::umma_commit(&last);
                tc::mbar_wait(&last, 0);
            }
            __syncwarp();
        }
        if (threadIdx.x == 0) await_loads(full, loads, a.stages);
        tc::tc_fence_before();
        __syncthreads();
        tc::tc_fence_after();
    }
    if (warp == kEpilogue + 1) tc::tmem_dealloc(tmem, tmem_columns(a.tokens, kBuffers));

    if constexpr (SPLIT) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        int lost = 0;
        for (int p = 0; p < parts; ++p) lost |= *cluster.map_shared_rank(&gave_up, p);
        const int c0 = first % a.channel_tiles * kChannels, t0 = first / a.channel_tiles * a.tokens;
        const int* partial = reinterpret_cast<const int*>(ring);
        // four channels a thread: 32 threads a token
        constexpr int kWarps = kThreads / 32;
        const int c4 = (threadIdx.x & 31) * 4;
        float ws[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ws[e] = c0 + c4 + e < a.n ? __ldg(a.w_scales + c0 + c4 + e) : 0.f;
        for (int t = part * kWarps + warp; t < a.tokens && t0 + t < a.m; t += kWarps * parts) {
            const float by = __ldg(a.x_scales + t0 + t);
            int s[4] = {0, 0, 0, 0};
            if (!lost) {
                int4 v[kMaxParts];   // under way together
#pragma unroll
                for (int p = 0; p < kMaxParts; ++p)
                    if (p < parts) v[p] = *reinterpret_cast<const int4*>(cluster.map_shared_rank(partial, p) + t * kChannels + c4);
#pragma unroll
                for (int p = 0; p < kMaxParts; ++p)
                    if (p < parts) { s[0] += v[p].x; s[1] += v[p].y; s[2] += v[p].z; s[3] += v[p].w; }
            } else {
                for (int e = 0; e < 4; ++e)
                    if (c0 + c4 + e < a.n) s[e] = dot_codes(a.x + (long long)(t0 + t) * a.x_stride, a.w + (long long)(c0 + c4 + e) * a.w_stride, a.k);
            }
            T* out = static_cast<T*>(a.out) + (long long)(t0 + t) * a.out_stride + c0 + c4;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c0 + c4 + e < a.n) out[e] = rounded<T>((float)s[e] * by * ws[e]);
        }
        cluster.sync();   // no block ends while another reads its sums
    } else if (gave_up) {
        for (int tile = first; tile < a.tiles; tile += step) {
            const int c0 = tile % a.channel_tiles * kChannels, t0 = tile / a.channel_tiles * a.tokens;
            for (int i = threadIdx.x; i < kChannels * a.tokens; i += kThreads) {
                const int c = c0 + i % kChannels, t = t0 + i / kChannels;
                if (c < a.n && t < a.m)
                    static_cast<T*>(a.out)[(long long)t * a.out_stride + c] =
                        rounded<T>((float)dot_codes(a.x + t * a.x_stride, a.w + c * a.w_stride, a.k) * __ldg(a.x_scales + t) * __ldg(a.w_scales + c));
            }
        }
    }
}

// ---- pairs of blocks ------------------------------------------------------------------------------------------------------------------------
//
// Many tokens: two blocks on neighbouring SMs take 256 channels and up to 256 tokens with one product (cta_group::2).  Each loads its 128 channels and half
// of the tokens, a third less per product than a block alone, whose loads (96 bytes a clock at the tensor cores' rate) are more than an SM gets from L2.
// The first block of the pair issues the products, when both blocks' loads have landed: they count on its barriers.
constexpr int kPairMin = 192;              // tokens from which pairs are taken
__device__ __forceinline__ uint32_t in_first(const void* p) {   // the address of the first block's copy of a shared variable
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(tc::smem_u32(p)));
    return r;
}
__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(tc::smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void pair_umma(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void pair_commit(uint64_t* bar) {   // both blocks' barriers
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(tc::smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

// The tile's channels and tokens: 8 tiles of tokens beside one another share the channels that they read.
__device__ __forceinline__ void place_of(const MatmulArgs& a, int tile, int* c0, int* t0) {
    constexpr int kBeside = 8;
    const int token_tiles = a.tiles / a.channel_tiles, band = kBeside * a.channel_tiles, first = tile / band * kBeside, beside = min(kBeside, token_tiles - first), i = tile % band;
    *c0 = i / beside * (2 * kChannels);
    *t0 = (first + i % beside) * a.tokens;
}

// Where a pair gave up: the copies of both blocks land, which count on the first block's barriers.  The blocks need not have come equally far.  A stage that one of them
// alone has filled expects both blocks' bytes if it is the first block (`mine` > `other`): the second's are made up for; if it is the second, nobody has told the
// barrier to expect anything.  No more such stages than the ring has, since their last filling before has been consumed.  For one thread of the first block.
__device__ __forceinline__ void await_pair_loads(uint64_t* full, int mine, int other, int stages, int stage_bytes) {
    for (int i = other; i < mine; ++i)
        asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(tc::smem_u32(&full[i % stages])), "r"(stage_bytes) : "memory");
    for (int i = mine; i < other; ++i) tc::mbar_expect_tx(&full[i % stages], stage_bytes);
    await_loads(full, max(mine, other), stages);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) k_i8_matmul_pair(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const MatmulArgs a) {
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], ready[2], drained[2], last;
    __shared__ uint32_t tmem_at;
    __shared__ int gave_up, loads;
    __shared__ __align__(16) float s_scales[2][kMaxTokens];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    cg::cluster_group cluster = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster.block_rank();
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int mine = a.tokens / 2, stage_bytes = (kChannels + mine) * kSlab;   // of this block
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) { tc::mbar_init(&full[i], 1); tc::mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { tc::mbar_init(&ready[i], 1); tc::mbar_init(&drained[i], 2 * kEpilogue); }
        tc::mbar_init(&last, 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const int columns = tmem_columns(a.tokens, 2);
    if (warp == kEpilogue + 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_at)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc::tc_fence_before();
    cluster.sync();
    tc::tc_fence_after();
    const uint32_t tmem = tmem_at;

    if (warp == kEpilogue) {
        if (tc::elect_one()) {
            int at = 0;
            bool ok = true;
            for (int tile = first; ok && tile < a.tiles; tile += step) {
                int c0, t0;
                place_of(a, tile, &c0, &t0);
                for (int slab = 0; slab < a.slabs; ++slab, ++at) {
                    const int st = at % a.stages;
                    if (at >= a.stages && !tc::mbar_wait(&empty[st], (at / a.stages - 1) & 1, a.polls)) { ok = false; break; }
                    if (rank == 0) tc::mbar_expect_tx(&full[st], 2 * stage_bytes);
                    unsigned char* to = ring + st * stage_bytes;
                    pair_load(to, &map_w, slab * kSlab, c0 + rank * kChannels, in_first(&full[st]));
                    pair_load(to + kChannels * kSlab, &map_x, slab * kSlab, t0 + rank * mine, in_first(&full[st]));
                }
            }
            // the other block's thread releases the ring's last stages here too: this block does not end before
            for (int i = max(0, at - a.stages); ok && i < at; ++i) ok = tc::mbar_wait(&empty[i % a.stages], (i / a.stages) & 1, a.polls);
            loads = at;
            if (!ok) gave_up = 1;
        }
        __syncwarp();
    } else if (warp == kEpilogue + 1) {
        if (rank == 0 && tc::elect_one()) {
            const uint32_t idesc = idesc_i8(2 * kChannels, a.tokens);
            int at = 0, count = 0;
            bool ok = true;
            for (int tile = first; ok && tile < a.tiles; tile += step, ++count) {
                const int buf = count & 1;
                if (count >= 2 && !tc::mbar_wait(&drained[buf], (count / 2 - 1) & 1, a.polls)) { ok = false; break; }
                if (tile >= a.issued) { ok = false; break; }
                tc::tc_fence_after();
                for (int slab = 0; slab < a.slabs; ++slab, ++at) {
                    const int st = at % a.stages;
                    if (!tc::mbar_wait(&full[st], (at / a.stages) & 1, a.polls)) { ok = false; break; }
                    tc::tc_fence_after();
                    const uint32_t w_at = tc::smem_u32(ring + st * stage_bytes);
                    const uint64_t dw = tc::make_sw128_desc(w_at), dx = tc::make_sw128_desc(w_at + kChannels * kSlab);
#pragma unroll
                    for (int q = 0; q < kSlab / 32; ++q) pair_umma(tmem + buf * a.tokens, dw + 2 * q, dx + 2 * q, idesc, slab > 0 || q > 0);
                    pair_commit(&empty[st]);
                }
                if (ok) pair_commit(&ready[buf]);
            }
            if (!ok) gave_up = 1;
        }
        __syncwarp();
    } else {
        int count = 0;
        auto scales = [&](int tile) {
            int c0 = 0, t0 = 0;
            if (tile < a.tiles) place_of(a, tile, &c0, &t0);
            return scales_of(a, tile < a.tiles, c0 + rank * kChannels + (warp & 3) * 32 + lane, t0, warp * 32 + lane);
        };
        Scales next = scales(first);
        for (int tile = first; tile < a.tiles; tile += step, ++count) {
            const int buf = count & 1;
            int c0, t0;
            place_of(a, tile, &c0, &t0);
            const Scales own = next;
            next = scales(tile + step);
            const bool ok = warp_wait(&ready[buf], (count / 2) & 1, a.polls);
            tc::tc_fence_after();
            const int quarter = warp & 3;
            if (!store_tile<T, false>(a, ok, s_scales[count & 1], own, tmem + buf * a.tokens + ((uint32_t)(quarter * 32) << 16), c0 + rank * kChannels + quarter * 32 + lane, t0, warp,
                                      lane)) {
                gave_up = 1;
                break;
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_first(&drained[buf])) : "memory");
        }
    }
    tc::tc_fence_before();
    cluster.sync();
    tc::tc_fence_after();
    const int lost = gave_up | *cluster.map_shared_rank(&gave_up, rank ^ 1);
    if (lost) {   // whichever block and role gave up: the products and copies under way end before the tensor memory is freed and the rings left
        if (warp == kEpilogue + 1) {
            if (tc::elect_one()) {   // in the first block the thread that issued them; both blocks' barriers hear of their end
                if (rank == 0) pair_commit(&last);
                tc::mbar_wait(&last, 0);
            }
            __syncwarp();
        }
        if (rank == 0 && threadIdx.x == 0) await_pair_loads(full, loads, *cluster.map_shared_rank(&loads, 1), a.stages, stage_bytes);
        tc::tc_fence_before();
        cluster.sync();
        tc::tc_fence_after();
    }
    if (warp == kEpilogue + 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    cluster.sync();   // neither block ends while the other looks
    if (lost) {
        for (int tile = first; tile < a.tiles; tile += step) {
            int c0, t0;
            place_of(a, tile, &c0, &t0);
            for (int i = threadIdx.x; i < kChannels * a.tokens; i += kThreads) {
                const int c = c0 + rank * kChannels + i % kChannels, t = t0 + i / kChannels;
                if (c < a.n && t < a.m)
                    static_cast<T*>(a.out)[(long long)t * a.out_stride + c] =
                        rounded<T>((float)dot_codes(a.x + (long long)t * a.x_stride, a.w + (long long)c * a.w_stride, a.k) * __ldg(a.x_scales + t) * __ldg(a.w_scales + c));
            }
        }
    }
}

// ---- few tokens -----------------------------------------------------------------------------------------------------------------------
//
// With few tokens the product is the reading of w, and the way to the tensor cores - a ring, tensor memory, an exchange between the blocks that
// share a tile - is longer than the product itself.  Here a warp takes four channels and all tokens, 512 codes of each at a time, by dp4a; where channels
// are few, several warps of a block share them along k and add their sums.
constexpr int kFewTokens = 4;
constexpr int kFewDepth = 128;
constexpr int kFewChannels = 4;            // a warp
constexpr int kFewWarps = 8;               // a block

__device__ __forceinline__ int dot16(int4 a, int4 b, int s) { return __dp4a(a.w, b.w, __dp4a(a.z, b.z, __dp4a(a.y, b.y, __dp4a(a.x, b.x, s)))); }

// w's codes pass through L1 once: x's stay there.  (With more tokens the compiler then waits for each load before the next: plain ones.)
template <int M>
__device__ __forceinline__ int4 stream16(const signed char* at) {
    if constexpr (M > 1) return __ldg(reinterpret_cast<const int4*>(at));
    int4 v;
    asm("ld.global.nc.L1::no_allocate.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
    return v;
}

// The codes of a row of k from `at` on, fewer than 16, and whatever lies behind them: what belongs to the row's stride can be read, but behind the last row
// there may be nothing.
__device__ __forceinline__ int4 last16(const signed char* row, int at, int k, bool inner) {
    if (inner) return __ldg(reinterpret_cast<const int4*>(row + at));
    unsigned v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i)
        if (at + i < k) v[i >> 2] |= (unsigned)(unsigned char)row[at + i] << 8 * (i & 3);
    return make_int4((int)v[0], (int)v[1], (int)v[2], (int)v[3]);
}
// The first n codes, zeros behind them.
__device__ __forceinline__ int4 codes_of(int4 v, int n) {
    auto word = [&](int w, int from) { const int bytes = n - from; return bytes >= 4 ? w : bytes <= 0 ? 0 : w & (int)((1u << 8 * bytes) - 1); };
    return make_int4(word(v.x, 0), word(v.y, 4), word(v.z, 8), word(v.w, 12));
}

// LANES of a warp take four channels, 16 codes a lane at a time.  share: warps of a block that take the same channels.
template <typename T, int M, int LANES>
__global__ void __launch_bounds__(32 * kFewWarps) k_i8_few_tokens(const MatmulArgs a, int share) {
    constexpr int kGroups = 32 / LANES;
    __shared__ int s_sums[kFewWarps][kGroups * kFewChannels * M];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % share, group = lane / LANES, in = lane % LANES;
    const long long c0 = (((long long)blockIdx.x * (kFewWarps / share) + warp / share) * kGroups + group) * kFewChannels;
    int sums[kFewChannels][M] = {};
    const signed char* w[kFewChannels];
    const signed char* x[M];
#pragma unroll
    for (int c = 0; c < kFewChannels; ++c) w[c] = a.w + min(c0 + c, (long long)a.n - 1) * a.w_stride;   // (behind the last: the last, not written)
#pragma unroll
    for (int t = 0; t < M; ++t) x[t] = a.x + min(t, a.m - 1) * a.x_stride;
    constexpr int kAhead = M <= 2 ? 4 : 2;      // rounds of loads at once
    const int step = LANES * 16 * share;
    int k0 = (part * LANES + in) * 16;
    const int whole = a.k - 15;                 // 16 codes from here on would pass the end
    for (; k0 + (kAhead - 1) * step < whole; k0 += kAhead * step) {
        int4 v[kAhead][kFewChannels];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int c = 0; c < kFewChannels; ++c) v[u][c] = stream16<M>(w[c] + k0 + u * step);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int t = 0; t < M; ++t) {
                const int4 y = __ldg(reinterpret_cast<const int4*>(x[t] + k0 + u * step));
#pragma unroll
                for (int c = 0; c < kFewChannels; ++c) sums[c][t] = dot16(y, v[u][c], sums[c][t]);
            }
    }
    for (; k0 < whole; k0 += step) {            // the last rounds
        int4 v[kFewChannels];
#pragma unroll
        for (int c = 0; c < kFewChannels; ++c) v[c] = stream16<M>(w[c] + k0);
#pragma unroll
        for (int t = 0; t < M; ++t) {
            const int4 y = __ldg(reinterpret_cast<const int4*>(x[t] + k0));
#pragma unroll
            for (int c = 0; c < kFewChannels; ++c) sums[c][t] = dot16(y, v[c], sums[c][t]);
        }
    }
    if (k0 < a.k) {                             // the last codes of the rows, fewer than 16
        int4 v[kFewChannels];
#pragma unroll
        for (int c = 0; c < kFewChannels; ++c) v[c] = last16(w[c], k0, a.k, c0 + c < a.n - 1);
#pragma unroll
        for (int t = 0; t < M; ++t) {
            const int4 y = codes_of(last16(x[t], k0, a.k, t < a.m - 1), a.k - k0);
#pragma unroll
            for (int c = 0; c < kFewChannels; ++c) sums[c][t] = dot16(y, v[c], sums[c][t]);
        }
    }
    // channel c and token t of a group to its lane (c * M + t) % LANES, in turn (c * M + t) / LANES
    constexpr int kTurns = (kFewChannels * M + LANES - 1) / LANES;
    int mine[kTurns] = {};
    __syncwarp();
#pragma unroll
    for (int c = 0; c < kFewChannels; ++c)
#pragma unroll
        for (int t = 0; t < M; ++t) {
            int s = sums[c][t];
            if constexpr (LANES == 32) s = __reduce_add_sync(0xffffffffu, s);
            else
#pragma unroll
                for (int o = LANES >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            const int i = c * M + t;
            if (in == i % LANES) mine[i / LANES] = s;
        }
    if (share > 1) {
#pragma unroll
        for (int j = 0; j < kTurns; ++j)
            if (in + j * LANES < kFewChannels * M) s_sums[warp][group * kFewChannels * M + in + j * LANES] = mine[j];
        __syncthreads();
        if (part != 0) return;
    }
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
        const int i = in + j * LANES, c = i / M, t = i % M;
        if (i >= kFewChannels * M || t >= a.m || c0 + c >= a.n) continue;
        for (int p = 1; p < share; ++p) mine[j] += s_sums[warp + p][group * kFewChannels * M + i];
        static_cast<T*>(a.out)[(long long)t * a.out_stride + c0 + c] = rounded<T>((float)mine[j] * __ldg(a.x_scales + t) * __ldg(a.w_scales + c0 + c));
    }
}

template <typename T, int M>
psb_status start_few(const MatmulArgs& a, int sms, cudaStream_t s) {
    int lanes = 4;   // as many as have codes
    while (lanes < 32 && a.k > lanes * 24) lanes *= 2;
    const long long groups = ((long long)a.n + kFewChannels * (32 / lanes) - 1) / (kFewChannels * (32 / lanes));   // warps
    int share = 1;
    while (share < kFewWarps && groups * share < 16ll * sms && a.k > lanes * 16 * share) share *= 2;
    const unsigned blocks = (unsigned)((groups * share + kFewWarps - 1) / kFewWarps);
    switch (lanes) {
        case 4: k_i8_few_tokens<T, M, 4><<<blocks, 32 * kFewWarps, 0, s>>>(a, share); break;
        case 8: k_i8_few_tokens<T, M, 8><<<blocks, 32 * kFewWarps, 0, s>>>(a, share); break;
        case 16: k_i8_few_tokens<T, M, 16><<<blocks, 32 * kFewWarps, 0, s>>>(a, share); break;
        default: k_i8_few_tokens<T, M, 32><<<blocks, 32 * kFewWarps, 0, s>>>(a, share); break;
    }
    PSB_LAUNCH_CHECK();
    count_launch();
    return PSB_OK;
}

template <typename T>
psb_status run_few(const MatmulArgs& a, int sms, cudaStream_t s) {
    return a.m == 1 ? start_few<T, 1>(a, sms, s) : a.m == 2 ? start_few<T, 2>(a, sms, s) : start_few<T, 4>(a, sms, s);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

psb_status encode_fn(EncodeTiledFn* out) {
    static std::atomic<EncodeTiledFn> known{nullptr};
    EncodeTiledFn fn = known.load(std::memory_order_acquire);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        PSB_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found));
        if (!p || found != cudaDriverEntryPointSuccess) return fail(PSB_CUDA_ERROR, "cuTensorMapEncodeTiled is not available");
        fn = reinterpret_cast<EncodeTiledFn>(p);
        known.store(fn, std::memory_order_release);
    }
    *out = fn;
    return PSB_OK;
}

// Rows of k codes, `box_rows` of them and a slab of codes at a time.
psb_status codes_map(CUtensorMap* map, const void* base, int64_t rows, int k, int64_t stride, int box_rows) {
    EncodeTiledFn fn;
    PSB_TRY(encode_fn(&fn));
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {(cuuint32_t)kSlab, (cuuint32_t)box_rows};
    const cuuint32_t every[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, every, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(PSB_CUDA_ERROR, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
    return PSB_OK;
}

// The tokens of each of `tiles` tiles of even size, a multiple of `step`.  (m + tiles leaves 32 bits from 2,139,127,681 rows on.)
int tokens_of(int m, int tiles, int step) { return (int)(((long long)m + tiles - 1) / tiles + step - 1) / step * step; }

template <typename T>
psb_status run_pairs(MatmulArgs a, int sms, cudaStream_t s) {
    const int token_tiles = (a.m + kMaxTokens - 1) / kMaxTokens;
    a.tokens = tokens_of(a.m, token_tiles, 32);
    a.channel_tiles = (a.n + 2 * kChannels - 1) / (2 * kChannels);
    const long long tiles = (long long)token_tiles * a.channel_tiles;
    if (tiles > 0x3fffffff) return fail(PSB_UNSUPPORTED_SHAPE, "product of codes: more than 2^30 - 1 tiles of 256 x 256 outputs");
    a.tiles = (int)tiles;
    a.slabs = (a.k + kSlab - 1) / kSlab;
    const int stage_bytes = (kChannels + a.tokens / 2) * kSlab;
    a.stages = std::min(kMaxStages, kRing / stage_bytes);
    const size_t smem = std::max(kAlone, 1024 + (size_t)a.stages * stage_bytes);
    CUtensorMap map_w, map_x;
    PSB_TRY(codes_map(&map_w, a.w, a.n, a.k, a.w_stride, kChannels));
    PSB_TRY(codes_map(&map_x, a.x, a.m, a.k, a.x_stride, a.tokens / 2));
    PSB_TRY(kernel_shared(reinterpret_cast<const void*>(k_i8_matmul_pair<T>), smem));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cfg.gridDim = dim3((unsigned)(2 * std::min<long long>(tiles, sms / 2)));
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    PSB_CUDA(cudaLaunchKernelEx(&cfg, k_i8_matmul_pair<T>, map_w, map_x, a));
    count_launch();
    return PSB_OK;
}

template <typename T>
psb_status run(MatmulArgs a, int sms, cudaStream_t s) {
    // By dp4a and on the tensor cores, k = 4,096: 1 token and 32,000 channels 21.6 and 25.7 us, 4,096 channels 4.2 to 5.4 and 7.1; 2 tokens 28.3 and 26.6, 5.3 and 7.1; 4 tokens
    // 30.4 and 26.5, 5.1 and 7.2.  Short rows: 2 tokens x 200,000 x 64 6.1 and 11.2; 4 x 200,000 x 64 7.3 and 10.6, 4 x 135,872 x 264 29 and 16.6.
    const bool few = a.m == 1 || (a.m <= kFewTokens && (a.n <= kChannels * (sms / 2) || a.k <= kFewDepth));
    if (few && a.issued == kAllTiles) return run_few<T>(a, sms, s);
    // tiles of tokens of even size, each a multiple of 16: of 256 at most, or of 128 where they would not fill half of the GPU (512 x 4,096 x 4,096: 17.9 and 16.2 us,
    // 609 x 641 x 797: 12.1 and 9.8)
    a.channel_tiles = (a.n + kChannels - 1) / kChannels;
    int token_tiles = (a.m + kMaxTokens - 1) / kMaxTokens;
    if (token_tiles > 1 && (long long)token_tiles * a.channel_tiles * 2 < sms) token_tiles = (a.m + 127) / 128;
    a.tokens = tokens_of(a.m, token_tiles, 16);
    const long long tiles = (long long)token_tiles * a.channel_tiles;
    // Pairs and single blocks: 1,024 x 32,000 x 4,096 96.9 and 122.8 us, 256 x 14,336 x 4,096 19.5 and 20.9, 200 x 32,000 x 4,096 32.1 and 33.6, 1,024 x 4,096 x 4,096 17.9 and 18.5
    if (a.m >= kPairMin && tiles * 2 >= sms) return run_pairs<T>(a, sms, s);
    if (tiles > 0x3fffffff) return fail(PSB_UNSUPPORTED_SHAPE, "product of codes: more than 2^30 - 1 tiles of 128 x 256 outputs");
    a.tiles = (int)tiles;
    a.slabs = (a.k + kSlab - 1) / kSlab;
    // blocks that share a tile: while the GPU has room for twice as many, and each two slabs or more (256 x 4,096 x 14,336: 4 blocks 23.4 us, 2 with tiles of 128 tokens 33)
    int parts = 1;
    while (parts < kMaxParts && tiles * parts * 2 <= sms && a.slabs >= parts * 4) parts *= 2;
    const int stage_bytes = (kChannels + a.tokens) * kSlab;
    a.stages = std::min(std::min(kMaxStages, std::max(2, (a.slabs + parts - 1) / parts)), kRing / stage_bytes);
    const size_t smem = std::max(kAlone, 1024 + std::max((size_t)a.stages * stage_bytes, parts > 1 ? (size_t)a.tokens * kChannels * 4 : 0));
    CUtensorMap map_w, map_x;
    PSB_TRY(codes_map(&map_w, a.w, a.n, a.k, a.w_stride, kChannels));
    PSB_TRY(codes_map(&map_x, a.x, a.m, a.k, a.x_stride, a.tokens));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr = {};
    if (parts > 1) {
        PSB_TRY(kernel_shared(reinterpret_cast<const void*>(k_i8_matmul<T, true>), smem));
        cfg.gridDim = dim3((unsigned)(a.tiles * parts));
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = parts; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr; cfg.numAttrs = 1;
        PSB_CUDA(cudaLaunchKernelEx(&cfg, k_i8_matmul<T, true>, map_w, map_x, a));
    } else {
        PSB_TRY(kernel_shared(reinterpret_cast<const void*>(k_i8_matmul<T, false>), smem));
        cfg.gridDim = dim3((unsigned)std::min<long long>(tiles, sms));
        PSB_CUDA(cudaLaunchKernelEx(&cfg, k_i8_matmul<T, false>, map_w, map_x, a));
    }
    count_launch();
    return PSB_OK;
}

constexpr int kMaxDepth = 131071;   // 128 * 128 * k stays below 2^31

psb_status matmul(const int8_t* d_x, int64_t x_stride, const float* d_x_scales, int64_t m, const int8_t* d_w, int64_t w_stride, const float* d_w_scales, int64_t n, int k,
                  void* d_out, int out_type, int64_t out_stride, long long issued, int polls, int device, void* stream) {
    if (m < 0 || n < 0 || k <= 0 || out_type < PSB_TYPE_F32 || out_type > PSB_TYPE_BF16) return fail(PSB_INVALID_ARGUMENT, "product of codes: a size below its least or an unknown type");
    if (k > kMaxDepth || m > 0x7fffff00 || n > 0x7fffff00) return fail(PSB_UNSUPPORTED_SHAPE, "product of codes: at most 131,071 codes a row and 2^31 - 256 rows");
    if (x_stride < k || w_stride < k || out_stride < n) return fail(PSB_INVALID_ARGUMENT, "product of codes: a stride is less than a row");
    if (m == 0 || n == 0) return PSB_OK;
    if (!d_x || !d_w || !d_x_scales || !d_w_scales || !d_out) return fail(PSB_INVALID_ARGUMENT, "product of codes: a null pointer");
    auto at = [](const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; };
    if (!at(d_x, 16) || !at(d_w, 16) || x_stride % 16 || w_stride % 16)
        return fail(PSB_INVALID_ARGUMENT, "product of codes: rows of codes begin at multiples of 16 bytes, their strides are multiples of 16");
    if (x_stride >= (1ll << 40) || w_stride >= (1ll << 40)) return fail(PSB_UNSUPPORTED_SHAPE, "product of codes: a stride of 2^40 bytes or more");
    const size_t e = out_type == PSB_TYPE_F32 ? 4 : 2;
    if (!at(d_out, e) || !at(d_x_scales, 4) || !at(d_w_scales, 4)) return fail(PSB_INVALID_ARGUMENT, "product of codes: a pointer is not aligned to its elements");
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(d_out), o1 = o0 + ((uintptr_t)(m - 1) * out_stride + n) * e;
    auto apart = [&](const void* p, int64_t rows, int64_t stride, int64_t width) {
        const uintptr_t b = reinterpret_cast<uintptr_t>(p);
        return b >= o1 || b + (uintptr_t)(rows - 1) * stride + width <= o0;
    };
    if (!apart(d_x, m, x_stride, k) || !apart(d_w, n, w_stride, k) || !apart(d_x_scales, m, 4, 4) || !apart(d_w_scales, n, 4, 4))
        return fail(PSB_INVALID_ARGUMENT, "product of codes: the output lies over an input");
    DeviceScope on;
    PSB_TRY(on.enter(device));
    MatmulArgs a{};
    a.x = reinterpret_cast<const signed char*>(d_x); a.w = reinterpret_cast<const signed char*>(d_w);
    a.x_scales = d_x_scales; a.w_scales = d_w_scales; a.out = d_out;
    a.x_stride = x_stride; a.w_stride = w_stride; a.out_stride = out_stride;
    a.m = (int)m; a.n = (int)n; a.k = k; a.issued = issued; a.polls = polls;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (out_type) {
        case PSB_TYPE_F32: return run<float>(a, on.sms, s);
        case PSB_TYPE_F16: return run<__half>(a, on.sms, s);
        default: return run<__nv_bfloat16>(a, on.sms, s);
    }
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" {

psb_status psb_i8_matmul(const int8_t* d_x, int64_t x_stride, const float* d_x_scales, int64_t m, const int8_t* d_w, int64_t w_stride, const float* d_w_scales, int64_t n,
                         int k, void* d_out, int out_type, int64_t out_stride, int device, void* stream) {
    return matmul(d_x, x_stride, d_x_scales, m, d_w, w_stride, d_w_scales, n, k, d_out, out_type, out_stride, kAllTiles, kWaitPolls, device, stream);
}

psb_status psb_i8_matmul_limited(const int8_t* d_x, int64_t x_stride, const float* d_x_scales, int64_t m, const int8_t* d_w, int64_t w_stride, const float* d_w_scales,
                                 int64_t n, int k, void* d_out, int out_type, int64_t out_stride, int64_t tiles, int polls, int device, void* stream) {
    if (polls <= 0) return fail(PSB_INVALID_ARGUMENT, "product of codes: a wait without polls");
    return matmul(d_x, x_stride, d_x_scales, m, d_w, w_stride, d_w_scales, n, k, d_out, out_type, out_stride, tiles < 0 ? kAllTiles : tiles, polls, device,
                  stream);
}

}  // extern "C"
