// Beam search: the best continuations of every batch item over its beams and the vocabulary, and the beams' states brought into the new
// order.
//
// Selection.  total(beam, token) = score + log p, log p = (x - max) - log sum exp(x - max); the k largest totals of an item, ties to the
// lowest (beam, token).  One cluster of blocks takes an item, and the logits are read once: a warp reduces its share of a beam's row to a
// maximum and a sum.  From those every block has each beam's log-sum, and a bound: of all shares' maxima, as totals, the k-th largest - at
// least k totals reach it.  Only shares whose maximum reaches the bound, hardly more than k of them, are looked through again for the totals
// that do; the few found are ranked by the cluster's first block.  Sums are held in fp32 within a lane (some hundred terms) and in 64 bits
// beyond, totals are compared in 64 bits.
//
// What a lane reads and adds depends on the tokens' numbers alone, not on a row's address, so that equal rows have equal totals.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace psb {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kLine = 256;              // tokens that a warp reads at once: 8 neighbouring ones a lane
constexpr int kMaxBeams = 64;
constexpr int kMaxChosen = 64;
constexpr int kMaxCluster = 16;
constexpr int kMaxGroups = 512;         // shares are joined to at most so many for the bound
constexpr int kFoundCap = 2048;

struct SelectArgs {
    const void* logits;
    const float* scores;
    int* parents;
    int* tokens;
    float* totals;
    long long row_stride;
    int beams, vocab, k, lines;
    int join;                           // shares of a beam joined for the bound
    bool wide;                          // rows begin at multiples of 16 bytes
};

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(__half v) { return __half2float(v); }
__device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }

// 2^v to 2 units in the last place; results below 2^-126 are zero, which a sum of one or more does not notice.
__device__ __forceinline__ float exp2_of(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// Eight neighbouring tokens' logits; -inf behind the vocabulary's end.
template <typename T>
__device__ __forceinline__ void read8(const T* row, int at, int vocab, bool wide, float (&x)[8]) {
    if (wide && at + 8 <= vocab) {
        alignas(16) T v[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(row + at) + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = value(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = at + i < vocab ? value(row[at + i]) : -INFINITY;
    }
}

// Totals as integers of the same order (a total is never NaN).
__device__ __forceinline__ unsigned long long ordered(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);   // -0 counts as 0
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double from_ordered(unsigned long long o) { return __longlong_as_double((long long)(o >> 63 ? o ^ (1ull << 63) : ~o)); }

struct Found { unsigned long long total; unsigned at; unsigned pad; };   // at = beam * vocab + token
__device__ __forceinline__ bool before(const Found& a, const Found& b) { return a.total > b.total || (a.total == b.total && a.at < b.at); }

struct Share { float top; double sum; };

struct SelectShared {
    Share shares[kMaxBeams][kWarps];
    Found found[kFoundCap];
    int count;
    // of the whole item, the same in every block
    float group_top[kMaxGroups];
    double group_sum[kMaxGroups];
    float reach[kMaxGroups];
    float top[kMaxBeams];
    double log_sum[kMaxBeams], score[kMaxBeams];
    bool open[kMaxBeams];               // the beam offers continuations
    float bound;
    Found all[kMaxCluster * kMaxChosen];
    int counts[kMaxCluster + 1];
};

// The found ones beyond the k best go; the k best stay in no order.  For all threads of the block.
__device__ void keep_best(SelectShared& s, int k) {
    const int n = s.count;
    Found mine[kFoundCap / kThreads];
    bool stays[kFoundCap / kThreads];
#pragma unroll
    for (int j = 0; j < kFoundCap / kThreads; ++j) {
        const int i = threadIdx.x + j * kThreads;
        stays[j] = false;
        if (i >= n) continue;
        mine[j] = s.found[i];
        int rank = 0;
        for (int o = 0; o < n; ++o) rank += before(s.found[o], mine[j]);
        stays[j] = rank < k;
    }
    __syncthreads();
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kFoundCap / kThreads; ++j)
        if (stays[j]) s.found[atomicAdd(&s.count, 1)] = mine[j];
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_beam_select(SelectArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    SelectShared& s = *reinterpret_cast<SelectShared*>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long item = blockIdx.x / blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int warps = blocks * kWarps, me = rank * kWarps + warp;
    const T* rows = static_cast<const T*>(a.logits) + item * a.beams * a.row_stride;
    if (threadIdx.x == 0) s.count = 0;

    // The warps take the lines of all beams in turn, so that short rows spread as well: line l of beam b goes to warp (b lines + l) % warps.
    auto first_line = [&](int b) { const int r = (int)((me - (long long)b * a.lines) % warps); return r < 0 ? r + warps : r; };
    for (int b = 0; b < a.beams; ++b) {
        const T* row = rows + b * a.row_stride;
        float top = -INFINITY, sum = 0.f;
        for (int l0 = first_line(b); l0 < a.lines; l0 += 4 * warps) {
            float x[4][8];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int l = l0 + u * warps;
                if (l < a.lines) read8(row, l * kLine + lane * 8, a.vocab, a.wide, x[u]);
                else
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[u][i] = -INFINITY;
            }
            float t = top;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) t = fmaxf(t, x[u][i]);
            // without a finite maximum only infinities or NaN were seen, which the sum has to show
            const float base = t == -INFINITY ? 0.f : t;
            sum *= exp2_of((top - base) * kLog2e);
            top = t;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += exp2_of((x[u][i] - base) * kLog2e);
        }
        // lanes to a share; a lane without a finite maximum has a sum of zero or NaN
        float all = top;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
        double part = top == -INFINITY ? (double)sum : (double)sum * (double)exp2_of((top - all) * kLog2e);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if (lane == 0) s.shares[b][warp] = Share{all, part};
    }
    cluster.sync();

    // Every block: all shares, joined to groups, and from them the beams' log-sums and the bound.
    const int per_beam = (warps + a.join - 1) / a.join, groups = per_beam * a.beams;
    for (int g = threadIdx.x; g < groups; g += kThreads) {
        const int b = g / per_beam, w0 = g % per_beam * a.join, w1 = min(w0 + a.join, warps);
        float top = -INFINITY;
        for (int w = w0; w < w1; ++w) top = fmaxf(top, cluster.map_shared_rank(&s.shares[b][w % kWarps], w / kWarps)->top);
        double sum = 0;
        for (int w = w0; w < w1; ++w) {
            const Share h = *cluster.map_shared_rank(&s.shares[b][w % kWarps], w / kWarps);
            sum += h.top == -INFINITY ? h.sum : h.sum * exp((double)h.top - (double)top);
        }
        s.group_top[g] = top;
        s.group_sum[g] = sum;
    }
    __syncthreads();
    for (int b = warp; b < a.beams; b += kWarps) {
        float top = -INFINITY;
        for (int g = lane; g < per_beam; g += 32) top = fmaxf(top, s.group_top[b * per_beam + g]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        double sum = 0;
        for (int g = lane; g < per_beam; g += 32) {
            const float t = s.group_top[b * per_beam + g];
            sum += t == -INFINITY ? s.group_sum[b * per_beam + g] : s.group_sum[b * per_beam + g] * exp((double)t - (double)top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const double ls = log(sum), score = a.scores[item * a.beams + b];
            s.top[b] = top; s.log_sum[b] = ls; s.score[b] = score;
            s.open[b] = isfinite(top) && isfinite(ls) && isfinite(score);
        }
    }
    __syncthreads();
    auto total = [&](int b, float x) { return s.score[b] + (((double)x - (double)s.top[b]) - s.log_sum[b]); };
    for (int g = threadIdx.x; g < groups; g += kThreads) {
        const int b = g / per_beam;
        s.reach[g] = s.open[b] ? __double2float_rd(total(b, s.group_top[g])) : -INFINITY;
    }
    if (threadIdx.x == 0) s.bound = -INFINITY;
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += kThreads) {
        const float mine = s.reach[g];
        int above = 0;
        for (int o = 0; o < groups; ++o) above += s.reach[o] > mine || (s.reach[o] == mine && o < g);
        if (above == a.k - 1) s.bound = mine;
    }
    __syncthreads();
    const double bound = s.bound;

    // The shares that reach the bound, again: their totals that do.
    for (int b = 0; b < a.beams; ++b) {
        const float top = s.shares[b][warp].top;
        if (s.open[b] && top != -INFINITY && total(b, top) >= bound) {
            const T* row = rows + b * a.row_stride;
            auto each = [&](auto&& what) {
                for (int l = first_line(b); l < a.lines; l += warps) {
                    float x[8];
                    read8(row, l * kLine + lane * 8, a.vocab, a.wide, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) what(x[i], (unsigned)(l * kLine + lane * 8 + i));
                }
            };
            int n = 0;
            each([&](float x, unsigned) { n += x != -INFINITY && total(b, x) >= bound; });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
            if (n <= a.k) {
                each([&](float x, unsigned token) {
                    if (x != -INFINITY && total(b, x) >= bound) {
                        const int at = atomicAdd(&s.count, 1);
                        s.found[at] = Found{ordered(total(b, x)), (unsigned)b * (unsigned)a.vocab + token, 0u};
                    }
                });
            } else {   // many: the k best of the share, one by one
                Found last{~0ull, 0u, 0u};
                bool any = false;
                for (int i = 0; i < a.k; ++i) {
                    Found best{0ull, ~0u, 0u};
                    each([&](float x, unsigned token) {
                        if (x == -INFINITY) return;
                        const Found f{ordered(total(b, x)), (unsigned)b * (unsigned)a.vocab + token, 0u};
                        if ((!any || before(last, f)) && before(f, best)) best = f;
                    });
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        const Found f{__shfl_xor_sync(0xffffffffu, best.total, o), __shfl_xor_sync(0xffffffffu, best.at, o), 0u};
                        if (before(f, best)) best = f;
                    }
                    if (lane == 0) s.found[atomicAdd(&s.count, 1)] = best;
                    last = best;
                    any = true;
                }
            }
        }
        // a beam adds at most kWarps * k
        __syncthreads();
        if (s.count > kFoundCap - kWarps * kMaxChosen) keep_best(s, a.k);
        __syncthreads();
    }
    if (s.count > a.k) keep_best(s, a.k);
    cluster.sync();

    if (rank == 0) {
        if (threadIdx.x == 0) {
            int n = 0;
            for (int r = 0; r < blocks; ++r) { s.counts[r] = n; n += *cluster.map_shared_rank(&s.count, r); }
            s.counts[blocks] = n;
        }
        __syncthreads();
        const int n = s.counts[blocks];
        for (int i = threadIdx.x; i < blocks * kMaxChosen; i += kThreads) {
            const int r = i / kMaxChosen, j = i % kMaxChosen;
            if (j < s.counts[r + 1] - s.counts[r]) s.all[s.counts[r] + j] = cluster.map_shared_rank(s.found, r)[j];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const Found mine = s.all[i];
            int place = 0;
            for (int o = 0; o < n; ++o) place += before(s.all[o], mine);
            if (place < a.k) {
                const long long to = item * a.k + place;
                a.parents[to] = (int)(mine.at / (unsigned)a.vocab);
                a.tokens[to] = (int)(mine.at % (unsigned)a.vocab);
                a.totals[to] = (float)from_ordered(mine.total);
            }
        }
        for (int i = n + threadIdx.x; i < a.k; i += kThreads) {
            a.parents[item * a.k + i] = -1;
            a.tokens[item * a.k + i] = -1;
            a.totals[item * a.k + i] = -INFINITY;
        }
    }
    cluster.sync();   // no block ends while the first reads what it found
}

template <typename T>
psb_status select(SelectArgs a, int batch, int sms, cudaStream_t s) {
    a.lines = (a.vocab + kLine - 1) / kLine;
    a.wide = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.row_stride * sizeof(T) % 16 == 0;
    // blocks an item: as many as fill the GPU, while each warp has a line
    int blocks = 1;
    while (blocks < kMaxCluster && (long long)batch * blocks * 2 <= 2 * sms && (long long)a.beams * a.lines >= (long long)blocks * kWarps * 2) blocks *= 2;
    // about 8 k groups for the bound
    const int shares = blocks * kWarps;
    a.join = 1;
    while (a.join < shares && ((long long)shares / a.join * a.beams > kMaxGroups || (shares / (2 * a.join)) * a.beams >= 8 * a.k)) a.join *= 2;
    const void* kernel = reinterpret_cast<const void*>(k_beam_select<T>);
    PSB_TRY(kernel_shared(kernel, sizeof(SelectShared)));
    if (blocks > 8) PSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * blocks)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = sizeof(SelectShared); cfg.stream = s;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = blocks; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    PSB_CUDA(cudaLaunchKernelEx(&cfg, k_beam_select<T>, a));
    count_launch();
    return PSB_OK;
}

// ---- states --------------------------------------------------------------------------------------------------------------------------
//
// A thread takes one column - the same few bytes of all beams' states of a layer, item and head - reads what the beams' parents hold there
// and then writes the beams, so that the states may be reordered where they are.  Bound by memory.  Only what moves is read and written.
constexpr int kMoveThreads = 256;

struct ReorderArgs {
    const unsigned char* in;
    unsigned char* out;
    const int* parents;
    const int* lengths;      // may be null
    int layers, batch, beams, heads, tokens;
    long long token_bytes;
};

template <typename U, int BEAMS>
__global__ void __launch_bounds__(kMoveThreads) k_beam_reorder(ReorderArgs a) {
    __shared__ int s_from[kMaxBeams];
    const int item = blockIdx.y % a.batch, layer = blockIdx.y / a.batch;
    const bool place = a.in == a.out;
    if (threadIdx.x < a.beams) {
        const int p = a.parents[item * (long long)a.beams + threadIdx.x];
        s_from[threadIdx.x] = p < 0 || p >= a.beams || (place && p == (int)threadIdx.x) ? -1 : p;
    }
    __syncthreads();
    const int length = a.lengths ? min(max(a.lengths[item], 0), a.tokens) : a.tokens;
    const long long columns = length * (a.token_bytes / (long long)sizeof(U)), pitch = a.tokens * (a.token_bytes / (long long)sizeof(U));
    const long long beam_pitch = pitch * a.heads, base = ((long long)layer * a.batch + item) * a.beams * beam_pitch;
    const U* in = reinterpret_cast<const U*>(a.in) + base;
    U* out = reinterpret_cast<U*>(a.out) + base;
    for (long long i = (long long)blockIdx.x * kMoveThreads + threadIdx.x; i < columns * a.heads; i += (long long)gridDim.x * kMoveThreads) {
        const long long head = i / columns, at = head * pitch + (i - head * columns);
        U v[BEAMS];
#pragma unroll
        for (int j = 0; j < BEAMS; ++j)
            if (j < a.beams && s_from[j] >= 0) v[j] = in[s_from[j] * beam_pitch + at];
#pragma unroll
        for (int j = 0; j < BEAMS; ++j)
            if (j < a.beams && s_from[j] >= 0) out[j * beam_pitch + at] = v[j];
    }
}

template <typename U>
psb_status reorder(const ReorderArgs& a, int sms, cudaStream_t s) {
    const long long columns = a.tokens * (a.token_bytes / (long long)sizeof(U)) * a.heads;
    const long long groups = (long long)a.layers * a.batch;
    const long long blocks = std::max<long long>(1, std::min((columns + kMoveThreads - 1) / kMoveThreads, std::max<long long>(1, 32ll * sms / groups)));
    const dim3 grid((unsigned)blocks, (unsigned)groups);
    if (a.beams <= 4) k_beam_reorder<U, 4><<<grid, kMoveThreads, 0, s>>>(a);
    else if (a.beams <= 8) k_beam_reorder<U, 8><<<grid, kMoveThreads, 0, s>>>(a);
    else if (a.beams <= 16) k_beam_reorder<U, 16><<<grid, kMoveThreads, 0, s>>>(a);
    else k_beam_reorder<U, kMaxBeams><<<grid, kMoveThreads, 0, s>>>(a);
    PSB_LAUNCH_CHECK();
    count_launch();
    return PSB_OK;
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" {

psb_status psb_beam_select(const void* d_logits, int type, int64_t row_stride, const float* d_scores, int batch, int beams, int vocab, int k, int* d_parents, int* d_tokens,
                           float* d_totals, int device, void* stream) {
    if (type < PSB_TYPE_F32 || type > PSB_TYPE_BF16 || batch < 0 || beams <= 0 || vocab <= 0 || k <= 0) return fail(PSB_INVALID_ARGUMENT, "beam selection: a size below its least or an unknown type");
    if (beams > kMaxBeams || k > kMaxChosen || vocab > (1 << 24) || batch > (1 << 20))
        return fail(PSB_UNSUPPORTED_SHAPE, "beam selection: at most 64 beams, 64 continuations an item, 2^24 tokens and 2^20 items");
    if (row_stride < vocab) return fail(PSB_INVALID_ARGUMENT, "beam selection: the stride is less than a row");
    if (batch == 0) return PSB_OK;
    if (!d_logits || !d_scores || !d_parents || !d_tokens || !d_totals) return fail(PSB_INVALID_ARGUMENT, "beam selection: a null pointer");
    auto at = [](const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; };
    if (!at(d_logits, type == PSB_TYPE_F32 ? 4 : 2) || !at(d_scores, 4) || !at(d_parents, 4) || !at(d_tokens, 4) || !at(d_totals, 4))
        return fail(PSB_INVALID_ARGUMENT, "beam selection: a pointer is not aligned to its elements");
    DeviceScope on;
    PSB_TRY(on.enter(device));
    SelectArgs a{};
    a.logits = d_logits; a.scores = d_scores; a.parents = d_parents; a.tokens = d_tokens; a.totals = d_totals;
    a.row_stride = row_stride; a.beams = beams; a.vocab = vocab; a.k = k;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (type) {
        case PSB_TYPE_F32: return select<float>(a, batch, on.sms, s);
        case PSB_TYPE_F16: return select<__half>(a, batch, on.sms, s);
        default: return select<__nv_bfloat16>(a, batch, on.sms, s);
    }
}

psb_status psb_beam_reorder(const void* d_in, void* d_out, const int* d_parents, int layers, int batch, int beams, int heads, int tokens, int64_t token_bytes,
                            const int* d_lengths, int device, void* stream) {
    if (layers < 0 || batch < 0 || beams <= 0 || heads <= 0 || tokens < 0 || token_bytes <= 0) return fail(PSB_INVALID_ARGUMENT, "beam reordering: a size below its least");
    if (beams > kMaxBeams) return fail(PSB_UNSUPPORTED_SHAPE, "beam reordering: at most 64 beams");
    if (batch > 0 && layers > 65535 / batch) return fail(PSB_UNSUPPORTED_SHAPE, "beam reordering: at most 65,535 items over all layers");
    if (layers == 0 || batch == 0 || tokens == 0) return PSB_OK;
    if (!d_in || !d_out || !d_parents) return fail(PSB_INVALID_ARGUMENT, "beam reordering: a null pointer");
    const double bytes = (double)layers * batch * beams * heads * tokens * (double)token_bytes;
    if (bytes > 1e15) return fail(PSB_UNSUPPORTED_SHAPE, "beam reordering: the states are larger than any memory");
    const uintptr_t b0 = reinterpret_cast<uintptr_t>(d_in), o0 = reinterpret_cast<uintptr_t>(d_out), size = (uintptr_t)layers * batch * beams * heads * tokens * token_bytes;
    if (b0 != o0 && b0 < o0 + size && o0 < b0 + size) return fail(PSB_INVALID_ARGUMENT, "beam reordering: the buffers overlap without being the same");
    if (reinterpret_cast<uintptr_t>(d_parents) % 4 || reinterpret_cast<uintptr_t>(d_lengths) % 4)
        return fail(PSB_INVALID_ARGUMENT, "beam reordering: a pointer is not aligned to its elements");
    DeviceScope on;
    PSB_TRY(on.enter(device));
    ReorderArgs a{};
    a.in = static_cast<const unsigned char*>(d_in); a.out = static_cast<unsigned char*>(d_out); a.parents = d_parents; a.lengths = d_lengths;
    a.layers = layers; a.batch = batch; a.beams = beams; a.heads = heads; a.tokens = tokens; a.token_bytes = token_bytes;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uintptr_t unit = b0 | o0 | (uintptr_t)token_bytes;
    if (unit % 16 == 0) return reorder<uint4>(a, on.sms, s);
    if (unit % 4 == 0) return reorder<unsigned>(a, on.sms, s);
    if (unit % 2 == 0) return reorder<unsigned short>(a, on.sms, s);
    return reorder<unsigned char>(a, on.sms, s);
}

}  // extern "C"
