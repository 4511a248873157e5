// Beam search: the best continuations of every batch item over its beams and the vocabulary, and the beams' states brought into the new
// order.
//
// Selection.  total(beam, token) = score + log p, log p = (x - max) - log sum exp(x - max); the k largest totals of an item, ties to the
// lowest (beam, token).  One cluster of blocks takes an item, and the logits are read once: a warp reduces its share of a beam's row to a
// maximum and a sum, and to the maxima of groups of its lanes.  From those every block has each beam's log-sum, and a bound that k of the
// groups' maxima, as totals, reach, so that at least k totals do.  Only the parts of a share whose maximum reaches the bound are looked through
// again; the few totals found are ranked by the cluster's first block.  The warps of a cluster are dealt out to the beams, so that a warp of a small
// call waits for one round of loads and reduces once.
//
// A lane adds its exponentials in fp32: a step's (16 or 32) in chains of four, the steps' sums with compensation, so that the error does not grow with the
// vocabulary (added one after the other, a lane's terms, where they are alike, were 2e-5 off with 100,000 tokens and 9e-4 with 4 million).  Beyond a lane sums are held in
// 64 bits, and totals are compared in 64 bits.
//
// What a lane reads and adds depends on the tokens' numbers alone, not on a row's address, so that equal rows have equal totals.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

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
constexpr int kMaxShares = kMaxCluster * kWarps;
constexpr int kMaxGroups = 2 * kThreads;   // groups of lanes, for the bound
constexpr int kFoundCap = 2048;

struct SelectArgs {
    const void* logits;
    const float* scores;
    int* parents;
    int* tokens;
    float* totals;
    long long row_stride;
    int beams, vocab, k, lines;
    int per_beam;                       // warps that share a beam's row; share s is part s % per_beam of beam s / per_beam, and its warp's (s / warps)-th
    unsigned by_beam;                   // 2^32 / per_beam, rounded up
    int groups;                         // of a share's lanes: a power of two
    bool wide;                          // rows begin at multiples of 16 bytes
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// 2^v to 2 units in the last place; results below 2^-126 are zero, which a sum of one or more does not notice.
__device__ __forceinline__ float exp2_of(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// The largest of a warp's values, for all its lanes.
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// Eight neighbouring tokens' logits as they lie in memory; -inf behind the vocabulary's end.
template <typename T> struct Raw8 {
    static constexpr int kWords = 2 * sizeof(T);
    static constexpr unsigned kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;   // -inf
    unsigned word[kWords];
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) word[i] = kNone;
    }
    // The largest of two words' logits, in pairs where a word holds two.
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
        if constexpr (sizeof(T) == 4) return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
        else if constexpr (std::is_same<T, __half>::value) { const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b)); return *reinterpret_cast<const unsigned*>(&m); }
        else { const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b)); return *reinterpret_cast<const unsigned*>(&m); }
    }
    static __device__ __forceinline__ float largest(unsigned m) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(m);
        else if constexpr (std::is_same<T, __half>::value) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m)); return fmaxf(f.x, f.y); }
        else return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    __device__ __forceinline__ void read(const T* row, int at, int vocab, bool wide) {
        if (wide && at + 8 <= vocab) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + at) + i);
                word[4 * i] = v.x; word[4 * i + 1] = v.y; word[4 * i + 2] = v.z; word[4 * i + 3] = v.w;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) word[i] = at + i < vocab ? __float_as_uint(__ldg(reinterpret_cast<const float*>(row) + at + i)) : 0xff800000u;
            else {
                constexpr unsigned kLow = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
                const unsigned short* u = reinterpret_cast<const unsigned short*>(row);
                const unsigned lo = at + 2 * i < vocab ? __ldg(u + at + 2 * i) : kLow, hi = at + 2 * i + 1 < vocab ? __ldg(u + at + 2 * i + 1) : kLow;
                word[i] = lo | hi << 16;
            }
        }
    }
    __device__ __forceinline__ float2 two(int i) const {   // logits 2 i and 2 i + 1
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(word[2 * i]), __uint_as_float(word[2 * i + 1]));
        else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&word[i]));
        else return make_float2(__uint_as_float(word[i] << 16), __uint_as_float(word[i] & 0xffff0000u));
    }
};

// Totals as integers of the same order (a total is never NaN).
__device__ __forceinline__ unsigned long long ordered(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);   // -0 counts as 0
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double from_ordered(unsigned long long o) { return __longlong_as_double((long long)(o >> 63 ? o ^ (1ull << 63) : ~o)); }

struct Found { unsigned long long total; unsigned at; unsigned pad; };   // at = beam * vocab + token
__device__ __forceinline__ bool before(const Found& a, const Found& b) { return a.total > b.total || (a.total == b.total && a.at < b.at); }

// The largest logit, and the sum of exp2((x - base) kLog2e) over the share's tokens.  base kLog2e is a whole number, `at`, the next above the largest logit's (or kLow,
// below every logit within kFar): an exponent is one fused operation, x kLog2e - at, exact but for its own rounding, and where a larger logit comes, the sum goes
// down by a power of two, exactly.  Where the largest logit lies beyond kFar, `at` cannot hold its fraction (from 1e10 on its own exponent came out in the
// hundreds, and its beam's sum as zero or infinite): such a share is summed again, less the largest logit, which is then the base.
struct Share { float top, at; double sum; };   // at: as long as |top| <= kFar
constexpr float kFar = 4e6f, kLow = -5770781.f;

// 2^v for v <= 2 with a relative error below 1e-9: the Taylor series of e^(f ln 2), |f| <= 1/2, to the eighth power.  (CUDA's own, exact to the last of
// 53 bits, took a quarter of a small call's time.)
__device__ __forceinline__ double exp2_64(double v) {
    if (!(v > -1000.0)) return v == v ? 0.0 : v;
    const double n = rint(v), f = (v - n) * 0.69314718055994531;
    double p = 1.0 / 40320;
    p = fma(p, f, 1.0 / 5040); p = fma(p, f, 1.0 / 720); p = fma(p, f, 1.0 / 120); p = fma(p, f, 1.0 / 24);
    p = fma(p, f, 1.0 / 6); p = fma(p, f, 0.5); p = fma(p, f, 1.0); p = fma(p, f, 1.0);
    return p * __longlong_as_double((long long)((int)n + 1023) << 52);
}
// log v for 1/4 <= v <= 2^25, in fp32 and one step of Newton's method on e^y = v, whose error is the square of fp32's.
__device__ __forceinline__ double log_64(double v) {
    const double y = (double)logf((float)v), e = v * exp2_64(-y * 1.4426950408889634) - 1.0;
    return y + (e - 0.5 * e * e);
}

struct SelectShared {
    Share shares[kMaxShares];                        // of the whole item, written by their warps in every block
    // of this block's shares: the largest logits of 32 parts, and of each lane's steps the three largest, with the numbers of two
    float parts[kMaxBeams / kWarps][kWarps][32];
    float4 steps[kMaxBeams / kWarps][kWarps][32];
    Found found[kFoundCap];
    int count;
    float tops[kMaxGroups];                          // of the groups of lanes of all shares, as `shares`
    float most[kWarps];
    double base[kMaxBeams], log_sum[kMaxBeams], score[kMaxBeams];
    bool open[kMaxBeams];                            // the beam offers continuations
    Found all[kMaxCluster][kMaxChosen];              // in the cluster's first block: what every block found
    int counts[kMaxCluster], first[kMaxCluster + 1];
};

// A lane's part of a share's sum of exp2((x - top) kLog2e), for logits too far from zero for the loop that takes all others.  (Not part of the kernel's code, whose
// registers it would take.)
template <typename T>
__device__ __noinline__ double far_sum(const T* row, int line, int lines, int apart, int vocab, bool wide, float top) {
    double sum = 0;
#pragma unroll 1
    for (; line < lines; line += apart) {
        Raw8<T> x;
        x.read(row, line * kLine + (int)(threadIdx.x & 31) * 8, vocab, wide);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 v = x.two(i); sum += (double)exp2_of((v.x - top) * kLog2e) + (double)exp2_of((v.y - top) * kLog2e); }
    }
    return sum;
}

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
__global__ void __launch_bounds__(kThreads, 2) k_beam_select(SelectArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    SelectShared& s = *reinterpret_cast<SelectShared*>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int item = (int)blockIdx.x / blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int warps = blocks * kWarps, me = rank * kWarps + warp, shares = a.per_beam * a.beams;
    auto beam_of = [&](int share) { return a.per_beam == 1 ? share : (int)__umulhi((unsigned)share, a.by_beam); };   // exact: shares are below 2^16
    auto part_of = [&](int share) { return share - beam_of(share) * a.per_beam; };
    auto row_of = [&](int share) { return static_cast<const T*>(a.logits) + ((long long)item * a.beams + beam_of(share)) * a.row_stride; };
    if (threadIdx.x == 0) s.count = 0;
    if (threadIdx.x < a.beams) s.score[threadIdx.x] = a.scores[(long long)item * a.beams + threadIdx.x];
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // waited for before the first write to another block

    // A share's lines are per_beam apart, kLines of them at a time, read ahead by as many.
    constexpr int kLines = 16 / sizeof(T) / 2;
    const int steps = (a.lines + kLines * a.per_beam - 1) / (kLines * a.per_beam);
    int shift = 0;   // 32 parts at most, of 2^shift steps
    while ((steps - 1) >> shift >= 32) ++shift;
    auto read = [&](const T* row, int line, Raw8<T> (&x)[kLines]) {
#pragma unroll
        for (int u = 0; u < kLines; ++u) {
            if (line + u * a.per_beam < a.lines) x[u].read(row, (line + u * a.per_beam) * kLine + lane * 8, a.vocab, a.wide);
            else x[u].none();
        }
    };
    for (int share = me, turn = 0; share < shares; share += warps, ++turn) {
        const T* row = row_of(share);
        float at = kLow, part = -INFINITY;
        float best = -INFINITY, second = -INFINITY, third = -INFINITY;   // of this lane's steps
        unsigned which = 0;                                             // best's number in the low half, second's in the high
        unsigned long long sums = 0, rest = 0;   // two sums of zero, and what their roundings have left out
        Raw8<T> x[kLines], next[kLines];
        int line = part_of(share);
        read(row, line, x);
#pragma unroll 1   // (twice, registers spill: 64 x 8 x 128,000 bf16 42.1 us instead of 40.0)
        for (int step = 0; step < steps; ++step, line += kLines * a.per_beam) {
            if (step + 1 < steps) read(row, line + kLines * a.per_beam, next);
            unsigned m = Raw8<T>::kNone;
#pragma unroll
            for (int u = 0; u < kLines; ++u)
#pragma unroll
                for (int i = 0; i < Raw8<T>::kWords; ++i) m = Raw8<T>::larger(m, x[u].word[i]);
            const float t = Raw8<T>::largest(m);
            const float most = warp_max(t);
            if (const float to = ceilf(most * kLog2e); to > at) {   // the same for all lanes: the sums come down to the new base
                const float by = at - to >= -126.f ? __int_as_float(((int)(at - to) + 127) << 23) : 0.f;
                sums = mul2(sums, pair(by, by));
                rest = mul2(rest, pair(by, by));
                at = to;
            }
            which = t > best ? which << 16 | (unsigned)step : t > second ? (which & 0xffffu) | (unsigned)step << 16 : which;
            third = t > second ? second : fmaxf(third, t);
            second = t > best ? best : fmaxf(second, t);
            best = fmaxf(best, t);
            if (lane == step >> shift) part = fmaxf(part, most);
            const unsigned long long scale = pair(kLog2e, kLog2e), less = pair(-at, -at);
            unsigned long long of[kLines];
#pragma unroll
            for (int u = 0; u < kLines; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 v = x[u].two(i), e = halves(fma2(pair(v.x, v.y), scale, less));
                    const unsigned long long term = pair(exp2_of(e.x), exp2_of(e.y));
                    of[u] = i ? add2(of[u], term) : term;
                }
#pragma unroll
            for (int apart = kLines / 2; apart > 0; apart /= 2)
#pragma unroll
                for (int u = 0; u < apart; ++u) of[u] = add2(of[u], of[u + apart]);
            const unsigned long long more = add2(of[0], rest), now = add2(sums, more), minus = pair(-1.f, -1.f);
            rest = fma2(fma2(sums, minus, now), minus, more);   // more - (now - sums)
            sums = now;
#pragma unroll
            for (int u = 0; u < kLines; ++u) x[u] = next[u];
        }
        const float top = warp_max(best);
        const float2 v = halves(sums), r = halves(rest);
        double sum = ((double)v.x + (double)r.x) + ((double)v.y + (double)r.y);
        // (without a finite maximum the sum is zero or, with a NaN or an infinity among the logits, NaN)
        if (fabsf(top) > kFar && top != -INFINITY) sum = far_sum(row, part_of(share), a.lines, a.per_beam, a.vocab, a.wide, top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        s.parts[turn][warp][lane] = part;
        s.steps[turn][warp][lane] = make_float4(best, second, third, __uint_as_float(which));
        if (turn == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int o = 16; o >= a.groups; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane < blocks) *cluster.map_shared_rank(&s.shares[share], lane) = Share{top, at, sum};
        if (lane < a.groups)
            for (int r = 0; r < blocks; ++r) *cluster.map_shared_rank(&s.tops[share * a.groups + lane], r) = best;
    }
    if (me >= shares) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    cluster.sync();

    // Every block: each beam's log-sum from its shares.
    for (int b = warp; b < a.beams; b += kWarps) {
        const Share* of = s.shares + b * a.per_beam;
        float top = -INFINITY, highest = -INFINITY;
        for (int j = lane; j < a.per_beam; j += 32) { top = fmaxf(top, of[j].top); highest = fmaxf(highest, fabsf(of[j].top) > kFar ? of[j].top : of[j].at * (1.f / kLog2e)); }
        top = warp_max(top);
        const double base = (double)warp_max(highest);
        double sum = 0;
#pragma unroll 1
        for (int j = lane; j < a.per_beam; j += 32) {
            const Share f = of[j];
            const double down = fabsf(f.top) > kFar ? ((double)f.top - base) * (double)kLog2e : (double)f.at - base * (double)kLog2e;
            sum += f.top == -INFINITY ? f.sum : f.sum * exp2_64(down);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            s.base[b] = base; s.log_sum[b] = log_64(sum);
            s.open[b] = isfinite(top) && isfinite(sum) && isfinite(s.score[b]);
        }
    }
    __syncthreads();
    auto total = [&](int b, float x) { return s.score[b] + (((double)x - s.base[b]) - s.log_sum[b]); };
    // The bound.  Totals rounded down, so that where k of these reach it, so do k totals.
    const int groups = shares * a.groups;
    float mine[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int g = threadIdx.x + i * kThreads, b = beam_of(min(g, groups - 1) / a.groups);
        mine[i] = g < groups && s.open[b] && s.tops[g] != -INFINITY ? __double2float_rd(total(b, s.tops[g])) : -INFINITY;
    }
    float most = warp_max(fmaxf(mine[0], mine[1]));
    if (lane == 0) s.most[warp] = most;
    auto reach = [&](float least) { return __syncthreads_count(mine[0] >= least) + (groups > kThreads ? __syncthreads_count(mine[1] >= least) : 0); };
    float low = -INFINITY;
    if (reach(-FLT_MAX) >= a.k) {
        most = warp_max(s.most[lane & (kWarps - 1)]);
        // steps down from the largest until k reach it, then halves of the last step while many more do
        float high = most, down = 2.f;
        low = most - down;
        int n = reach(low);
        while (n < a.k && low > -FLT_MAX) { high = low; down *= 2.f; low = fmaxf(most - down, -FLT_MAX); n = reach(low); }
        for (int i = 0; i < 8 && n > a.k + 1 + a.k / 4; ++i) {
            const float mid = 0.5f * low + 0.5f * high;
            if (!(mid > low && mid < high)) break;
            const int m = reach(mid);
            if (m >= a.k) { low = mid; n = m; } else high = mid;
        }
    }
    const double bound = low;

    // The shares that reach the bound, again: their totals that do.
    auto reaches = [&](int share) {
        const int b = beam_of(share);
        const float top = s.shares[share].top;
        return s.open[b] && top != -INFINITY && total(b, top) >= bound;
    };
    // what(logit, token) for those of this lane's tokens in a step that reach `least`.  Few do: a mask of them first, then one after the other, so that
    // the code for one is not laid out for every token (instructions that are fetched once cost a small call more than what they do).
    auto few = [&](const T* row, int line, float least, auto&& what) {
        Raw8<T> x[kLines];
        read(row, line, x);
        unsigned mask = 0;
#pragma unroll
        for (int u = 0; u < kLines; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = x[u].two(i);
                mask |= (unsigned)(v.x >= least) << (8 * u + 2 * i) | (unsigned)(v.y >= least) << (8 * u + 2 * i + 1);
            }
#pragma unroll 1
        for (; mask; mask &= mask - 1) {
            const int bit = __ffs(mask) - 1, token = (line + (bit >> 3) * a.per_beam) * kLine + lane * 8 + (bit & 7);
            what(to_float(row[token]), (unsigned)token);
        }
    };
    auto each = [&](int share, int turn, float least, auto&& what) {   // of a share's tokens those of the parts that reach `least`
        const T* row = row_of(share);
        const unsigned parts = __ballot_sync(0xffffffffu, s.parts[turn][warp][lane] >= least);
#pragma unroll 1
        for (int step = 0; step < steps; ++step)
            if (parts >> (step >> shift) & 1) few(row, part_of(share) + step * kLines * a.per_beam, least, what);
    };
    for (int share = me, turn = 0; share < shares; share += warps, ++turn) {
        if (!reaches(share)) continue;
        const int b = beam_of(share);
        // a logit that may reach the bound, a little less than the one that does
        const double from = s.base[b] + (s.log_sum[b] + (bound - s.score[b]));
        const float least = bound == -INFINITY ? -FLT_MAX : fmaxf(-FLT_MAX, __double2float_rd(from - fabs(from) * 1e-12 - (fabs(s.base[b]) + fabs(s.score[b]) + fabs(s.log_sum[b])) * 1e-12));   // never -inf: a token without a logit is none
        auto take = [&](float x, unsigned token) {
            if (total(b, x) >= bound) {
                const int at = atomicAdd(&s.count, 1);
                if (at < kFoundCap) s.found[at] = Found{ordered(total(b, x)), (unsigned)b * (unsigned)a.vocab + token, 0u};
            }
        };
        const float4 top = s.steps[turn][warp][lane];
        if (__any_sync(0xffffffffu, top.z >= least)) { each(share, turn, least, take); continue; }
        // no lane has more than two steps that reach it: every lane reads its own, all at once
        const T* row = row_of(share);
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            const bool there = (i ? top.y : top.x) >= least;
            if (!__any_sync(0xffffffffu, there)) break;
            const unsigned which = __float_as_uint(top.w);
            if (there) few(row, part_of(share) + (int)(i ? which >> 16 : which & 0xffffu) * kLines * a.per_beam, least, take);
            __syncwarp();
        }
    }
    __syncthreads();
    if (s.count > kFoundCap) {   // many totals alike: the k best of each share, one by one, and after each turn of the warps the block's k best
        __syncthreads();
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        for (int first = rank * kWarps, turn = 0; first < shares; first += warps, ++turn) {
            const int share = first + warp, b = beam_of(share);
            if (share < shares && reaches(share)) {
                Found last{~0ull, 0u, 0u};
                for (int i = 0; i < a.k; ++i) {
                    Found best{0ull, ~0u, 0u};
                    each(share, turn, -FLT_MAX, [&](float x, unsigned token) {
                        const Found f{ordered(total(b, x)), (unsigned)b * (unsigned)a.vocab + token, 0u};
                        if ((i == 0 || before(last, f)) && before(f, best)) best = f;
                    });
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        const Found f{__shfl_xor_sync(0xffffffffu, best.total, o), __shfl_xor_sync(0xffffffffu, best.at, o), 0u};
                        if (before(f, best)) best = f;
                    }
                    if (best.total == 0) break;   // the share has no more
                    if (lane == 0) s.found[atomicAdd(&s.count, 1)] = best;
                    last = best;
                }
            }
            __syncthreads();
            if (s.count > kFoundCap - kWarps * kMaxChosen) keep_best(s, a.k);
            __syncthreads();
        }
    }
    __syncthreads();
    if (s.count > a.k) keep_best(s, a.k);
    {
        SelectShared* first = cluster.map_shared_rank(&s, 0);
        if (threadIdx.x < s.count) first->all[rank][threadIdx.x] = s.found[threadIdx.x];
        if (threadIdx.x == 0) first->counts[rank] = s.count;
    }
    cluster.sync();
    if (rank != 0) return;   // nobody looks into the other blocks any more
    if (warp == 0) {
        const int mine = lane < blocks ? s.counts[lane] : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane <= blocks) s.first[lane] = upto - mine;
    }
    __syncthreads();
    const int n = s.first[blocks];
    for (int i = threadIdx.x; i < kMaxCluster * kMaxChosen; i += kThreads) {
        const int r = i % kMaxCluster, j = i / kMaxCluster;
        if (r < blocks && j < s.counts[r]) s.found[s.first[r] + j] = s.all[r][j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const Found mine = s.found[i];
        int place = 0;
        for (int o = 0; o < n; ++o) place += before(s.found[o], mine);
        if (place < a.k) {
            const long long to = (long long)item * a.k + place;
            const unsigned parent = mine.at / (unsigned)a.vocab;
            a.parents[to] = (int)parent;
            a.tokens[to] = (int)(mine.at - parent * (unsigned)a.vocab);
            a.totals[to] = (float)from_ordered(mine.total);
        }
    }
    for (int i = n + threadIdx.x; i < a.k; i += kThreads) {
        const long long to = (long long)item * a.k + i;
        a.parents[to] = -1;
        a.tokens[to] = -1;
        a.totals[to] = -INFINITY;
    }
}

template <typename T>
psb_status select(SelectArgs a, int batch, int sms, cudaStream_t s) {
    a.lines = (a.vocab + kLine - 1) / kLine;
    a.wide = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.row_stride * sizeof(T) % 16 == 0;
    // blocks an item: as many as fill the GPU once (two an SM), while each warp has a line.  64 x 8 x 128,000 bf16: 4 blocks 39.7 us, 2 51.0, 8 49.0; 38 x 16 x 24,800 fp16:
    // 4 blocks 20.4, 2 22.0, 8 25.0; one item of 4 x 32,000 fp32: 16 blocks 8.9
    int blocks = 1;
    while (blocks < kMaxCluster && (long long)batch * blocks * 2 <= 2 * sms && (long long)a.beams * a.lines >= (long long)blocks * kWarps * 2) blocks *= 2;
    const int warps = blocks * kWarps;
    a.per_beam = std::max(1, warps / a.beams);
    a.by_beam = (unsigned)(((1ull << 32) + a.per_beam - 1) / a.per_beam);
    a.groups = 32;
    // (about 32 k of them make the bound tight enough, and up to kThreads are counted at once)
    while (a.groups > 1 && (a.per_beam * a.beams * a.groups > kMaxGroups || a.per_beam * a.beams * a.groups / 2 >= 32 * a.k)) a.groups /= 2;
    const void* kernel = reinterpret_cast<const void*>(k_beam_select<T>);
    PSB_TRY(kernel_shared(kernel, sizeof(SelectShared)));
    if (blocks > 8) {   // clusters of more than 8 are asked for once a device
        static std::atomic<unsigned long long> asked{0};
        int device = 0;
        PSB_CUDA(cudaGetDevice(&device));
        const unsigned long long bit = device < 64 ? 1ull << device : 0;
        if (!(asked.load(std::memory_order_relaxed) & bit)) {
            PSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            asked.fetch_or(bit, std::memory_order_relaxed);
        }
    }
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
    const int item = blockIdx.y, layer = blockIdx.z;
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
    const dim3 grid((unsigned)blocks, (unsigned)a.batch, (unsigned)a.layers);
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
    // An item's blocks read its scores before they write, but other items' blocks may not have read theirs: in place an item's totals are its own scores.
    const int64_t e = type == PSB_TYPE_F32 ? 4 : 2;
    const Span logits(d_logits, (int64_t)batch * beams, vocab * e, row_stride * e), scores(d_scores, batch, 4 * beams, 4 * beams);
    const Span parents(d_parents, batch, 4 * k, 4 * k), tokens(d_tokens, batch, 4 * k, 4 * k), totals(d_totals, batch, 4 * k, 4 * k);
    const bool over_scores = totals.meets(scores) && !(d_totals == d_scores && k == beams);
    if (over_scores || parents.meets(scores) || tokens.meets(scores) || parents.meets(logits) || tokens.meets(logits) || totals.meets(logits) || parents.meets(tokens) ||
        parents.meets(totals) || tokens.meets(totals))
        return fail(PSB_INVALID_ARGUMENT, "beam selection: an output lies over another array (the totals may be the scores themselves where k is the number of beams)");
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
    if (batch > 65535 || layers > 65535) return fail(PSB_UNSUPPORTED_SHAPE, "beam reordering: at most 65,535 items and 65,535 layers");
    if (layers == 0 || batch == 0 || tokens == 0) return PSB_OK;
    if (!d_in || !d_out || !d_parents) return fail(PSB_INVALID_ARGUMENT, "beam reordering: a null pointer");
    const double bytes = (double)layers * batch * beams * heads * tokens * (double)token_bytes;
    if (bytes > 1e15) return fail(PSB_UNSUPPORTED_SHAPE, "beam reordering: the states are larger than any memory");
    const uintptr_t b0 = reinterpret_cast<uintptr_t>(d_in), o0 = reinterpret_cast<uintptr_t>(d_out), size = (uintptr_t)layers * batch * beams * heads * tokens * token_bytes;
    if (b0 != o0 && b0 < o0 + size && o0 < b0 + size) return fail(PSB_INVALID_ARGUMENT, "beam reordering: the buffers overlap without being the same");
    if (reinterpret_cast<uintptr_t>(d_parents) % 4 || reinterpret_cast<uintptr_t>(d_lengths) % 4)
        return fail(PSB_INVALID_ARGUMENT, "beam reordering: a pointer is not aligned to its elements");
    const Span states(d_out, 1, size, 0);
    if (states.meets(Span(d_parents, batch, 4 * beams, 4 * beams)) || states.meets(Span(d_lengths, d_lengths ? batch : 0, 4, 4)))
        return fail(PSB_INVALID_ARGUMENT, "beam reordering: the states lie over the parents or the lengths");
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
