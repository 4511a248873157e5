// Rows to 8-bit codes with one scale a row, plain or behind a residual addition and a root-mean-square norm:
//   h = x + r,  u = h w,  code = rint(127 u / max|u|) (ties to even),  scale = max|u| / (127 rms),  rms = sqrt(mean h^2 + eps);
// without the norm u = x and scale = max|x| / 127.  The norm's 1/rms is common to the row, so the codes do not depend on it.
//
// Codes are those of 64-bit arithmetic.  A code is first formed in fp32: with the norm u has a relative error of 2^-23 at most (one rounding in h, one
// in the product), and so has the largest |u|; 127 / max|u| adds 2^-24, and the last product goes into a fused sum.  So t is off by less than
// 127 * 5 * 2^-24 = 3.8e-5; without the norm by 127 * 2^-24 = 7.6e-6.  Only where t lies so near to a tie (one element in 12,500, or 50,000) it is
// formed again in 64 bits from the row's own values, and for it the row's largest |u|, sought among the elements within 2^-21 of fp32's.  Rows whose
// magnitudes leave fp32's safe range go through 64 bits altogether.
//
// Bound by memory: one pass over the row, which stays in registers between the reduction and the codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace psb {

namespace {

template <bool NORM> constexpr float kNearTie = 0.5f - (NORM ? 4e-5f : 1e-5f);
constexpr float kNearTop = 1.0f - 1.0f / (1 << 21);
constexpr float kSafeLow = 1e-30f, kSafeHigh = 1e30f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of neighbouring elements.
template <typename T> struct Pack {
    static constexpr int VEC = 16 / sizeof(T);
    unsigned word[4];
    // Elements [at, at + VEC) of a row, which begin a pack of memory.
    __device__ __forceinline__ void read(const T* row, int at) { set(*reinterpret_cast<const uint4*>(row + at)); }
    // A second time, rather than held in registers.
    __device__ __forceinline__ void read_again(const T* row, int at) {
        asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(word[0]), "=r"(word[1]), "=r"(word[2]), "=r"(word[3]) : "l"(row + at));
    }
    __device__ __forceinline__ void read_each(const T* row, int at) {   // wherever the row begins
        T v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = row[at + e];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) word[i] = *reinterpret_cast<const unsigned*>(&v[i]);
            else word[i] = *reinterpret_cast<const unsigned short*>(&v[2 * i]) | (unsigned)*reinterpret_cast<const unsigned short*>(&v[2 * i + 1]) << 16;
        }
    }
    __device__ __forceinline__ void zeros() { set(make_uint4(0, 0, 0, 0)); }
    __device__ __forceinline__ void ones() {
        constexpr unsigned kOnes = sizeof(T) == 4 ? 0x3f800000u : std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;
        set(make_uint4(kOnes, kOnes, kOnes, kOnes));
    }
    __device__ __forceinline__ void set(uint4 v) { word[0] = v.x; word[1] = v.y; word[2] = v.z; word[3] = v.w; }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(word[e]);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(e & 1 ? word[e >> 1] & 0xffff0000u : word[e >> 1] << 16);
        else { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&word[e >> 1])); return e & 1 ? f.y : f.x; }
    }
    static __device__ __forceinline__ void write(T* at, const unsigned long long* pairs) {
        unsigned o[4];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const float2 v = halves(pairs[i]);
            if constexpr (sizeof(T) == 4) { o[2 * i] = __float_as_uint(v.x); o[2 * i + 1] = __float_as_uint(v.y); }
            else if constexpr (std::is_same<T, __nv_bfloat16>::value) { const __nv_bfloat162 p = __floats2bfloat162_rn(v.x, v.y); o[i] = *reinterpret_cast<const unsigned*>(&p); }
            else { const __half2 p = __floats2half2_rn(v.x, v.y); o[i] = *reinterpret_cast<const unsigned*>(&p); }
        }
        *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
    }
};


struct MaxOp { template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct SumOp { template <typename V> __device__ V operator()(V a, V b) const { return a + b; } };

template <int WIDTH, typename V, typename Op>
__device__ __forceinline__ V lanes_reduce(V v, Op op) {
#pragma unroll
    for (int o = WIDTH >> 1; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// Over the THREADS threads of a block.  `slots` holds a value a warp and is used once.
template <int THREADS, typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* slots, Op op) {
    v = lanes_reduce<32>(v, op);
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    return lanes_reduce<THREADS / 32>(slots[threadIdx.x & (THREADS / 32 - 1)], op);
}

// A magnitude's bits: their order as integers is that of the magnitudes, and a NaN's are above all.
__device__ __forceinline__ unsigned long long magnitude(double v) { return (unsigned long long)__double_as_longlong(v) & 0x7fffffffffffffffull; }
// The larger magnitude; NaN where either is.
__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}
struct LargerOp { __device__ float operator()(float a, float b) const { return larger(a, b); } };

__device__ __forceinline__ signed char code64(double u, double top) { return (signed char)(int)rint(127.0 * u / top); }

constexpr float kRint = 12582912.f;   // 1.5 * 2^23: a sum with it is rounded to whole numbers, which its lowest bits hold

// Four codes' lowest bytes in one word.
__device__ __forceinline__ unsigned four(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// The largest of a warp's values, NaN where there is one.
__device__ __forceinline__ float warp_larger(float v) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// Blocks of MOST threads that an SM's registers shall hold.  More blocks hide more of each other's waits until their registers spill.  Times in us at full clocks, and
// where a second figure stands, after a second of calls, at the power limit, by which choices are made that differ there:
//
//   form (kEach, threads a block)           measured on                  blocks an SM and times
//   24 or 32, 256, norm, whole packs        16,384 x 8,192 bf16          3: 170 / 182    4: 164 / 186   5: 216
//   24 or 32, 256, norm, SHIFT              200,000 x 500 bf16           3: 141          4: 160
//   24 or 32, 256, whole packs              30,000 x 4,096 bf16          4: 68           5: 64.5        6: 63
//   32, 256, SHIFT, a part of a warp a row  1M x 101 fp16                4: 82 / 86      5: 82 / 91     6: 101 / 113
//                                           150,000 x 701 bf16           4: 94 / 95      5: 87 / 87     6: 92 / 92
//   32, 256, SHIFT, a block a row           30,000 x 4,001 bf16          4: 80 / 81      5: 74 / 77     6: 74 / 79
//   12 or 16, 256, norm                     100,000 x 1,000 fp32         4: 189          5: 225
//   12 or 16, 256, whole packs              1M x 96 fp32                 6: 74           7: 70
//   16, 256, SHIFT                          100,000 x 333 fp32           6: 34           7: 38
//   512 threads, whole packs                8,000 x 16,384 bf16          1: 125          2: 85    (with norm 235 and 181)
template <int kEach, int MOST, bool NORM, bool SHIFT> constexpr int blocks_of() {
    return MOST == 256 ? (kEach >= 24 ? (NORM ? 3 : SHIFT ? 5 : 6) : NORM ? 4 : SHIFT ? 6 : 7) : MOST == 288 || (MOST == 512 && !(NORM && SHIFT)) ? 2 : 1;
}

// One row for each group of TPR threads of a warp, or for each block (TPR = 0, blocks of at most MOST threads), in registers: kEach elements a thread, in
// packs of 16 bytes.
//
// What few elements need is done apart: 64 bits next to ties, at the top, in rows out of fp32's range.  Such an element is read again from memory, before the
// sum is written, by the 32 lanes of a warp for the one that found it.  (16,384 rows of 8,192 in bf16 with norm: 789 us with that code beside every element, 499 with
// a thread of its own doing it while the block waited, 239 this way.)  fp32 arithmetic then goes two elements an instruction, since the kernel was bound by issue (212).
//
// SHIFT: rows that begin and end anywhere.  Packs are those of memory.  The elements before the row's first pack and behind its last, fewer than a pack each, go
// to threads one by one, beside their packs.  The weight's packs lie otherwise: a block takes every G-th row, G a multiple of a pack's elements, so that it is
// put in place once, in shared memory.  7,000 rows of 8,191 in bf16 with norm and sum:
//   317 us  element by element
//   273 us  the first and last packs checked element by element within every pack's code, the weight's packs shifted anew for each row
//   128 us  the weight put in place once
//   102 us  the first and last elements one by one
// Rows that begin at packs lose by keeping the weight (74 us, kept 82).
template <typename T, int kEach, int TPR, int MOST, bool NORM, bool SHIFT>
__global__ void __launch_bounds__(MOST, (blocks_of<kEach, MOST, NORM, SHIFT>())) k_i8_rows(RowArgs a) {
    constexpr bool kBlock = TPR == 0;
    constexpr int kPart = kBlock ? 32 : TPR;   // threads that exchange by shuffles
    const int each_row = kBlock ? (int)blockDim.x : TPR;
    using P = Pack<T>;
    constexpr int VEC = P::VEC, NV = kEach / VEC;
    constexpr bool kKeep = NORM && SHIFT;
    static_assert(kEach <= 32, "a warp takes a lane's elements at once");
    __shared__ float s_sum[MOST / 32], s_top[MOST / 32];
    __shared__ unsigned long long s_tops64[2];   // of this row and the next
    __shared__ double s_sum64[MOST / 32];
    const int lane = kBlock ? threadIdx.x : threadIdx.x % kPart, lane32 = threadIdx.x & 31, warps = blockDim.x >> 5;
    const T* w = NORM ? static_cast<const T*>(a.weight) : nullptr;
    const long long first = kBlock ? blockIdx.x : (long long)blockIdx.x * (MOST / kPart) + threadIdx.x / kPart, step = kBlock ? gridDim.x : (long long)gridDim.x * (MOST / kPart);
    // the row's first pack begins at `head`, behind `packs` of them lie `tail` elements
    const int away = SHIFT ? (int)(reinterpret_cast<uintptr_t>(static_cast<const T*>(a.x) + first * a.x_stride) / sizeof(T)) & (VEC - 1) : 0;
    const int head = SHIFT ? min((VEC - away) & (VEC - 1), a.dim) : 0, packs = (a.dim - head) / VEC, tail = a.dim - head - packs * VEC;
    auto begin = [&](int j) { return head + (j * each_row + lane) * VEC; };    // of this thread's pack j in the row
    constexpr int kSingle = !SHIFT ? 0 : kBlock || TPR >= 2 * VEC ? 1 : 2 * VEC / (TPR ? TPR : 1);
    auto single = [&](int q, int of) {                                          // element of thread `of` beside its packs; -1: none
        const int i = of + q * (kBlock ? 0 : kPart);
        return i < VEC ? (i < head ? i : -1) : i < VEC + tail ? head + packs * VEC + i - VEC : -1;
    };
    if (kBlock && threadIdx.x == 0) s_tops64[0] = 0;
    extern __shared__ uint4 s_weight[];   // kKeep: the weight's packs of each thread
    if (kKeep)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            P p;
            p.ones();
            if (w && begin(j) + VEC <= a.dim) p.read_each(w, begin(j));
            s_weight[j * blockDim.x + threadIdx.x] = make_uint4(p.word[0], p.word[1], p.word[2], p.word[3]);
        }
    float alone_w[kSingle + 1];   // the weight of the elements beside the packs
#pragma unroll
    for (int q = 0; q < kSingle; ++q) {
        const int i = single(q, lane);
        alone_w[q] = NORM && w && i >= 0 ? to_float(w[i]) : 1.f;
    }
    auto weighed = [&](int q, float v) { return NORM ? v * alone_w[q] : v; };
    int turn = 0;
    long long row = first;
    // (a part of a warp whose rows have ended stays for the others)
    do {
    const bool live = row < a.n;
    const int dim = live ? a.dim : 0;   // (no pack of a row that is none)
    unsigned long long h[kEach / 2];   // the row, or its sum with the residual, two elements each
    float alone[kSingle + 1];          // and the elements beside its packs
    float mine = 0.f, sum = 0.f;
    {
        const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride;
        const T* r = NORM && a.residual ? static_cast<const T*>(a.residual) + (live ? row : 0) * a.residual_stride : nullptr;
        P px[NV], pr[NORM ? NV : 1], pw[NORM ? NV : 1];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            px[j].zeros();
            if (NORM) { pr[j].zeros(); pw[j].ones(); }
            const int at = begin(j);
            if (at + VEC <= dim) {
                px[j].read(x, at);
                if (NORM && r) pr[j].read(r, at);
                if (NORM && !kKeep && w) pw[j].read(w, at);
            }
        }
#pragma unroll
        for (int q = 0; q < kSingle; ++q) {
            const int i = live ? single(q, lane) : -1;
            alone[q] = i >= 0 ? to_float(x[i]) : 0.f;
            if (NORM && r && i >= 0) alone[q] += to_float(r[i]);
        }
        unsigned long long sums = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (kKeep) pw[j].set(s_weight[j * blockDim.x + threadIdx.x]);
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const int i = (j * VEC + e) / 2;
                h[i] = pair(px[j].get(e), px[j].get(e + 1));
                if (NORM && r) h[i] = add2(h[i], pair(pr[j].get(e), pr[j].get(e + 1)));
                if (NORM) sums = fma2(h[i], h[i], sums);
                const float2 u = halves(NORM ? mul2(h[i], pair(pw[j].get(e), pw[j].get(e + 1))) : h[i]);
                mine = larger(larger(mine, u.x), u.y);
            }
        }
        const float2 s = halves(sums);
        sum = s.x + s.y;
#pragma unroll
        for (int q = 0; q < kSingle; ++q) {
            if (NORM) sum = fmaf(alone[q], alone[q], sum);
            mine = larger(mine, weighed(q, alone[q]));
        }
    }
    float top32 = kPart == 32 ? warp_larger(mine) : lanes_reduce<kPart>(mine, LargerOp());
    if (NORM) sum = lanes_reduce<kPart>(sum, SumOp());
    if constexpr (kBlock) {
        if (lane32 == 0) { s_top[threadIdx.x >> 5] = top32; s_sum[threadIdx.x >> 5] = sum; }
        __syncthreads();
        if (threadIdx.x == 0) s_tops64[(turn + 1) & 1] = 0;
        top32 = warp_larger(lane32 < warps ? s_top[lane32] : 0.f);
        if (NORM) sum = lanes_reduce<32>(lane32 < warps ? s_sum[lane32] : 0.f, SumOp());
    }
    // (a NaN fails every comparison; a row without a norm has no sum to look at)
    bool wild = !(top32 >= kSafeLow && top32 <= kSafeHigh) || (NORM && !(sum >= kSafeLow && sum <= kSafeHigh));
    if (kBlock ? top32 == 0.f : __any_sync(0xffffffffu, top32 == 0.f)) {   // perhaps a row of zeros
        bool some = false;
#pragma unroll
        for (int i = 0; i < kEach / 2; ++i) { const float2 v = halves(h[i]); some = some || v.x != 0.f || v.y != 0.f; }
#pragma unroll
        for (int q = 0; q < kSingle; ++q) some = some || alone[q] != 0.f;
        some = kBlock ? __syncthreads_or(some) : lanes_reduce<kPart>((int)some, MaxOp());
        if (top32 == 0.f && !some) wild = false;
    }

    // For each lane of the warp that needs it: f(lane, its row, element of the row, its value in 32 bits, its sum and value in 64), an element of that
    // lane's packs for each of the 32 (an element < 0: none), and then those beside its packs.
    auto together = [&](bool need, auto&& f) {
        __syncwarp();   // what f writes lies over what its lane wrote, what it reads under what that writes next
        for (unsigned todo = __ballot_sync(0xffffffffu, need && live); todo; todo &= todo - 1) {
            const int whose = __ffs(todo) - 1;
            const long long of = __shfl_sync(0xffffffffu, row, whose);
            const int l = kBlock ? (int)(threadIdx.x & ~31u) + whose : whose % kPart, first_pack = SHIFT ? __shfl_sync(0xffffffffu, head, whose) : 0;
            int i = first_pack + (lane32 / VEC * each_row + l) * VEC + lane32 % VEC, beside = -1;
            if (lane32 >= kEach || i - lane32 % VEC + VEC > a.dim) i = -1;
#pragma unroll
            for (int q = 0; q < kSingle; ++q) {
                const int e = __shfl_sync(0xffffffffu, single(q, lane), whose);
                if (lane32 == q) beside = e;
            }
#pragma unroll 1
            for (int turn = 0; turn < (SHIFT ? 2 : 1); ++turn) {
                if (SHIFT && turn) i = beside;
                float v = 0.f;
                double s64 = 0, v64 = 0;
                if (i >= 0) {
                    const float x = to_float(static_cast<const T*>(a.x)[of * a.x_stride + i]);
                    const float r = NORM && a.residual ? to_float(static_cast<const T*>(a.residual)[of * a.residual_stride + i]) : 0.f;
                    const float by = NORM && w ? to_float(w[i]) : 1.f;
                    v = NORM ? (x + r) * by : x;
                    s64 = (double)x + (double)r;
                    v64 = s64 * (double)by;
                }
                f(whose, of, i, v, s64, v64);
            }
        }
        __syncwarp();
    };
    const float inverse = top32 > 0 ? 127.f / top32 : 0.f;
    signed char* out = a.codes + (live ? row : 0) * a.code_stride;
    float off = 0.f;   // the furthest from a whole number
    const unsigned long long by = pair(inverse, inverse), whole = pair(kRint, kRint), back = pair(-kRint, -kRint), less = pair(-inverse, -inverse);
    unsigned c[kEach];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        P pw;
        if (NORM) pw.ones();
        if (kKeep) pw.set(s_weight[j * blockDim.x + threadIdx.x]);
        else if (NORM && w && begin(j) + VEC <= dim) pw.read_again(w, begin(j));
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
            const int i = (j * VEC + e) / 2;
            unsigned long long u = h[i];
            if (NORM) u = mul2(u, pair(pw.get(e), pw.get(e + 1)));
            const unsigned long long m = fma2(u, by, whole), away = fma2(u, less, add2(m, back));
            const float2 code = halves(m), d = halves(away);
            c[2 * i] = __float_as_uint(code.x);
            c[2 * i + 1] = __float_as_uint(code.y);
            off = fmaxf(fmaxf(off, fabsf(d.x)), fabsf(d.y));
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int at = begin(j);
        if (at + VEC > dim) continue;
        const unsigned* v = c + j * VEC;
        if (!SHIFT || (reinterpret_cast<uintptr_t>(out + at) & (VEC - 1)) == 0) {
            if constexpr (VEC == 8) *reinterpret_cast<uint2*>(out + at) = make_uint2(four(v[0], v[1], v[2], v[3]), four(v[4], v[5], v[6], v[7]));
            else *reinterpret_cast<unsigned*>(out + at) = four(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[at + e] = (signed char)v[e];
        }
    }
#pragma unroll
    for (int q = 0; q < kSingle; ++q) {
        const int i = live ? single(q, lane) : -1;
        const float u = weighed(q, alone[q]), m = fmaf(u, inverse, kRint);
        off = fmaxf(off, fabsf(fmaf(u, inverse, kRint - m)));
        if (i >= 0) out[i] = (signed char)__float_as_uint(m);
    }
    const bool unsure = wild || off > kNearTie<NORM>;
    float scale = !(top32 > 0) ? 0.f : NORM ? top32 / (127.f * sqrtf(sum / (float)a.dim + a.eps)) : top32 / 127.f;
    if (kBlock ? __syncthreads_or(unsure) : __any_sync(0xffffffffu, unsure)) {   // the row's largest magnitude in 64 bits, and the codes that need it
        double top64 = top32;   // exact without a norm
        if (NORM || (kBlock ? wild : __any_sync(0xffffffffu, wild))) {
            unsigned long long t = 0;
            const float near = top32 * kNearTop;
            const bool of_row = kBlock ? true : lanes_reduce<kPart>((int)unsure, MaxOp()) != 0;   // (a part of a warp: the rows that need it)
            together(wild || (NORM && of_row && mine >= near), [&](int whose, long long, int, float v, double, double v64) {
                const bool all = __shfl_sync(0xffffffffu, (int)wild, whose);
                const float least = __shfl_sync(0xffffffffu, near, whose);
                const unsigned long long m = lanes_reduce<32>(all || fabsf(v) >= least ? magnitude(v64) : 0ull, MaxOp());
                if (lane32 == whose) t = max(t, m);
            });
            if constexpr (!kBlock) t = lanes_reduce<kPart>(t, MaxOp());
            else {
                if (t) atomicMax(&s_tops64[turn & 1], t);
                __syncthreads();
                t = s_tops64[turn & 1];
            }
            if (NORM || wild) top64 = __longlong_as_double((long long)t);
        }
        bool dead = false;   // an infinity or a NaN: no codes, and a scale that says so
        if (kBlock ? wild : __any_sync(0xffffffffu, wild)) {
            double s = 0;
            if (NORM) {
                together(wild, [&](int whose, long long, int, float, double s64, double) {
                    const double m = lanes_reduce<32>(s64 * s64, SumOp());
                    if (lane32 == whose) s += m;
                });
                s = lanes_reduce<kPart>(s, SumOp());
                if constexpr (kBlock) {
                    if (lane32 == 0) s_sum64[threadIdx.x >> 5] = s;
                    __syncthreads();
                    s = lanes_reduce<32>(lane32 < warps ? s_sum64[lane32] : 0.0, SumOp());
                }
            }
            if (wild) {
                dead = !(top64 <= 1.7e308) || !(s <= 1.7e308);
                scale = dead ? __int_as_float(0x7fffffff) : top64 > 0 ? (float)(top64 / (NORM ? 127.0 * sqrt(s / a.dim + (double)a.eps) : 127.0)) : 0.f;
            }
        }
        together(unsure, [&](int whose, long long of, int i, float v, double, double v64) {
            const bool all = __shfl_sync(0xffffffffu, (int)wild, whose), none = __shfl_sync(0xffffffffu, (int)dead, whose);
            const double top = __shfl_sync(0xffffffffu, top64, whose);
            const float by = __shfl_sync(0xffffffffu, inverse, whose), m = fmaf(v, by, kRint);
            if (i >= 0 && (all || fabsf(fmaf(v, by, kRint - m)) > kNearTie<NORM>)) a.codes[of * a.code_stride + i] = none || top == 0 ? (signed char)0 : code64(v64, top);
        });
    }
    if (NORM && a.sum) {
        T* to = static_cast<T*>(a.sum) + (live ? row : 0) * a.sum_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (begin(j) + VEC <= dim) P::write(to + begin(j), h + j * (VEC / 2));
#pragma unroll
        for (int q = 0; q < kSingle; ++q)
            if (live && single(q, lane) >= 0) to[single(q, lane)] = from_float<T>(alone[q]);
    }
    if (live && lane == 0) a.scales[row] = scale;
    row += step;
    ++turn;
    } while (kKeep && (kBlock ? row < a.n : __any_sync(0xffffffffu, row < a.n)));
}

// Rows too long for registers, or whose arrays begin at places that differ within a pack: a block a row, which is read again for the codes (from L2, as a rule).  A
// thread takes four elements at once, THREADS apart, or a pack of 16 bytes where rows are whole packs.  Each thread writes only elements it has read itself, so the
// sum may lie over the rows or the residual.  (Element by element and by packs, 2,000 x 40,000 bf16: 137 and 87 us.  4,000 x 20,001 fp32: 151 us with every code in
// 64 bits, 132 with those next to ties alone.)
template <typename T, bool NORM, int THREADS, bool PACKS>
__global__ void __launch_bounds__(THREADS) k_i8_rows_any(RowArgs a) {
    __shared__ double s_sum64[32];
    __shared__ float s_top[32], s_sum[32];
    __shared__ unsigned long long s_top64;
    constexpr int VEC = Pack<T>::VEC, kOnce = PACKS ? VEC : 4, kApart = PACKS ? 1 : THREADS;   // elements of a thread at once, from one to the next
    const int begin = PACKS ? threadIdx.x * VEC : threadIdx.x;
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = NORM && a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    const T* w = NORM ? static_cast<const T*>(a.weight) : nullptr;
    const int lane32 = threadIdx.x & 31;
    if (threadIdx.x == 0) s_top64 = 0;
    // this thread's elements from i on, kOnce of them: sums and values in 32 bits (zeros behind the row's end)
    auto read = [&](int i, float (&h)[kOnce], float (&u)[kOnce]) {
        if constexpr (PACKS) {
            Pack<T> px, pr, pw;
            px.read(x, i);
            if (NORM && r) pr.read(r, i);
            if (NORM && w) pw.read(w, i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[e] = NORM && r ? px.get(e) + pr.get(e) : px.get(e);
                u[e] = NORM && w ? h[e] * pw.get(e) : h[e];
            }
        } else {
        T vx[kOnce], vr[kOnce], vw[kOnce];
#pragma unroll
        for (int e = 0; e < kOnce; ++e) {
            const int at = min(i + e * THREADS, a.dim - 1);
            vx[e] = x[at];
            if (NORM && r) vr[e] = r[at];
            if (NORM && w) vw[e] = w[at];
        }
#pragma unroll
        for (int e = 0; e < kOnce; ++e) {
            h[e] = i + e * THREADS < a.dim ? to_float(vx[e]) : 0.f;
            if (NORM && r && i + e * THREADS < a.dim) h[e] += to_float(vr[e]);
            u[e] = NORM && w ? h[e] * to_float(vw[e]) : h[e];
        }
        }
    };
    auto sum64 = [&](int i) { return (double)to_float(x[i]) + (NORM && r ? (double)to_float(r[i]) : 0.0); };
    auto value64 = [&](int i) { return NORM && w ? sum64(i) * (double)to_float(w[i]) : sum64(i); };
    float mine = 0.f;
    double squares = 0;   // (in fp32 a thread's 256 squares of a long row of alike values were 4e-6 off)
    bool some = false;
#pragma unroll 2
    for (int i = begin; i < a.dim; i += kOnce * THREADS) {
        float h[kOnce], u[kOnce], sum = 0.f;
        read(i, h, u);
#pragma unroll
        for (int e = 0; e < kOnce; ++e) {
            if (i + e * kApart >= a.dim) continue;   // (a weight of infinity times the zeros behind the end would be NaN)
            if (NORM) sum = fmaf(h[e], h[e], sum);
            mine = larger(mine, u[e]);
            some = some || h[e] != 0.f;
        }
        if (NORM) squares += (double)sum;
    }
    float sum = (float)squares;
    float top32 = block_reduce<THREADS>(mine, s_top, LargerOp());
    if (NORM) sum = block_reduce<THREADS>(sum, s_sum, SumOp());
    bool wild = !(top32 >= kSafeLow && top32 <= kSafeHigh) || (NORM && !(sum >= kSafeLow && sum <= kSafeHigh));
    if (top32 == 0.f && !__syncthreads_or(some)) wild = false;   // a row of zeros
    double top64 = top32;
    float scale = !(top32 > 0) ? 0.f : NORM ? top32 / (127.f * sqrtf(sum / (float)a.dim + a.eps)) : top32 / 127.f;
    bool dead = false;
    if (wild) {
        double s = 0;
        unsigned long long t = 0;
        for (int i = threadIdx.x; i < a.dim; i += THREADS) {
            const double h = sum64(i);
            s = fma(h, h, s);
            t = max(t, magnitude(value64(i)));
        }
        if (t) atomicMax(&s_top64, t);
        s = block_reduce<THREADS>(s, s_sum64, SumOp());   // (and its barrier)
        top64 = __longlong_as_double((long long)s_top64);
        dead = !(top64 <= 1.7e308) || (NORM && !(s <= 1.7e308));
        scale = dead ? __int_as_float(0x7fffffff) : top64 > 0 ? (float)(top64 / (NORM ? 127.0 * sqrt(s / a.dim + (double)a.eps) : 127.0)) : 0.f;
    } else if (NORM && top32 > 0.f) {   // the largest in 64 bits, by the lanes of a warp for each of its threads that holds one near fp32's
        const float near = top32 * kNearTop;
        for (unsigned todo = __ballot_sync(0xffffffffu, mine >= near); todo; todo &= todo - 1) {
            unsigned long long t = 0;
            const int of = (int)(threadIdx.x & ~31u) + __ffs(todo) - 1;
            const int first = PACKS ? (of + lane32 / VEC * THREADS) * VEC + lane32 % VEC : of + lane32 * THREADS;
            for (int i = first; i < a.dim; i += 32 * THREADS) t = max(t, magnitude(value64(i)));
            t = lanes_reduce<32>(t, MaxOp());
            if (lane32 == 0) atomicMax(&s_top64, t);
        }
        __syncthreads();
        top64 = __longlong_as_double((long long)s_top64);
    }
    const float inverse = top32 > 0 ? 127.f / top32 : 0.f;
    signed char* out = a.codes + row * a.code_stride;
    for (int i = begin; i < a.dim; i += kOnce * THREADS) {
        float h[kOnce], u[kOnce];
        read(i, h, u);
        unsigned c[kOnce];
        float off = 0.f;
#pragma unroll
        for (int e = 0; e < kOnce; ++e) {
            const float m = fmaf(u[e], inverse, kRint);
            c[e] = __float_as_uint(m);
            off = fmaxf(off, i + e * kApart < a.dim ? fabsf(fmaf(u[e], inverse, kRint - m)) : 0.f);
        }
        if (wild || off > kNearTie<NORM>)
#pragma unroll
            for (int e = 0; e < kOnce; ++e) {
                const float m = __uint_as_float(c[e]);
                if (i + e * kApart < a.dim && (wild || fabsf(fmaf(u[e], inverse, kRint - m)) > kNearTie<NORM>)) c[e] = dead || top64 == 0 ? 0u : (unsigned)code64(value64(i + e * kApart), top64);
            }
        if constexpr (PACKS) {
            if constexpr (VEC == 8) *reinterpret_cast<uint2*>(out + i) = make_uint2(four(c[0], c[1], c[2], c[3]), four(c[4], c[5], c[6], c[7]));
            else *reinterpret_cast<unsigned*>(out + i) = four(c[0], c[1], c[2], c[3]);
            if (NORM && a.sum) {
                unsigned long long pairs[VEC / 2];
#pragma unroll
                for (int e = 0; e < VEC / 2; ++e) pairs[e] = pair(h[2 * e], h[2 * e + 1]);
                Pack<T>::write(static_cast<T*>(a.sum) + row * a.sum_stride + i, pairs);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kOnce; ++e) {
                const int at = i + e * THREADS;
                if (at >= a.dim) break;
                out[at] = (signed char)c[e];
                if (NORM && a.sum) static_cast<T*>(a.sum)[row * a.sum_stride + at] = from_float<T>(h[e]);
            }
        }
    }
    if (threadIdx.x == 0) a.scales[row] = scale;
}

template <typename T, int kEach, int TPR, int MOST, bool NORM, bool SHIFT>
psb_status start(const RowArgs& a, int threads, int sms, cudaStream_t s) {
    if (TPR) threads = MOST;
    const long long rows = TPR ? MOST / (TPR ? TPR : 1) : 1, blocks = (a.n + rows - 1) / rows;
    long long grid = blocks;
    if (NORM && SHIFT) {   // as many blocks as fit, of as many rows each as the others, a multiple of a pack's elements
        const long long fit = (long long)sms * std::max(1, blocks_of<kEach, MOST, NORM, SHIFT>() * MOST / threads), turns = (blocks + fit - 1) / fit;
        grid = (blocks + turns - 1) / turns;
        if (grid < blocks) grid = std::min(blocks, std::max(8ll, std::min((grid + 7) / 8 * 8, fit / 8 * 8)));
    }
    const size_t weight = NORM && SHIFT ? (size_t)threads * kEach * sizeof(T) : 0;
    if (weight > 48 * 1024) PSB_TRY(kernel_shared(reinterpret_cast<const void*>(k_i8_rows<T, kEach, TPR, MOST, NORM, SHIFT>), weight));
    k_i8_rows<T, kEach, TPR, MOST, NORM, SHIFT><<<(unsigned)grid, threads, weight, s>>>(a);
    PSB_LAUNCH_CHECK();
    count_launch();
    return PSB_OK;
}

// TPR threads a row, each with three quarters of the elements where those hold it.  At the power limit, with all the elements and with three quarters:
// 1M x 96 fp32 82.4 and 79.2 us, 500,000 x 96 bf16 with norm 72.7 and 66.8, 60,000 x 768 bf16 with norm 68.8 and 63.8.
template <typename T, int TPR, bool NORM, bool SHIFT>
psb_status start_of(const RowArgs& a, int sms, cudaStream_t s) {
    constexpr int kMost = Pack<T>::VEC == 8 ? 32 : 16;
    if constexpr (!SHIFT)
        if (a.dim <= TPR * kMost / 4 * 3) return start<T, kMost / 4 * 3, TPR, 256, NORM, SHIFT>(a, 0, sms, s);
    return start<T, kMost, TPR, 256, NORM, SHIFT>(a, 0, sms, s);
}

// As few threads a row as hold it in registers, 32 elements of two bytes or 16 of four each, since what a thread does once a row is then shared among
// most (16,384 rows of 8,192 in bf16: 172 us with 32 elements, 212 with 16); more of them, with 16 elements, where rows are too few to fill the
// GPU (one row of 4,096: 3.0 us, with 32 3.6).
template <typename T, bool NORM, bool SHIFT>
psb_status by_length(const RowArgs& a, int sms, cudaStream_t s) {
    constexpr int VEC = Pack<T>::VEC, kMost = VEC == 8 ? 32 : 16;
    const int span = a.dim;
    auto warps = [&](int each) { return ((span + each - 1) / each + 31) / 32 * 32; };   // threads, in whole warps
    if (span > 512 && a.n * (long long)warps(kMost) < 1024ll * sms && warps(16) <= 1024) {
        int threads = warps(16);
        while (threads <= 512 && threads < warps(VEC) && a.n * (long long)threads * 2 <= 1024ll * sms) threads *= 2;   // (all rows at once)
        return start<T, 16, 0, 1024, NORM, SHIFT>(a, std::min(threads, warps(VEC)), sms, s);
    }
    if constexpr (VEC == 8)
        if (span <= 4 * 16) return start<T, 16, 4, 256, NORM, SHIFT>(a, 0, sms, s);
    if (span <= 4 * kMost) return start_of<T, 4, NORM, SHIFT>(a, sms, s);
    if (span <= 8 * kMost) return start_of<T, 8, NORM, SHIFT>(a, sms, s);
    if (span <= 16 * kMost) return start_of<T, 16, NORM, SHIFT>(a, sms, s);
    if (span <= 32 * kMost) return start_of<T, 32, NORM, SHIFT>(a, sms, s);
    if (span <= 256 * kMost) return start<T, kMost, 0, 256, NORM, SHIFT>(a, warps(kMost), sms, s);
    if (span <= 288 * kMost) return start<T, kMost, 0, 288, NORM, SHIFT>(a, warps(kMost), sms, s);
    if (span <= 512 * kMost) return start<T, kMost, 0, 512, NORM, SHIFT>(a, warps(kMost), sms, s);
    return start<T, kMost, 0, 1024, NORM, SHIFT>(a, warps(kMost), sms, s);
}

template <typename T, bool NORM>
psb_status by_layout(const RowArgs& a, int sms, cudaStream_t s) {
    constexpr int VEC = Pack<T>::VEC;
    auto place = [](const void* p, long long each) { return (int)(reinterpret_cast<uintptr_t>(p) / each & (VEC - 1)); };   // within a pack
    const int e = sizeof(T), at = place(a.x, e), step = (int)(a.x_stride & (VEC - 1));
    // the rows' arrays begin at the same place of a pack in every row
    auto as_rows = [&](const void* p, long long stride) { return !p || (place(p, e) == at && (int)(stride & (VEC - 1)) == step); };
    const bool packs = as_rows(a.residual, a.residual_stride) && as_rows(a.sum, a.sum_stride) && place(a.weight, e) == 0;
    const bool plain = packs && at == 0 && step == 0 && a.dim % VEC == 0 && place(a.codes, 1) == 0 && (a.code_stride & (VEC - 1)) == 0;
    if (packs && a.dim <= 1024 * (VEC == 8 ? 32 : 16)) return plain ? by_length<T, NORM, false>(a, sms, s) : by_length<T, NORM, true>(a, sms, s);
    if (plain) k_i8_rows_any<T, NORM, 512, true><<<(unsigned)a.n, 512, 0, s>>>(a);
    else if (a.dim <= 4096) k_i8_rows_any<T, NORM, 128, false><<<(unsigned)a.n, 128, 0, s>>>(a);
    else k_i8_rows_any<T, NORM, 512, false><<<(unsigned)a.n, 512, 0, s>>>(a);
    PSB_LAUNCH_CHECK();
    count_launch();
    return PSB_OK;
}

}  // namespace

// What an element type's file defines.
template <typename T> psb_status launch_i8_rows(const RowArgs& a, bool norm, int sms, cudaStream_t s) {
    return norm ? by_layout<T, true>(a, sms, s) : by_layout<T, false>(a, sms, s);
}

}  // namespace psb
