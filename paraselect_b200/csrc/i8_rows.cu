// Rows to 8-bit codes with one scale a row, plain or behind a residual addition and a root-mean-square norm:
//   h = x + r,  u = h w,  code = rint(127 u / max|u|) (ties to even),  scale = max|u| / (127 rms),  rms = sqrt(mean h^2 + eps);
// without the norm u = x and scale = max|x| / 127.  The norm's 1/rms is common to the row, so the codes do not depend on it.
//
// Codes are those of 64-bit arithmetic.  A code is first formed in fp32: u with a relative error of 2^-23 at most (one rounding in h,
// one in the product), 127 / max|u| with another 2^-23, the last product with 2^-24, so t is off by less than 127 * 2.5 * 2^-23 =
// 3.8e-5.  Only where t lies within 6e-5 of a tie (one element in 8,000) it is formed again in 64 bits from the row's own values.
// The largest |u| is found in fp32 and then, among the elements within 2^-21 of it, in 64 bits.  Rows whose magnitudes leave fp32's
// safe range go through 64 bits altogether.
//
// Bound by memory: one pass over the row, which stays in registers between the reduction and the codes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace psb {

namespace {

constexpr float kNearTie = 0.5f - 6e-5f;
constexpr float kNearTop = 1.0f - 1.0f / (1 << 21);
constexpr float kSafeLow = 1e-30f, kSafeHigh = 1e30f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC neighbouring elements: one, or 16 bytes.
template <typename T, int VEC> struct Pack {
    static_assert(VEC * sizeof(T) == 16, "16 bytes or one element");
    unsigned word[4];
    __device__ __forceinline__ void read(const T* at) { set(*reinterpret_cast<const uint4*>(at)); }
    // a second time, rather than held in registers
    __device__ __forceinline__ void read_again(const T* at) {
        asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(word[0]), "=r"(word[1]), "=r"(word[2]), "=r"(word[3]) : "l"(at));
    }
    __device__ __forceinline__ void set(uint4 v) { word[0] = v.x; word[1] = v.y; word[2] = v.z; word[3] = v.w; }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(word[e]);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(e & 1 ? word[e >> 1] & 0xffff0000u : word[e >> 1] << 16);
        else { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&word[e >> 1])); return e & 1 ? f.y : f.x; }
    }
    static __device__ __forceinline__ void write(T* at, const float (&v)[VEC]) {
        unsigned o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) o[i] = __float_as_uint(v[i]);
            else if constexpr (std::is_same<T, __nv_bfloat16>::value) { const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); o[i] = *reinterpret_cast<const unsigned*>(&p); }
            else { const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]); o[i] = *reinterpret_cast<const unsigned*>(&p); }
        }
        *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
    }
};
template <typename T> struct Pack<T, 1> {
    float v;
    __device__ __forceinline__ void read(const T* at) { v = to_float(*at); }
    __device__ __forceinline__ void read_again(const T* at) { v = to_float(*at); }
    __device__ __forceinline__ float get(int) const { return v; }
    static __device__ __forceinline__ void write(T* at, const float (&v)[1]) { *at = from_float<T>(v[0]); }
};

struct RowArgs {
    const void* x;
    const void* residual;   // may be null
    const void* weight;     // may be null (ones)
    void* sum;              // may be null; may be x or residual
    signed char* codes;
    float* scales;
    long long n, x_stride, residual_stride, sum_stride, code_stride;
    int dim;
    float eps;
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

// One row for each group of TPR threads, in registers: at most NV packs of VEC elements a thread.  What few elements need - 64 bits next to
// ties, at the top, in rows out of fp32's range - is read again from memory, before the sum is written, by the 32 lanes of a warp for the one
// that found it.  Code for it beside every element took five times the kernel's time, and a thread of its own for it half of the rest, the
// block waiting (16,384 rows of 8,192 in bf16: 789 and 499 us).
template <typename T, int VEC, int NV, int TPR, bool NORM>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_i8_rows(RowArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR;
    using P = Pack<T, VEC>;
    static_assert(TPR <= 32 || TPR == kThreads, "a row's threads are part of a warp or the whole block");
    static_assert(NV * VEC <= 32, "a warp takes a lane's elements at once");
    __shared__ float s_sum[kThreads / 32], s_top[kThreads / 32];
    __shared__ unsigned long long s_top64[kThreads / 32];
    __shared__ double s_sum64[kThreads / 32];
    const int lane = threadIdx.x % TPR, lane32 = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
    const bool live = row < a.n;
    const T* w = NORM ? static_cast<const T*>(a.weight) : nullptr;
    const int dim = live ? a.dim : 0;
    float h[NV][VEC];   // the row, or its sum with the residual
    float sum = 0.f, mine = 0.f;
    {
        const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride;
        const T* r = NORM && a.residual ? static_cast<const T*>(a.residual) + (live ? row : 0) * a.residual_stride : nullptr;
        P px[NV], pr[NORM ? NV : 1], pw[NORM ? NV : 1];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = (j * TPR + lane) * VEC;
            if (at < dim) {
                px[j].read(x + at);
                if (NORM && r) pr[j].read(r + at);
                if (NORM && w) pw[j].read(w + at);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const bool in = (j * TPR + lane) * VEC < dim;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[j][e] = in ? px[j].get(e) : 0.f;
                if (NORM) {
                    if (r && in) h[j][e] += pr[j].get(e);
                    sum = fmaf(h[j][e], h[j][e], sum);
                }
                mine = larger(mine, NORM && w && in ? h[j][e] * pw[j].get(e) : h[j][e]);
            }
        }
    }
    float top32 = mine;
    if constexpr (TPR <= 32) {
        top32 = lanes_reduce<TPR>(top32, LargerOp());
        if (NORM) sum = lanes_reduce<TPR>(sum, SumOp());
    } else {
        top32 = lanes_reduce<32>(top32, LargerOp());
        if (NORM) sum = lanes_reduce<32>(sum, SumOp());
        if (lane32 == 0) { s_top[threadIdx.x >> 5] = top32; s_sum[threadIdx.x >> 5] = sum; }
        __syncthreads();
        top32 = lanes_reduce<kThreads / 32>(s_top[threadIdx.x & (kThreads / 32 - 1)], LargerOp());
        if (NORM) sum = lanes_reduce<kThreads / 32>(s_sum[threadIdx.x & (kThreads / 32 - 1)], SumOp());
    }
    // (a NaN fails every comparison; a row without a norm has no sum to look at)
    bool wild = !(top32 >= kSafeLow && top32 <= kSafeHigh) || (NORM && !(sum >= kSafeLow && sum <= kSafeHigh));
    if (TPR > 32 ? top32 == 0.f : __any_sync(0xffffffffu, top32 == 0.f)) {   // perhaps a row of zeros
        bool some = false;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) some = some || h[j][e] != 0.f;
        some = TPR > 32 ? __syncthreads_or(some) : lanes_reduce<(TPR < 32 ? TPR : 32)>((int)some, MaxOp());
        if (top32 == 0.f && !some) wild = false;
    }

    // For each lane of the warp that needs it: f(lane, its row, element of the row, its value in 32 bits, its sum and value in 64), an element
    // of that lane's for each of the 32 (an element < 0: none).
    auto together = [&](bool need, auto&& f) {
        __syncwarp();   // what f writes lies over what its lane wrote, what it reads under what that writes next
        for (unsigned todo = __ballot_sync(0xffffffffu, need && live); todo; todo &= todo - 1) {
            const int whose = __ffs(todo) - 1;
            const long long of = __shfl_sync(0xffffffffu, row, whose);
            const int l = TPR <= 32 ? whose % TPR : (int)(threadIdx.x & ~31u) + whose;
            int i = (lane32 / VEC * TPR + l) * VEC + lane32 % VEC;
            if (lane32 >= NV * VEC || i >= a.dim) i = -1;
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
        __syncwarp();
    };
    double top64 = top32, mean = NORM ? (double)sum / a.dim : 0;
    // the whole warp or block takes the 64-bit reductions where a row of it needs them
    const bool any_wild = TPR > 32 ? wild : __any_sync(0xffffffffu, wild);
    if (NORM || any_wild) {
        unsigned long long t = 0;
        const float near = top32 * kNearTop;
        together(wild || mine >= near, [&](int whose, long long, int, float v, double, double v64) {
            const bool all = __shfl_sync(0xffffffffu, (int)wild, whose);
            const float least = __shfl_sync(0xffffffffu, near, whose);
            const unsigned long long m = lanes_reduce<32>(all || fabsf(v) >= least ? magnitude(v64) : 0ull, MaxOp());
            if (lane32 == whose) t = m;
        });
        t = TPR <= 32 ? lanes_reduce<(TPR < 32 ? TPR : 32)>(t, MaxOp()) : block_reduce<kThreads>(t, s_top64, MaxOp());
        top64 = __longlong_as_double((long long)t);
    }
    if (NORM && any_wild) {
        double s = 0;
        together(wild, [&](int whose, long long, int, float, double s64, double) {
            const double m = lanes_reduce<32>(s64 * s64, SumOp());
            if (lane32 == whose) s = m;
        });
        s = TPR <= 32 ? lanes_reduce<(TPR < 32 ? TPR : 32)>(s, SumOp()) : block_reduce<kThreads>(s, s_sum64, SumOp());
        if (wild) mean = s / a.dim;
    }
    const bool dead = !(top64 <= 1.7e308) || (NORM && !(mean <= 1.7e308));   // an infinity or a NaN: no codes, and a scale that says so
    const float inverse = top64 > 0 ? 127.f / (float)top64 : 0.f;
    signed char* out = a.codes + (live ? row : 0) * a.code_stride;
    float off = 0.f;   // the furthest from a whole number
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int at = (j * TPR + lane) * VEC;
        if (at >= dim) continue;
        P pw;
        if (NORM && w) pw.read_again(w + at);
        unsigned c[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float t = (NORM && w ? h[j][e] * pw.get(e) : h[j][e]) * inverse, m = t + kRint;
            c[e] = __float_as_uint(m);
            off = fmaxf(off, fabsf(t - (m - kRint)));
        }
        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(out + at) = make_uint2(four(c[0], c[1], c[2], c[3]), four(c[4], c[5], c[6], c[7]));
        else if constexpr (VEC == 4) *reinterpret_cast<unsigned*>(out + at) = four(c[0], c[1], c[2], c[3]);
        else out[at] = (signed char)c[0];
    }
    together(wild || off > kNearTie, [&](int whose, long long of, int i, float v, double, double v64) {
        const bool all = __shfl_sync(0xffffffffu, (int)wild, whose), none = __shfl_sync(0xffffffffu, (int)dead, whose);
        const double top = __shfl_sync(0xffffffffu, top64, whose);
        const float t = v * __shfl_sync(0xffffffffu, inverse, whose);
        if (i >= 0 && (all || fabsf(t - ((t + kRint) - kRint)) > kNearTie)) a.codes[of * a.code_stride + i] = none || top == 0 ? (signed char)0 : code64(v64, top);
    });
    if (NORM && a.sum) {
        T* to = static_cast<T*>(a.sum) + (live ? row : 0) * a.sum_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = (j * TPR + lane) * VEC;
            if (at >= dim) continue;
            P::write(to + at, h[j]);
        }
    }
    if (live && lane == 0) {
        const double by = NORM ? 127.0 * sqrt(mean + (double)a.eps) : 127.0;
        a.scales[row] = dead ? __int_as_float(0x7fffffff) : top64 > 0 ? (float)(top64 / by) : 0.f;
    }
}

// Rows too long for registers: a block a row, element by element, read again for the codes (from L2, as a rule).  Each thread writes only
// elements it has read itself, so the sum may lie over the rows or the residual.
template <typename T, bool NORM>
__global__ void __launch_bounds__(1024) k_i8_rows_long(RowArgs a) {
    __shared__ double s_sum64[32];
    __shared__ unsigned long long s_top64[32];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = NORM && a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    const T* w = NORM ? static_cast<const T*>(a.weight) : nullptr;
    auto sum_of = [&](int i) { return (double)to_float(x[i]) + (r ? (double)to_float(r[i]) : 0.0); };
    double sum = 0;
    unsigned long long t = 0;
    for (int i = threadIdx.x; i < a.dim; i += 1024) {
        const double h = sum_of(i);
        if (NORM) sum = fma(h, h, sum);
        t = max(t, magnitude(w ? h * (double)to_float(w[i]) : h));
    }
    const double top = __longlong_as_double((long long)block_reduce<1024>(t, s_top64, MaxOp()));
    const double mean = NORM ? block_reduce<1024>(sum, s_sum64, SumOp()) / a.dim : 0;
    const bool dead = !(top <= 1.7e308) || !(mean <= 1.7e308);
    if (threadIdx.x == 0) {
        const double by = NORM ? 127.0 * sqrt(mean + (double)a.eps) : 127.0;
        a.scales[row] = dead ? __int_as_float(0x7fffffff) : top > 0 ? (float)(top / by) : 0.f;
    }
    for (int i = threadIdx.x; i < a.dim; i += 1024) {
        const double h = sum_of(i);
        const float h32 = r ? to_float(x[i]) + to_float(r[i]) : to_float(x[i]);
        a.codes[row * a.code_stride + i] = dead || top == 0 ? 0 : code64(w ? h * (double)to_float(w[i]) : h, top);
        if (NORM && a.sum) static_cast<T*>(a.sum)[row * a.sum_stride + i] = from_float<T>(h32);
    }
}

template <typename T, int VEC, int NV, int TPR, bool NORM>
psb_status start(const RowArgs& a, cudaStream_t s) {
    constexpr int threads = TPR < 256 ? 256 : TPR;
    const long long blocks = (a.n + threads / TPR - 1) / (threads / TPR);
    k_i8_rows<T, VEC, NV, TPR, NORM><<<(unsigned)blocks, threads, 0, s>>>(a);
    PSB_LAUNCH_CHECK();
    count_launch();
    return PSB_OK;
}

// Threads a row: the fewest whose registers hold it, 16 elements each; more where rows are too few to fill the GPU.
template <typename T, int VEC, bool NORM>
psb_status by_length(const RowArgs& a, int sms, cudaStream_t s) {
    constexpr int NV = 16 / VEC;
    int tpr = 8;
    if (a.dim > 8 * 16) tpr = 32;
    if (a.dim > 32 * 16) tpr = 256;
    if (a.dim > 256 * 16) tpr = 512;
    if (a.dim > 512 * 16) tpr = 1024;
    while (tpr < 1024 && a.dim > tpr * VEC && a.n * tpr < (long long)sms * 1024) tpr = tpr == 8 ? 32 : tpr == 32 ? 256 : 2 * tpr;
    switch (tpr) {
        case 8: return start<T, VEC, NV, 8, NORM>(a, s);
        case 32: return start<T, VEC, NV, 32, NORM>(a, s);
        case 256: return start<T, VEC, NV, 256, NORM>(a, s);
        case 512: return start<T, VEC, NV, 512, NORM>(a, s);
        default: return start<T, VEC, NV, 1024, NORM>(a, s);
    }
}

template <typename T, bool NORM>
psb_status by_layout(const RowArgs& a, int sms, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    auto at = [](const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; };
    const bool wide = a.dim % VEC == 0 && at(a.x, 16) && a.x_stride % VEC == 0 && at(a.codes, VEC) && a.code_stride % VEC == 0 &&
                      (!a.residual || (at(a.residual, 16) && a.residual_stride % VEC == 0)) && (!a.sum || (at(a.sum, 16) && a.sum_stride % VEC == 0)) && at(a.weight, 16);
    if (a.dim <= 1024 * 16) return wide ? by_length<T, VEC, NORM>(a, sms, s) : by_length<T, 1, NORM>(a, sms, s);
    k_i8_rows_long<T, NORM><<<(unsigned)a.n, 1024, 0, s>>>(a);
    PSB_LAUNCH_CHECK();
    count_launch();
    return PSB_OK;
}

template <bool NORM>
psb_status by_type(const RowArgs& a, int type, int sms, cudaStream_t s) {
    if (a.n == 0) return PSB_OK;
    switch (type) {
        case PSB_TYPE_F32: return by_layout<float, NORM>(a, sms, s);
        case PSB_TYPE_F16: return by_layout<__half, NORM>(a, sms, s);
        default: return by_layout<__nv_bfloat16, NORM>(a, sms, s);
    }
}

size_t type_bytes(int type) { return type == PSB_TYPE_F32 ? 4 : 2; }
bool type_known(int type) { return type >= PSB_TYPE_F32 && type <= PSB_TYPE_BF16; }

constexpr int kMaxRowDim = 131071;   // what psb_i8_matmul takes

// Bytes [begin, end) that `n` rows of `width` bytes span, `stride` bytes apart.
struct Span {
    uintptr_t begin, end;
    Span(const void* p, int64_t n, size_t width, int64_t stride)
        : begin(reinterpret_cast<uintptr_t>(p)), end(begin + (n > 0 ? (uintptr_t)(n - 1) * (uintptr_t)stride + width : 0)) {}
    bool meets(const Span& o) const { return begin < o.end && o.begin < end; }
};

psb_status check_rows(const void* d_rows, int type, int64_t n, int dim, int64_t row_stride, const int8_t* d_codes, int64_t code_stride, const float* d_scales) {
    if (!type_known(type)) return fail(PSB_INVALID_ARGUMENT, "the element type is none of PSB_TYPE_*");
    if (n < 0 || dim <= 0) return fail(PSB_INVALID_ARGUMENT, "rows to encode: a count below zero or rows without elements");
    if (dim > kMaxRowDim || n > 0x7fffffff) return fail(PSB_UNSUPPORTED_SHAPE, "rows to encode: at most 131,071 elements a row and 2^31 - 1 rows");
    if (n > 0 && (!d_rows || !d_codes || !d_scales)) return fail(PSB_INVALID_ARGUMENT, "rows to encode: a null pointer");
    if (row_stride < dim || code_stride < dim) return fail(PSB_INVALID_ARGUMENT, "rows to encode: a stride is less than a row");
    if (reinterpret_cast<uintptr_t>(d_rows) % type_bytes(type) || reinterpret_cast<uintptr_t>(d_scales) % 4)
        return fail(PSB_INVALID_ARGUMENT, "rows to encode: a pointer is not aligned to its elements");
    return PSB_OK;
}

}  // namespace
}  // namespace psb

using namespace psb;

extern "C" {

psb_status psb_i8_encode_rows(const void* d_rows, int type, int64_t n, int dim, int64_t row_stride, int8_t* d_codes, int64_t code_stride, float* d_scales,
                              int device, void* stream) {
    PSB_TRY(check_rows(d_rows, type, n, dim, row_stride, d_codes, code_stride, d_scales));
    const size_t e = type_bytes(type);
    const Span rows(d_rows, n, dim * e, row_stride * e), codes(d_codes, n, dim, code_stride), scales(d_scales, n, 4, 4);
    if (codes.meets(rows) || codes.meets(scales) || scales.meets(rows)) return fail(PSB_INVALID_ARGUMENT, "rows to encode: an output lies over another array");
    DeviceScope on;
    PSB_TRY(on.enter(device));
    RowArgs a{};
    a.x = d_rows; a.codes = reinterpret_cast<signed char*>(d_codes); a.scales = d_scales;
    a.n = n; a.dim = dim; a.x_stride = row_stride; a.code_stride = code_stride;
    return by_type<false>(a, type, on.sms, static_cast<cudaStream_t>(stream));
}

psb_status psb_i8_norm_rows(const void* d_rows, const void* d_residual, const void* d_weight, int type, int64_t n, int dim, int64_t row_stride,
                            int64_t residual_stride, float eps, void* d_sum, int64_t sum_stride, int8_t* d_codes, int64_t code_stride, float* d_scales, int device,
                            void* stream) {
    PSB_TRY(check_rows(d_rows, type, n, dim, row_stride, d_codes, code_stride, d_scales));
    const size_t e = type_bytes(type);
    if ((d_residual && residual_stride < dim) || (d_sum && sum_stride < dim)) return fail(PSB_INVALID_ARGUMENT, "rows to encode: a stride is less than a row");
    if (!(eps >= 0.f) || !(eps <= FLT_MAX)) return fail(PSB_INVALID_ARGUMENT, "the norm's epsilon is negative or not finite");
    for (const void* p : {d_residual, d_weight, (const void*)d_sum})
        if (reinterpret_cast<uintptr_t>(p) % e) return fail(PSB_INVALID_ARGUMENT, "rows to encode: a pointer is not aligned to its elements");
    const Span rows(d_rows, n, dim * e, row_stride * e), codes(d_codes, n, dim, code_stride), scales(d_scales, n, 4, 4);
    const Span residual(d_residual, d_residual ? n : 0, dim * e, residual_stride * e), sum(d_sum, d_sum ? n : 0, dim * e, sum_stride * e);
    const Span weight(d_weight, d_weight && n > 0 ? 1 : 0, dim * e, dim * e);
    const bool over_rows = sum.meets(rows) && !(d_sum == d_rows && sum_stride == row_stride);
    const bool over_residual = sum.meets(residual) && !(d_sum == d_residual && sum_stride == residual_stride);
    if (codes.meets(rows) || codes.meets(residual) || codes.meets(weight) || codes.meets(sum) || codes.meets(scales) || scales.meets(rows) || scales.meets(residual) ||
        scales.meets(weight) || scales.meets(sum) || sum.meets(weight) || over_rows || over_residual)
        return fail(PSB_INVALID_ARGUMENT, "rows to encode: an output lies over another array (the sum may be the rows or the residual themselves)");
    DeviceScope on;
    PSB_TRY(on.enter(device));
    RowArgs a{};
    a.x = d_rows; a.residual = d_residual; a.weight = d_weight; a.sum = d_sum; a.codes = reinterpret_cast<signed char*>(d_codes); a.scales = d_scales;
    a.n = n; a.dim = dim; a.x_stride = row_stride; a.residual_stride = residual_stride; a.sum_stride = sum_stride; a.code_stride = code_stride; a.eps = eps;
    return by_type<true>(a, type, on.sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
