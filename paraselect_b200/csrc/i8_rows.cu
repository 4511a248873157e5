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

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };
template <int VEC> struct alignas(VEC) Codes { signed char v[VEC]; };

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

// Reductions over the TPR threads of a row.  Every thread of the block takes part; `slots` holds a value a warp.
template <int TPR, typename V, typename Op>
__device__ __forceinline__ V row_reduce(V v, V* slots, Op op) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) >> 1; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
        __syncthreads();
        v = slots[threadIdx.x & 31 & (TPR / 32 - 1)];
#pragma unroll
        for (int o = TPR / 64; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
        __syncthreads();
    }
    return v;
}
struct MaxOp { template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct SumOp { template <typename V> __device__ V operator()(V a, V b) const { return a + b; } };

// A magnitude's bits: their order as integers is that of the magnitudes, and a NaN's are above all.
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ unsigned long long magnitude(double v) { return (unsigned long long)__double_as_longlong(v) & 0x7fffffffffffffffull; }

__device__ __forceinline__ signed char code64(double u, double top) { return (signed char)(int)rint(127.0 * u / top); }

// What a row's reductions gave.
struct RowTop { double top; float inverse; bool wild, dead; };

// One row for each group of TPR threads, in registers: at most NV packs of VEC elements a thread.
template <typename T, int VEC, int NV, int TPR, bool NORM>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_i8_rows(RowArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR;
    constexpr int kSlots = kThreads / 32;
    using P = Pack<T, VEC>;
    // one set of slots for each group of TPR threads
    __shared__ float s_sum[kSlots];
    __shared__ unsigned s_top[kSlots];
    __shared__ unsigned long long s_top64[kSlots];
    __shared__ double s_sum64[kSlots];
    static_assert(TPR <= 32 || TPR == kThreads, "a row's threads are part of a warp or the whole block");
    const int lane = threadIdx.x % TPR;
    const long long row = (long long)blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
    const bool live = row < a.n;
    const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride;
    const T* r = NORM && a.residual ? static_cast<const T*>(a.residual) + (live ? row : 0) * a.residual_stride : nullptr;
    const T* w = NORM ? static_cast<const T*>(a.weight) : nullptr;
    P px[NV], pr[NV], pw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int at = (j * TPR + lane) * VEC;
        const bool in = live && at < a.dim;
#pragma unroll
        for (int e = 0; e < VEC; ++e) { px[j].v[e] = from_float<T>(0.f); pr[j].v[e] = from_float<T>(0.f); pw[j].v[e] = from_float<T>(1.f); }
        if (in) {
            px[j] = *reinterpret_cast<const P*>(x + at);
            if (NORM) {
                if (r) pr[j] = *reinterpret_cast<const P*>(r + at);
                if (w) pw[j] = *reinterpret_cast<const P*>(w + at);
            }
        }
    }
    auto value = [&](int j, int e) { return NORM ? (to_float(px[j].v[e]) + to_float(pr[j].v[e])) * to_float(pw[j].v[e]) : to_float(px[j].v[e]); };
    auto value64 = [&](int j, int e) {
        return NORM ? ((double)to_float(px[j].v[e]) + (double)to_float(pr[j].v[e])) * (double)to_float(pw[j].v[e]) : (double)to_float(px[j].v[e]);
    };
    float sum = 0.f;
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (NORM) { const float h = to_float(px[j].v[e]) + to_float(pr[j].v[e]); sum = fmaf(h, h, sum); }
            top = max(top, magnitude(value(j, e)));
        }
    top = row_reduce<TPR>(top, s_top, MaxOp());
    if (NORM) sum = row_reduce<TPR>(sum, s_sum, SumOp());
    const float top32 = __uint_as_float(top);
    // (a NaN fails every comparison; a row without a norm has no sum to look at)
    const bool wild = !(top32 >= kSafeLow && top32 <= kSafeHigh) || (NORM && !(sum >= kSafeLow && sum <= kSafeHigh));
    double top64 = top32, mean = NORM ? (double)sum / a.dim : 0;
    // The whole block takes the 64-bit reductions where a row of it needs them.
    const bool any_wild = TPR > 32 ? wild : __any_sync(0xffffffffu, wild);
    if (NORM || any_wild) {
        unsigned long long t = 0;
        const float near = wild ? -1.f : top32 * kNearTop;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (wild || fabsf(value(j, e)) >= near) t = max(t, magnitude(value64(j, e)));
        top64 = __longlong_as_double((long long)row_reduce<TPR>(t, s_top64, MaxOp()));
    }
    if (NORM && any_wild) {
        double s = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) { const double h = (double)to_float(px[j].v[e]) + (double)to_float(pr[j].v[e]); s = fma(h, h, s); }
        s = row_reduce<TPR>(s, s_sum64, SumOp());
        if (wild) mean = s / a.dim;
    }
    if (!live) return;
    const bool dead = !(top64 <= 1.7e308) || (NORM && !(mean <= 1.7e308));   // an infinity or a NaN: no codes, and a scale that says so
    if (lane == 0) {
        const double by = NORM ? 127.0 * sqrt(mean + (double)a.eps) : 127.0;
        a.scales[row] = dead ? __int_as_float(0x7fffffff) : top64 > 0 ? (float)(top64 / by) : 0.f;
    }
    const float inverse = 127.f / (float)top64;
    signed char* out = a.codes + row * a.code_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int at = (j * TPR + lane) * VEC;
        if (at >= a.dim) continue;
        Codes<VEC> c;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float t = value(j, e) * inverse, q = rintf(t);
            int code = (int)q;
            if (wild || fabsf(t - q) > kNearTie) code = dead || top64 == 0 ? 0 : code64(value64(j, e), top64);
            c.v[e] = (signed char)code;
        }
        *reinterpret_cast<Codes<VEC>*>(out + at) = c;
        if (NORM && a.sum) {
            P s;
#pragma unroll
            for (int e = 0; e < VEC; ++e) s.v[e] = from_float<T>(to_float(px[j].v[e]) + to_float(pr[j].v[e]));
            *reinterpret_cast<P*>(static_cast<T*>(a.sum) + row * a.sum_stride + at) = s;
        }
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
    const double top = __longlong_as_double((long long)row_reduce<1024>(t, s_top64, MaxOp()));
    const double mean = NORM ? row_reduce<1024>(sum, s_sum64, SumOp()) / a.dim : 0;
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

// Threads a row: the fewest whose registers hold it; more where rows are too few to fill the GPU.
template <typename T, int VEC, int NV, bool NORM>
psb_status by_length(const RowArgs& a, int sms, cudaStream_t s) {
    constexpr int each = VEC * NV;
    int tpr = 8;
    if (a.dim > 8 * each) tpr = 32;
    if (a.dim > 32 * each) tpr = 256;
    if (a.dim > 256 * each) tpr = 512;
    if (a.dim > 512 * each) tpr = 1024;
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
    if (wide && a.dim <= 1024 * VEC * 4) return by_length<T, VEC, 4, NORM>(a, sms, s);
    if (a.dim <= 1024 * 16) return by_length<T, 1, 16, NORM>(a, sms, s);
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
