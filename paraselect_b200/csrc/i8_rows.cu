// Rows to 8-bit codes: checks of arguments and the way to the element type's kernels (i8_rows.cuh).
#include "common.cuh"
#include "kernels.h"

namespace psb {

namespace {

psb_status by_type(const RowArgs& a, int type, bool norm, int sms, cudaStream_t s) {
    if (a.n == 0) return PSB_OK;
    switch (type) {
        case PSB_TYPE_F32: return i8_rows_f32(a, norm, sms, s);
        case PSB_TYPE_F16: return i8_rows_f16(a, norm, sms, s);
        default: return i8_rows_bf16(a, norm, sms, s);
    }
}

size_t type_bytes(int type) { return type == PSB_TYPE_F32 ? 4 : 2; }
bool type_known(int type) { return type >= PSB_TYPE_F32 && type <= PSB_TYPE_BF16; }

constexpr int kMaxRowDim = 131071;   // what psb_i8_matmul takes

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
    return by_type(a, type, false, on.sms, static_cast<cudaStream_t>(stream));
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
    return by_type(a, type, true, on.sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
