#include "i8_rows.cuh"

namespace psb {
psb_status i8_rows_bf16(const RowArgs& a, bool norm, int sms, cudaStream_t s) { return launch_i8_rows<__nv_bfloat16>(a, norm, sms, s); }
}  // namespace psb
