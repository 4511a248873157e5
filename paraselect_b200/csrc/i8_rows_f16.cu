#include "i8_rows.cuh"

namespace psb {
psb_status i8_rows_f16(const RowArgs& a, bool norm, int sms, cudaStream_t s) { return launch_i8_rows<__half>(a, norm, sms, s); }
}  // namespace psb
