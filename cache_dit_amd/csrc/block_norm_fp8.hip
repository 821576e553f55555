// The block norm that writes h and FP8 codes of y (block_norm_device.h): a row's largest magnitude is taken while its y
// is in registers, so the codes cost one more exchange between the wavefronts of a row and no pass over memory. Bound by HBM: 32760 x 5120
// with an fp32 stream, 1.85 GB, 377 to 387 us, 4.8 TB/s, in place of 392 for the norm with y in bf16 and 79 for a quantizer; one row
// 4.3 in place of 3.7 and 2.6. Some hundred rows, a workgroup each, take what the CUs with most of them take, 4096 values with norms on
// both sides: 256 rows (one a CU) 5.4, 512 8.4, 666 and 768 (three on some or on all) 9.5, in place of 9.1 and 4.4.
#include "block_norm_device.h"

namespace cdit {

int launch_gate_residual_norm_fp8(const cdit_gate_residual_norm_args& a, uint8_t* q, int64_t ld_q, float* scale,
                                  int scale_mode, hipStream_t stream) {
  const Fp8Codes o = {q, ld_q, scale, scale_mode};
  return a.x_dtype == CDIT_DT_F32 ? launch_types<CDIT_DT_F32, CDIT_DT_BF16, true>(a, o, stream)
                                  : launch_types<CDIT_DT_BF16, CDIT_DT_BF16, true>(a, o, stream);
}

}  // namespace cdit
