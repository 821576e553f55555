// Weight-only GEMM with an MXFP4 weight (w4a16): out = epi(X W^T + bias), X bf16.
//
// The weight's codes become bf16 with v_cvt_scalef32_pk_bf16_fp4, which applies the block's scale (exact: a code
// has two significant bits), and are multiplied with v_mfma_f32_16x16x32_bf16. Lane l holds row l & 15; of a step of
// 128 along K its 16 bytes of codes are block l >> 4, 32 consecutive k, which feed four instructions of 8 k each.
#include "gemm_common.h"
#include "mxfp4_device.h"

namespace cdit {
namespace {

// The scale of a block as the converter takes it; NaN for a NaN block.
__device__ __forceinline__ float mx_weight_scale(int e) { return e == kMxNan ? __uint_as_float(0x7fc00000u) : mx_scale_f32(e); }

// A wavefront per 32 x 32 outputs, operands straight from memory.
__global__ __launch_bounds__(256) void gemm_w4a16_direct(Mx4Gemm g) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kg = lane >> 4;
  const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 128 + wave * 32;
  if (n0 >= g.N) return;
  const int blocks = g.K / kMxBlock, steps = (g.K + 127) / 128;
  const uint8_t *a[2], *w[2], *ws[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = min(m0 + 16 * i + r, g.M - 1), n = min(n0 + 16 * i + r, g.N - 1);
    a[i] = g.a + 2 * m * g.lda + 64 * kg;
    w[i] = g.b + n * g.ldb + 16 * kg;
    ws[i] = g.b_scale + n * g.ldbs + kg;
  }
  v4f acc[2][2] = {};
  for (int s = 0; s < steps; ++s) {
    const bool in = 4 * s + kg < blocks;  // behind K: zeros in both operands
    v8bf av[2][4];
    v4u wv[2];
    float wsv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v4u z = {0, 0, 0, 0};
        av[i][q] = __builtin_bit_cast(v8bf, in ? *reinterpret_cast<const v4u*>(a[i] + 256 * (int64_t)s + 16 * q) : z);
      }
      wv[i] = in ? *reinterpret_cast<const v4u*>(w[i] + 64 * (int64_t)s) : v4u{0, 0, 0, 0};
      wsv[i] = in ? mx_weight_scale(ws[i][4 * s]) : 1.0f;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const v8bf b = mx_to_bf16(wv[j][q], wsv[j]);
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, av[i][q], acc[i][j], 0, 0, 0);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + 16 * i + r, n = n0 + 16 * j + 4 * kg + e;
        if (m >= g.M || n >= g.N) continue;
        float v = acc[i][j][e];
        if (g.bias) v += bias_to_f32<CDIT_DT_BF16>(static_cast<const uint16_t*>(g.bias)[n]);
        if (g.epilogue & CDIT_EPI_GELU_TANH) v = gelu_tanh(v);
        static_cast<uint16_t*>(g.out)[(int64_t)m * g.ldo + n] = (uint16_t)f32_to_bf16_bits(v);
      }
}

}  // namespace

int launch_gemm_w4a16(const Mx4Gemm& g, int variant, hipStream_t stream) {
  if (variant < 0 && mx_rows_fit(g.M)) return launch_gemm_w4a16_rows(g, stream);
  const dim3 grid((unsigned)((g.N + 127) / 128), (unsigned)((g.M + 31) / 32));
  hipLaunchKernelGGL(gemm_w4a16_direct, grid, dim3(256), 0, stream, g);
  return 0;
}

}  // namespace cdit
