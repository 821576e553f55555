// MXFP4 x MXFP4 GEMM (w4a4): out = epi(A W^T + bias) on codes of 4 bits with a scale per 32 of them along K.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands in this format: lane l holds the 32 codes (16 bytes) of
// row l & 15, K block l >> 4 of a step of 128, and the scale of that block in a byte of its own.
#include "gemm_common.h"
#include "mxfp4_device.h"

namespace cdit {
namespace {

__device__ __forceinline__ v4f mfma_mx(v4i w, v4i a, v4f acc, int w_scale, int a_scale) {
  const v8i w8 = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const v8i a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a8, acc, 4, 4, 0, w_scale, 0, a_scale);
}

// One element of the output from its sum.
template <int OUT>
__device__ __forceinline__ void store_one(const Mx4Gemm& g, int m, int n, float v) {
  if (g.bias) v += OUT == CDIT_DT_F32 ? static_cast<const float*>(g.bias)[n]
                                      : bias_to_f32<OUT>(static_cast<const uint16_t*>(g.bias)[n]);
  if (g.epilogue & CDIT_EPI_GELU_TANH) v = gelu_tanh(v);
  const int64_t at = (int64_t)m * g.ldo + n;
  if constexpr (OUT == CDIT_DT_F32) {
    static_cast<float*>(g.out)[at] = v;
  } else if constexpr (OUT == CDIT_DT_F16) {
    static_cast<uint16_t*>(g.out)[at] = __builtin_bit_cast(uint16_t, (_Float16)v);
  } else {
    static_cast<uint16_t*>(g.out)[at] = (uint16_t)f32_to_bf16_bits(v);
  }
}

// A wavefront per 32 x 32 outputs, operands straight from memory.
template <int OUT>
__global__ __launch_bounds__(256) void gemm_mxfp4_direct(Mx4Gemm g) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kg = lane >> 4;
  const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 128 + wave * 32;
  if (n0 >= g.N) return;
  const int blocks = g.K / kMxBlock, steps = (g.K + 127) / 128;
  const uint8_t *a[2], *as[2], *w[2], *ws[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = min(m0 + 16 * i + r, g.M - 1), n = min(n0 + 16 * i + r, g.N - 1);
    a[i] = g.a + m * g.lda + 16 * kg;
    as[i] = g.a_scale + m * g.ldas + kg;
    w[i] = g.b + n * g.ldb + 16 * kg;
    ws[i] = g.b_scale + n * g.ldbs + kg;
  }
  v4f acc[2][2] = {};
  for (int s = 0; s < steps; ++s) {
    const bool in = 4 * s + kg < blocks;  // codes behind K count as zeros; the scale rows are padded
    v4i av[2], wv[2];
    int asv[2], wsv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      av[i] = in ? *reinterpret_cast<const v4i*>(a[i] + 64 * (int64_t)s) : v4i{0, 0, 0, 0};
      wv[i] = in ? *reinterpret_cast<const v4i*>(w[i] + 64 * (int64_t)s) : v4i{0, 0, 0, 0};
      asv[i] = as[i][4 * s];
      wsv[i] = ws[i][4 * s];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma_mx(wv[j], av[i], acc[i][j], wsv[j], asv[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + 16 * i + r, n = n0 + 16 * j + 4 * kg + e;
        if (m < g.M && n < g.N) store_one<OUT>(g, m, n, acc[i][j][e]);
      }
}

}  // namespace

int launch_gemm_mxfp4(const Mx4Gemm& g, hipStream_t stream) {
  const dim3 grid((unsigned)((g.N + 127) / 128), (unsigned)((g.M + 31) / 32));
  switch (g.out_dtype) {
    case CDIT_DT_F16: hipLaunchKernelGGL(gemm_mxfp4_direct<CDIT_DT_F16>, grid, dim3(256), 0, stream, g); break;
    case CDIT_DT_F32: hipLaunchKernelGGL(gemm_mxfp4_direct<CDIT_DT_F32>, grid, dim3(256), 0, stream, g); break;
    default: hipLaunchKernelGGL(gemm_mxfp4_direct<CDIT_DT_BF16>, grid, dim3(256), 0, stream, g);
  }
  return 0;
}

}  // namespace cdit
