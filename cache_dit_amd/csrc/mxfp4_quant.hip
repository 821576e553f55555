// MXFP4 quantizer and its inverse (include/cdit_hip.h): both are bound by HBM.
//
// A lane takes 8 consecutive elements (16 bytes of a 16-bit type), so that a wavefront reads 1 KiB in a
// row; the four lanes of a quad hold the 32 elements of a block, whose largest magnitude meets in two DPP
// steps; the hardware converters do scaling and rounding. Nothing goes through LDS.
#include <algorithm>

#include "cdit_internal.h"
#include "mxfp4_device.h"

namespace cdit {
namespace {

constexpr int kThreads = 256;

// Which pieces of 8 elements a workgroup takes: `span` of a run of `rows` rows, walked as one line of rows * per_row pieces, so that
// short rows share a workgroup and long ones are shared. Piece -> row by a multiplication: magic = ceil(2^32 / per_row) is exact
// while piece * per_row < 2^32 (at most 2^11 pieces where rows > 1).
struct Runs {
  int rows, per_row, span;
  uint32_t magic;
  dim3 grid(int64_t M) const {
    return dim3((unsigned)((M + rows - 1) / rows), (unsigned)((rows * per_row + span - 1) / span));
  }
};
// 2048 pieces a workgroup, eight a thread, where there are many; one a thread where that leaves CUs idle.
Runs runs_of(int64_t M, int64_t K, int cus) {
  const int per_row = (int)(K / 8);
  const int rows = per_row >= 1024 ? 1 : 2048 / per_row;
  const int64_t pieces = M * per_row, wanted = 4 * (int64_t)cus;
  const int span = (int)std::min<int64_t>(2048, std::max<int64_t>(kThreads, (pieces / wanted + kThreads - 1) / kThreads * kThreads));
  return {rows, per_row, span, (uint32_t)(((uint64_t(1) << 32) + per_row - 1) / per_row)};
}
__device__ __forceinline__ void locate(const Runs& r, uint32_t piece, uint32_t* row, uint32_t* at) {
  *row = r.rows == 1 ? 0u : __umulhi(piece, r.magic);
  *at = piece - *row * (uint32_t)r.per_row;
}

// ONCE: non-temporal accesses to the side that is not in 4 bits. For 16-bit types above 64 MB, us: quantizer 32760 x 5120 84.0 ->
// 71.9 (5.9 TB/s), 32760 x 13824 213 -> 187 (6.15); inverse 83.7 -> 66.1 (6.4), 210 -> 165 (6.9). Below it makes no difference (4608
// x 5120 11.4 and 11.3; 11.1 and 10.1); with fp32, where a lane's 32 bytes take two instructions on the same lines, it costs 20 to
// 40 %. fp32 without: 4608 x 5120 16.9 (6.3) and 18.7 (5.7), 32760 x 5120 147 (5.2) and 200 (3.8).
constexpr int64_t kOnceBytes = (int64_t)64 << 20;
template <int DT, bool ONCE>
__global__ __launch_bounds__(kThreads) void mxfp4_quant_rows(const uint8_t* __restrict__ x, int64_t ld_x,
                                                             uint8_t* __restrict__ codes, int64_t ld_codes,
                                                             uint8_t* __restrict__ scales, int64_t ld_scales,
                                                             int64_t M, Runs r) {
  constexpr int ES = DT == CDIT_DT_F32 ? 4 : 2, U = 4;  // pieces of a thread in flight
  const int64_t row0 = (int64_t)blockIdx.x * r.rows;
  const uint32_t n = (uint32_t)min((int64_t)r.rows, M - row0) * (uint32_t)r.per_row, first = blockIdx.y * (uint32_t)r.span;
  const uint32_t end = min(n, first + (uint32_t)r.span);
  const int blocks = r.per_row / 4;
  for (uint32_t p0 = first + threadIdx.x; p0 < end; p0 += U * kThreads) {
    Mx8<DT> v[U] = {};
    int64_t row[U];
    uint32_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t dr;
      locate(r, p0 + u * kThreads, &dr, &at[u]);
      row[u] = row0 + dr;
      if (p0 + u * kThreads < end) v[u] = mx_load8<DT, ONCE>(x + (row[u] * ld_x + (int64_t)at[u] * 8) * ES);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (per_row is a multiple of 4: a quad is in the row, and in the loop, as a whole)
      const int e = mx_exponent(mx_quad_max(mx_amax8<DT>(v[u])));
      if (p0 + u * kThreads >= end) continue;
      const uint32_t c = mx_codes8<DT>(v[u], e);
      *reinterpret_cast<uint32_t*>(codes + row[u] * ld_codes + (int64_t)at[u] * 4) = c;
      if (at[u] % 4 == 0) {
        uint8_t* const s = scales + row[u] * ld_scales;
        const int b = at[u] / 4;
        s[b] = (uint8_t)e;
        if (b == blocks - 1)
          for (int pad = blocks; pad % 4 != 0; ++pad) s[pad] = (uint8_t)kMxPad;
      }
    }
  }
}

template <int DT, bool ONCE>
__global__ __launch_bounds__(kThreads) void mxfp4_dequant_rows(const uint8_t* __restrict__ codes, int64_t ld_codes,
                                                               const uint8_t* __restrict__ scales, int64_t ld_scales,
                                                               uint8_t* __restrict__ out, int64_t ld_out, int64_t M,
                                                               Runs r) {
  constexpr int ES = DT == CDIT_DT_F32 ? 4 : 2, U = 4;
  const int64_t row0 = (int64_t)blockIdx.x * r.rows;
  const uint32_t n = (uint32_t)min((int64_t)r.rows, M - row0) * (uint32_t)r.per_row, first = blockIdx.y * (uint32_t)r.span;
  const uint32_t end = min(n, first + (uint32_t)r.span);
  for (uint32_t p0 = first + threadIdx.x; p0 < end; p0 += U * kThreads) {
    uint32_t c[U] = {}, at[U];
    int e[U] = {};
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t dr;
      locate(r, p0 + u * kThreads, &dr, &at[u]);
      row[u] = row0 + dr;
      if (p0 + u * kThreads < end) {
        c[u] = *reinterpret_cast<const uint32_t*>(codes + row[u] * ld_codes + (int64_t)at[u] * 4);
        e[u] = scales[row[u] * ld_scales + at[u] / 4];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p0 + u * kThreads < end)
        mx_store8<DT, ONCE>(out + (row[u] * ld_out + (int64_t)at[u] * 8) * ES, mx_values8<DT>(c[u], e[u]));
  }
}
}  // namespace

int launch_mxfp4_quant(const void* x, int dtype, int64_t M, int64_t K, int64_t ld_x, void* codes, int64_t ld_codes,
                       void* scales, int64_t ld_scales, hipStream_t stream) {
  const int cus = cu_count();
  if (cus <= 0) {
    set_error("cannot query the CU count of the current device");
    return CDIT_EHIP;
  }
  const Runs r = runs_of(M, K, cus);
  const dim3 grid = r.grid(M);
  const bool once = 2 * M * K > kOnceBytes;
#define CDIT_MXQ(DT, ONCE)                                                                                          \
  hipLaunchKernelGGL((mxfp4_quant_rows<DT, ONCE>), grid, dim3(kThreads), 0, stream, static_cast<const uint8_t*>(x), \
                     ld_x, static_cast<uint8_t*>(codes), ld_codes, static_cast<uint8_t*>(scales), ld_scales, M, r)
  if (dtype == CDIT_DT_F32)
    CDIT_MXQ(CDIT_DT_F32, false);
  else if (dtype == CDIT_DT_BF16 && once)
    CDIT_MXQ(CDIT_DT_BF16, true);
  else if (dtype == CDIT_DT_BF16)
    CDIT_MXQ(CDIT_DT_BF16, false);
  else if (once)
    CDIT_MXQ(CDIT_DT_F16, true);
  else
    CDIT_MXQ(CDIT_DT_F16, false);
#undef CDIT_MXQ
  return 0;
}

int launch_mxfp4_dequant(const void* codes, int64_t ld_codes, const void* scales, int64_t ld_scales, int64_t M, int64_t K,
                         void* out, int dtype, int64_t ld_out, hipStream_t stream) {
  const int cus = cu_count();
  if (cus <= 0) {
    set_error("cannot query the CU count of the current device");
    return CDIT_EHIP;
  }
  const Runs r = runs_of(M, K, cus);
  const dim3 grid = r.grid(M);
  const bool once = 2 * M * K > kOnceBytes;
#define CDIT_MXD(DT, ONCE)                                                                                               \
  hipLaunchKernelGGL((mxfp4_dequant_rows<DT, ONCE>), grid, dim3(kThreads), 0, stream, static_cast<const uint8_t*>(codes), \
                     ld_codes, static_cast<const uint8_t*>(scales), ld_scales, static_cast<uint8_t*>(out), ld_out, M, r)
  if (dtype == CDIT_DT_F32)
    CDIT_MXD(CDIT_DT_F32, false);
  else if (dtype == CDIT_DT_BF16 && once)
    CDIT_MXD(CDIT_DT_BF16, true);
  else if (dtype == CDIT_DT_BF16)
    CDIT_MXD(CDIT_DT_BF16, false);
  else if (once)
    CDIT_MXD(CDIT_DT_F16, true);
  else
    CDIT_MXD(CDIT_DT_F16, false);
#undef CDIT_MXD
  return 0;
}

}  // namespace cdit
