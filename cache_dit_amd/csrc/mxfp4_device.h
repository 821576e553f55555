// Device-side arithmetic of microscaled 4-bit floating point (OCP MX, E2M1 elements, one E8M0 scale
// per 32 of them), shared by the quantizer, the GEMMs that read its codes and the block norm.
#ifndef CDIT_MXFP4_DEVICE_H_
#define CDIT_MXFP4_DEVICE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cdit_internal.h"
#include "gemm_common.h"

namespace cdit {
namespace {

constexpr int kMxBlock = 32;     // elements that share a scale
constexpr int kMxNan = 255;      // scale byte of a block with a value that is not finite
constexpr int kMxPad = 127;      // scale bytes behind the last block of a row: 2^0

typedef __bf16 mx_v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 mx_v2h __attribute__((ext_vector_type(2)));
typedef float mx_v2f __attribute__((ext_vector_type(2)));
typedef unsigned int mx_v4u __attribute__((ext_vector_type(4)));
typedef unsigned short mx_v2us __attribute__((ext_vector_type(2)));

// The scale byte of a block from the fp32 bits of its largest magnitude: its exponent less 2, so that
// the largest magnitude lands in [3.5, 7) of the element format, whose largest value is 6. Exponents
// are counted after rounding up at a significand of 1.75: 7 and above would be cut to 6 (an error of
// 1 and more in units of the scale); with the scale doubled it is rounded to 4, off by half at most. Never
// below 1, which keeps 2^(e - 127) and its reciprocal normal fp32 numbers, nor above 252, so that no finite block
// has a value beyond fp32 (magnitudes from 1.75 * 2^127 on are cut to 1.5 * 2^127); 255 (NaN) where the
// magnitude is an infinity or a NaN: the element format has neither, and a block that hid them
// would hand finite numbers on.
__device__ __forceinline__ int mx_exponent(uint32_t amax_bits) {
  const int e = (int)((amax_bits + 0x200000u) >> 23) - 2;
  return amax_bits >= 0x7f800000u ? kMxNan : min(max(e, 1), 252);
}

// 2^(e - 127) as the converters take it: they read the exponent bits alone.
__device__ __forceinline__ float mx_scale_f32(int e) { return __uint_as_float((uint32_t)e << 23); }

// The same, NaN for a block that is not finite.
__device__ __forceinline__ float mx_scale_or_nan(int e) { return e == kMxNan ? __uint_as_float(0x7fc00000u) : mx_scale_f32(e); }

// Eight consecutive elements as they lie in memory (four words of 16-bit types, eight of fp32).
template <int DT>
struct Mx8 {
  uint32_t w[DT == CDIT_DT_F32 ? 8 : 4];
};
// At 16 bytes, or (ANY) wherever an element may be: the hardware takes such accesses.
template <bool ANY>
struct MxPart {
  typedef mx_v4u type;
};
template <>
struct MxPart<true> {
  typedef mx_v4u type __attribute__((aligned(2)));
};
template <int DT, bool ONCE = false, bool ANY = false>  // ONCE: non-temporal, read by nobody else soon
__device__ __forceinline__ Mx8<DT> mx_load8(const void* p) {
  typedef typename MxPart<ANY>::type Part;
  Mx8<DT> v;
  auto load = [](const Part* q) -> mx_v4u { return ONCE ? __builtin_nontemporal_load(q) : *q; };
  const mx_v4u a = load(static_cast<const Part*>(p));
#pragma unroll
  for (int i = 0; i < 4; ++i) v.w[i] = a[i];
  if constexpr (DT == CDIT_DT_F32) {
    const mx_v4u b = load(static_cast<const Part*>(p) + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[4 + i] = b[i];
  }
  return v;
}
// fp32 bits of the largest magnitude; an infinity or NaN gives 0x7f800000 or more.
template <int DT>
__device__ __forceinline__ uint32_t mx_amax8(const Mx8<DT>& v) {
  if constexpr (DT == CDIT_DT_F32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, v.w[i] & 0x7fffffffu);
    return m;
  } else {
    mx_v2us m = {0, 0};  // magnitudes of 16-bit floats order like their bits
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(mx_v2us, v.w[i] & 0x7fff7fffu));
    const uint32_t top = max((uint32_t)m[0], (uint32_t)m[1]);
    if constexpr (DT == CDIT_DT_BF16) return top << 16;
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)top));
  }
}
// The largest of the four lanes of a quad, in all four: two DPP steps.
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));  // [2,3,0,1]
}
// Eight codes, element i in bits 4i .. 4i + 3: the hardware converters divide by the scale (exactly: it
// is a power of two), round to the nearest code, ties to even, and cut to 6. A block with the NaN
// scale has codes 0.
template <int DT>
__device__ __forceinline__ uint32_t mx_codes8(const Mx8<DT>& v, int e) {
  if (e == kMxNan) return 0u;
  const float s = mx_scale_f32(e);
  uint32_t r = 0;
  if constexpr (DT == CDIT_DT_F32) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v.w[0]), __uint_as_float(v.w[1]), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v.w[2]), __uint_as_float(v.w[3]), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v.w[4]), __uint_as_float(v.w[5]), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v.w[6]), __uint_as_float(v.w[7]), s, 3);
  } else if constexpr (DT == CDIT_DT_BF16) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_v2bf, v.w[0]), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_v2bf, v.w[1]), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_v2bf, v.w[2]), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_v2bf, v.w[3]), s, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(mx_v2h, v.w[0]), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(mx_v2h, v.w[1]), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(mx_v2h, v.w[2]), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(mx_v2h, v.w[3]), s, 3);
  }
  return r;
}
// The values eight codes stand for, in the target type (bf16 and fp32: exact; fp16: rounded).
template <int DT>
__device__ __forceinline__ Mx8<DT> mx_values8(uint32_t c, int e) {
  const float s = mx_scale_f32(e);
  Mx8<DT> v;
  if constexpr (DT == CDIT_DT_F32) {
    const mx_v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
    const mx_v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
    const float all[8] = {a[0], a[1], b[0], b[1], d[0], d[1], f[0], f[1]};
#pragma unroll
    for (int i = 0; i < 8; ++i) v.w[i] = e == kMxNan ? 0x7fc00000u : __float_as_uint(all[i]);
  } else if constexpr (DT == CDIT_DT_BF16) {
    v.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0));
    v.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1));
    v.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2));
    v.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3));
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = e == kMxNan ? 0x7fc07fc0u : v.w[i];
  } else {
    v.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 0));
    v.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 1));
    v.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 2));
    v.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 3));
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = e == kMxNan ? 0x7e007e00u : v.w[i];
  }
  return v;
}
template <int DT, bool ONCE = false, bool ANY = false>
__device__ __forceinline__ void mx_store8(void* p, const Mx8<DT>& v) {
  typedef typename MxPart<ANY>::type Part;
  auto store = [](mx_v4u d, Part* q) {
    if (ONCE)
      __builtin_nontemporal_store(d, q);
    else
      *q = d;
  };
  store(mx_v4u{v.w[0], v.w[1], v.w[2], v.w[3]}, static_cast<Part*>(p));
  if constexpr (DT == CDIT_DT_F32) store(mx_v4u{v.w[4], v.w[5], v.w[6], v.w[7]}, static_cast<Part*>(p) + 1);
}

// Eight codes as bf16, times their scale.
__device__ __forceinline__ v8bf mx_to_bf16(uint32_t c, float scale) {
  const v2bf c0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0), c1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
  const v2bf c2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2), c3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
  return v8bf{c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
}
// One element of the output from its sum.
template <int OUT>
__device__ __forceinline__ void store_mx_one(const Mx4Gemm& g, int m, int n, float v) {
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

}  // namespace
}  // namespace cdit
#endif
