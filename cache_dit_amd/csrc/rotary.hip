// Rotary positions of queries and keys (include/cdit_hip.h, cdit_rotary): pairs (a, b) of a head's values are turned by an
// angle of the token's position, optionally behind an RMSNorm of the head. Bound by HBM: q and k are read once and written
// once.
//
//   v = x                     or  x / sqrt(mean(x^2) + eps) * weight
//   (a, b) -> scale (a cos t - b sin t, a sin t + b cos t),  t = position[axis of the pair] * inv_freq[pair]
//
// The angles are not read from a table that grows with the context but made here, once per token and pair, and used for
// all heads: the position times the frequency in turns, in fp64 (three roundings), so that what is left behind the whole turns is
// exact to 2^-51 of the angle (at position 2^20 and frequency 1 to 7e-11 of a turn; in fp32 it would be 2 % of one). The rest, at
// most an eighth of a turn, is rounded to fp32, 2^-24 of it, and its sine and cosine are their Taylor series in fp32: what an output in
// fp32 loses to that is a unit or two in its last place, and one in 16 bits nothing.
#include <algorithm>

#include "gemm_common.h"
#include "mxfp4_device.h"
#include "quant_device.h"

namespace cdit {
namespace {

typedef cdit_rotary_args Args;

constexpr int kThreads = 256;
// Heads a lane has under way. us, 2 x 4096 tokens of 20 + 20 heads of 128 with norms (168 MB) and 32760 of 40 + 40 (1.34 GB): 1 39.9 and
// 241, 2 35.2 and 239 (5.6 TB/s), 4 38.6 and 257, 8 39.9 and 259. One token 2.8.
constexpr int kUnits = 2;
constexpr int kMostTokens = 16; // of a workgroup

// cos and sin of 2 pi t. The quarter turns are taken off exactly; |w| <= 1/8, |z| <= pi/4, where the first terms left out
// are below 2e-9 (sine: z^11 / 11!) and 2e-10 (cosine: z^12 / 12!).
__device__ __forceinline__ float2 turn(double t) {
  const double quarter = rint(4.0 * t);
  const float z = (float)(t - 0.25 * quarter) * 6.283185307179586f, z2 = z * z;
  float s = __fmaf_rn(z2, 1.0f / 362880, -1.0f / 5040);
  s = __fmaf_rn(z2, s, 1.0f / 120);
  s = __fmaf_rn(z2, s, -1.0f / 6);
  s = __fmaf_rn(z2 * z, s, z);
  float c = __fmaf_rn(z2, -1.0f / 3628800, 1.0f / 40320);
  c = __fmaf_rn(z2, c, -1.0f / 720);
  c = __fmaf_rn(z2, c, 1.0f / 24);
  c = __fmaf_rn(z2, c, -0.5f);
  c = __fmaf_rn(z2, c, 1.0f);
  // quarter mod 4: exact, whatever its size
  const int n = (int)(quarter - 4.0 * floor(0.25 * quarter));
  const float co = n & 1 ? s : c, si = n & 1 ? c : s;
  return float2{n == 1 || n == 2 ? -co : co, n >= 2 ? -si : si};
}

__device__ __forceinline__ double position_at(const Args& a, int64_t at) {
  if (a.position_type == CDIT_POS_I32) return (double)static_cast<const int32_t*>(a.positions)[at];
  if (a.position_type == CDIT_POS_I64) return (double)static_cast<const int64_t*>(a.positions)[at];
  return (double)static_cast<const float*>(a.positions)[at];
}

// n of the 8 elements at p; eight at once where there are eight (16 bytes, aligned unless ANY).
template <int DT, bool ANY>
__device__ __forceinline__ Mx8<DT> load_piece(const uint8_t* p, int n) {
  if (!ANY || n == 8) return mx_load8<DT, false, ANY>(p);
  Mx8<DT> v = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= n) continue;
    if constexpr (DT == CDIT_DT_F32)
      v.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    else
      v.w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
  }
  return v;
}
template <int DT, bool ANY>
__device__ __forceinline__ void store_piece(uint8_t* p, int n, const Mx8<DT>& v) {
  if (!ANY || n == 8) {
    mx_store8<DT, false, ANY>(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= n) continue;
    if constexpr (DT == CDIT_DT_F32)
      reinterpret_cast<uint32_t*>(p)[i] = v.w[i];
    else
      reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(v.w[i / 2] >> (16 * (i & 1)));
  }
}
template <int DT>
__device__ __forceinline__ float value(const Mx8<DT>& v, int i) {
  if constexpr (DT == CDIT_DT_F32) return __uint_as_float(v.w[i]);
  if constexpr (DT == CDIT_DT_BF16) return i & 1 ? bf16_hi(v.w[i / 2]) : bf16_lo(v.w[i / 2]);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(v.w[i / 2] >> (16 * (i & 1))));
}
template <int DT>
__device__ __forceinline__ Mx8<DT> packed(const float* f) {
  Mx8<DT> v;
  if constexpr (DT == CDIT_DT_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v.w[i] = DT == CDIT_DT_BF16 ? pack_bf16x2(f[2 * i], f[2 * i + 1]) : pack_f16x2(f[2 * i], f[2 * i + 1]);
  }
  return v;
}

// Sum over the 2^log lanes of a head, in all of them.
__device__ __forceinline__ float head_sum(float v, int log) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  if (log > 0) v += dpp(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  if (log > 1) v += dpp(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  if (log > 2) v += dpp(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  if (log > 3) v += dpp(v, std::integral_constant<int, 0x140>{});  // row_mirror
  if (log > 4) v += __shfl_xor(v, 16);
  if (log > 5) v += __shfl_xor(v, 32);
  return v;
}

// A workgroup takes `tokens` tokens of a sequence and `heads` of q's and k's heads (k's behind q's). The tokens' sines and
// cosines go through LDS. A head belongs to 2^log lanes, each with two pieces of 8 elements: 8 pairs (halves: a's and b's;
// neighbours: 16 elements in a row), or 16 elements that stay as they are.
//
// ANY: pieces that start anywhere. The last 8 pairs end with the pairs and begin with some of the lane's before, which are
// turned and stored twice, alike, and counted once in the norm; fewer than 8 are taken one by one.
template <int DT, bool ANY>
__global__ __launch_bounds__(kThreads) void rotary_heads(Args a, int tokens, int heads, int tiles, int log) {
  constexpr int ES = DT == CDIT_DT_F32 ? 4 : 2;
  extern __shared__ float shared[];
  const int pairs = a.rot / 2;
  float2* const turns = reinterpret_cast<float2*>(shared);  // [tokens][pairs]
  float* const weights = shared + 2 * tokens * pairs;       // [2][D]
  const int64_t batch = blockIdx.x / tiles, s0 = (int64_t)(blockIdx.x % tiles) * tokens;
  const int here = (int)min((int64_t)tokens, a.S - s0);
  const int h0 = blockIdx.y * heads, all = a.heads[0] + a.heads[1], hc = min(heads, all - h0);

  const float inv_pairs = 1.0f / (float)max(pairs, 1);
  for (int i = threadIdx.x; i < here * pairs; i += kThreads) {
    // (i + 1/2) / pairs is at least 1 / (2 pairs) off a whole number, its rounding error below 2^-22 of it: i < 2^13
    const int t = (int)(((float)i + 0.5f) * inv_pairs), p = i - t * pairs;
    const int64_t s = s0 + t;
    float2 cs;
    if (a.inv_freq) {
      int axis = 0;
      while (axis < a.axes - 1 && p >= a.section_end[axis]) ++axis;
      const double pos = position_at(a, batch * a.position_stride_b + s * a.position_stride_s + axis * a.position_stride_axis);
      cs = turn(pos * (a.inv_freq[p] * 0.15915494309189535));
    } else {
      const int64_t at = batch * a.table_stride_b + s * a.table_stride_s + p * a.table_stride_p;
      cs = float2{a.cos[at], a.sin[at]};
    }
    turns[i] = float2{cs.x * a.scale, cs.y * a.scale};
  }
#pragma unroll
  for (int w = 0; w < 2; ++w)
    if (a.weight[w])
      for (int i = threadIdx.x; i < a.D; i += kThreads)
        weights[w * a.D + i] = a.weight_f32 ? static_cast<const float*>(a.weight[w])[i]
                               : DT == CDIT_DT_BF16 ? bf16_lo(static_cast<const uint16_t*>(a.weight[w])[i])
                                                    : (float)static_cast<const _Float16*>(a.weight[w])[i];
  __syncthreads();

  // this lane's pieces: first element, how many, how many of them an earlier lane has
  const int lane = threadIdx.x & ((1 << log) - 1), group = threadIdx.x >> log, groups = kThreads >> log;
  const int turning = (pairs + 7) / 8;
  const bool turns_here = lane < turning, half = a.layout == CDIT_ROTARY_HALF;
  int p0 = 0, at0, at1, n0 = 8, n1 = 8, skip0 = 0, skip1 = 0;
  if (turns_here) {
    p0 = 8 * lane;
    if (ANY) {
      p0 = max(min(p0, pairs - 8), 0);
      const int n = min(pairs, 8), again = 8 * lane - p0;
      n0 = half ? n : min(2 * n, 8);
      n1 = half ? n : max(2 * n - 8, 0);
      skip0 = half ? again : min(2 * again, 8);
      skip1 = half ? again : max(2 * again - 8, 0);
    }
    at0 = half ? p0 : 2 * p0;
    at1 = half ? pairs + p0 : 2 * p0 + 8;
  } else {
    at0 = a.rot + 16 * (lane - turning);
    at1 = at0 + 8;
    if (ANY) {
      auto place = [&](int& at, int& n, int& skip) {
        const int from = at;
        n = min(max(a.D - at, 0), 8);
        if (n > 0 && n < 8 && a.D - a.rot >= 8) {
          at = a.D - 8;
          n = 8;
        }
        skip = n > 0 ? from - at : 0;
      };
      place(at0, n0, skip0);
      place(at1, n1, skip1);
    } else if (at0 >= a.D) {
      n0 = n1 = 0;
    }
  }
  const bool live = n0 > 0;
  const int units = here * hc;
  const float inv_hc = 1.0f / (float)hc, inv_d = 1.0f / (float)a.D;

  for (int u0 = group; u0 - group < units; u0 += groups * kUnits) {  // (whole wavefronts: the lanes of a head exchange sums)
    Mx8<DT> r0[kUnits], r1[kUnits];
    int tok[kUnits], head[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int u = u0 + k * groups;
      tok[k] = (int)(((float)u + 0.5f) * inv_hc);  // u < 2^21
      head[k] = h0 + u - tok[k] * hc;
      r0[k] = {};
      r1[k] = {};
      if (u < units && live) {
        const int w = head[k] >= a.heads[0];
        const int h = w ? head[k] - a.heads[0] : head[k];
        const uint8_t* const p = static_cast<const uint8_t*>(w ? a.x[1] : a.x[0]) +
                                 (batch * (w ? a.stride_b[1] : a.stride_b[0]) + (s0 + tok[k]) * (w ? a.stride_s[1] : a.stride_s[0]) +
                                  h * (w ? a.stride_h[1] : a.stride_h[0])) * ES;
        r0[k] = load_piece<DT, ANY>(p + at0 * ES, n0);
        if (!ANY || n1 > 0) r1[k] = load_piece<DT, ANY>(p + at1 * ES, n1);
      }
    }
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int u = u0 + k * groups;
      if (u - group >= units) continue;  // the same for the whole workgroup
      const int w = head[k] >= a.heads[0];
      float v[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = value<DT>(r0[k], i);
        v[8 + i] = value<DT>(r1[k], i);
      }
      if (w ? a.weight[1] : a.weight[0]) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x0 = ANY && i < skip0 ? 0.0f : v[i], x1 = ANY && i < skip1 ? 0.0f : v[8 + i];
          s = __fmaf_rn(x0, x0, s);
          s = __fmaf_rn(x1, x1, s);
        }
        const float rstd = 1.0f / __fsqrt_rn(head_sum(s, log) * inv_d + a.eps);
        if (live) {
          const float* const f = weights + w * a.D;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (!ANY || i < n0) v[i] *= rstd * f[at0 + i];
            if (!ANY || i < n1) v[8 + i] *= rstd * f[at1 + i];
          }
        }
      }
      if (u >= units || !live) continue;
      if (turns_here) {
        const float2* const cs = turns + tok[k] * pairs + p0;
        if (half) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 t = !ANY || i < n0 ? cs[i] : float2{1.0f, 0.0f};
            const float x = v[i], y = v[8 + i];
            v[i] = x * t.x - y * t.y;
            v[8 + i] = x * t.y + y * t.x;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 t = !ANY || i < pairs ? cs[i] : float2{1.0f, 0.0f};
            const float x = v[2 * i], y = v[2 * i + 1];
            v[2 * i] = x * t.x - y * t.y;
            v[2 * i + 1] = x * t.y + y * t.x;
          }
        }
      }
      const int h = w ? head[k] - a.heads[0] : head[k];
      uint8_t* const o = static_cast<uint8_t*>(w ? a.out[1] : a.out[0]) +
                         (((batch * a.S + s0 + tok[k]) * (w ? a.heads[1] : a.heads[0]) + h) * (int64_t)a.D) * ES;
      store_piece<DT, ANY>(o + at0 * ES, n0, packed<DT>(v));
      if (!ANY || n1 > 0) store_piece<DT, ANY>(o + at1 * ES, n1, packed<DT>(v + 8));
    }
  }
}

// Whether every piece starts on 16 bytes and is whole.
bool aligned(const Args& a, int es) {
  bool ok = a.rot % 16 == 0 && (a.D - a.rot) % 16 == 0;
  for (int w = 0; w < 2; ++w) {
    if (a.heads[w] == 0) continue;
    auto on16 = [&](int64_t stride) { return stride * es % 16 == 0; };
    ok = ok && reinterpret_cast<uintptr_t>(a.x[w]) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out[w]) % 16 == 0 &&
         on16(a.stride_b[w]) && on16(a.stride_s[w]) && on16(a.stride_h[w]);
  }
  return ok;
}

template <int DT>
int launch_type(const Args& a, hipStream_t stream) {
  constexpr int ES = DT == CDIT_DT_F32 ? 4 : 2;
  const int cus = cu_count();
  if (cus <= 0) {
    set_error("cannot query the CU count of the current device");
    return CDIT_EHIP;
  }
  const int pairs = a.rot / 2, lanes = std::max(1, (pairs + 7) / 8 + (a.D - a.rot + 15) / 16);
  int log = 0;
  while ((1 << log) < lanes) ++log;
  const int groups = kThreads >> log, all = a.heads[0] + a.heads[1];
  // Two rounds of kUnits heads for each group of lanes (us of the two sizes at kUnits: one round 39 and 238, four 37 and 264), where
  // that leaves enough workgroups; else fewer, down to one head.
  int64_t tokens = std::min<int64_t>(std::max<int64_t>(2 * kUnits * groups / all, 1), kMostTokens);
  tokens = std::max<int64_t>(1, std::min(tokens, a.B * a.S / (2 * cus)));
  int heads = all;
  while (heads > groups && a.B * a.S * ((all + heads - 1) / heads) < 2 * cus) heads = std::max(groups, (heads + 1) / 2);
  const int64_t tiles = (a.S + tokens - 1) / tokens;
  if (tiles * a.B > UINT32_MAX / kThreads) {
    set_error("cdit_rotary: %lld sequences of %lld tokens are more workgroups than a launch has", (long long)a.B, (long long)a.S);
    return CDIT_EINVAL;
  }
  const dim3 grid((unsigned)(tiles * a.B), (unsigned)((all + heads - 1) / heads));
  const size_t lds = (2 * tokens * pairs + 2 * a.D) * sizeof(float);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, stream, a, (int)tokens, heads, (int)tiles, log);
    return 0;
  };
  return aligned(a, ES) ? launch(rotary_heads<DT, false>) : launch(rotary_heads<DT, true>);
}

}  // namespace

int launch_rotary(const cdit_rotary_args& args, hipStream_t stream) {
  cdit_rotary_args a = args;
  if (a.S == 1) {  // one token of each of many sequences: a sequence of tokens with positions of their own
    a.S = a.B;
    a.B = 1;
    for (int w = 0; w < 2; ++w) a.stride_s[w] = a.stride_b[w];
    a.position_stride_s = a.position_stride_b;
    a.table_stride_s = a.table_stride_b;
  }
  if (a.dtype == CDIT_DT_F32) return launch_type<CDIT_DT_F32>(a, stream);
  if (a.dtype == CDIT_DT_BF16) return launch_type<CDIT_DT_BF16>(a, stream);
  return launch_type<CDIT_DT_F16>(a, stream);
}

}  // namespace cdit
