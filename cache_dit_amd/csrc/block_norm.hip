// What stands between two branches of a transformer block (include/cdit_hip.h, cdit_gate_residual_norm): the
// branch's own norm, its gate, the residual sum, the next norm and its modulation in one pass, and the MXFP4 codes
// of the result where a 4-bit Linear reads it. Bound by HBM: x and the branch are read once, h and y written once.
//
//   t = branch                      or  w_post * branch / sqrt(mean(branch^2) + eps)   (or LayerNorm of it)
//   h = r x + gate t
//   y = norm(h) [* w] [* (1 + scale)] [+ shift]
//
// All in fp32 from the loads to the two roundings at the end: h is rounded to the stream's type where it is stored,
// and y is computed from the unrounded h, so that a 16-bit stream costs the norm nothing.
#include "gemm_common.h"
#include "mxfp4_device.h"
#include "quant_device.h"

namespace cdit {
namespace {

typedef cdit_gate_residual_norm_args Args;

template <int DT>
__device__ __forceinline__ void widen8(const Mx8<DT>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == CDIT_DT_F32) {
      f[i] = __uint_as_float(v.w[i]);
    } else if constexpr (DT == CDIT_DT_BF16) {
      f[i] = i & 1 ? bf16_hi(v.w[i / 2]) : bf16_lo(v.w[i / 2]);
    } else {
      f[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(v.w[i / 2] >> (16 * (i & 1))));
    }
  }
}
template <int DT>
__device__ __forceinline__ Mx8<DT> narrow8(const float (&f)[8]) {
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
template <int DT>
__host__ __device__ constexpr int size_of() {
  return DT == CDIT_DT_F32 ? 4 : 2;
}

// n <= 8 elements at p, the others zero.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int n, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = 0.0f;
    if (i >= n) continue;
    if constexpr (DT == CDIT_DT_F32) {
      f[i] = static_cast<const float*>(p)[i];
    } else if constexpr (DT == CDIT_DT_BF16) {
      f[i] = __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
    } else {
      f[i] = (float)static_cast<const _Float16*>(p)[i];
    }
  }
}
template <int DT>
__device__ __forceinline__ void store8(void* p, int n, const float (&f)[8]) {
  const Mx8<DT> v = narrow8<DT>(f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= n) continue;
    if constexpr (DT == CDIT_DT_F32) {
      static_cast<uint32_t*>(p)[i] = v.w[i];
    } else {
      static_cast<uint16_t*>(p)[i] = (uint16_t)(v.w[i / 2] >> (16 * (i & 1)));
    }
  }
}

// Sums over a workgroup of WAVES wavefronts, in an order of their own that does not change from call to call.
template <int WAVES>
struct BlockSum {
  float (*slot)[WAVES];  // two sets in turn: a set is read by all before the one after next is written
  int turn;
  __device__ __forceinline__ float operator()(float v) {
    v = wave_sum_f32(v);
    if constexpr (WAVES > 1) {
      float* const s = slot[turn];
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
      __syncthreads();
      v = s[0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) v += s[w];
    }
    return v;
  }
};

// The codes of a piece c of y as it is (or would be) stored. K is a multiple of 32: the quad of lanes that holds a block is in the
// row, and here, as a whole.
template <int DT>
__device__ __forceinline__ void put_codes(const Args& a, int64_t row, int c, const Mx8<DT>& v) {
  const int e = mx_exponent(mx_quad_max(mx_amax8<DT>(v)));
  *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.codes) + row * a.ld_codes + 4 * c) = mx_codes8<DT>(v, e);
  if (c % 4 == 0) {
    uint8_t* const s = static_cast<uint8_t*>(a.code_scales) + row * a.ld_code_scales;
    const int b = c / 4, blocks = (int)a.K / kMxBlock;
    s[b] = (uint8_t)e;
    if (b == blocks - 1)
      for (int pad = blocks; pad % 4 != 0; ++pad) s[pad] = (uint8_t)kMxPad;
  }
}

// A piece of 8 columns of the row: where it is, and what of it exists.
template <int ST, int DT>
struct Row {
  const Args& a;
  int64_t row;
  __device__ __forceinline__ int n_of(int c) const { return min(max((int)a.K - 8 * c, 0), 8); }
  __device__ __forceinline__ void vec(const void* p, int64_t ld, int64_t rows_per, int c, float (&f)[8]) const {
    const int64_t at = (rows_per > 0 ? row / rows_per * ld : 0) + 8 * c;
    if (a.vec_f32)
      load8<CDIT_DT_F32>(static_cast<const float*>(p) + at, n_of(c), f);
    else
      load8<DT>(static_cast<const uint8_t*>(p) + at * size_of<DT>(), n_of(c), f);
  }
  __device__ __forceinline__ void branch(int c, float (&t)[8]) const {
    load8<DT>(static_cast<const uint8_t*>(a.branch) + (row * a.ld_branch + 8 * c) * size_of<DT>(), n_of(c), t);
  }
  // t -> post norm of t; mean and rstd of the branch's row
  __device__ __forceinline__ void post(int c, float mean, float rstd, float (&t)[8]) const {
    float w[8];
    if (a.post_weight) vec(a.post_weight, 0, 0, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (t[i] - mean) * rstd * (a.post_weight ? w[i] : 1.0f);
  }
  __device__ __forceinline__ void stream(int c, float (&x)[8]) const {
    load8<ST>(static_cast<const uint8_t*>(a.x) + (row * a.ld_x + 8 * c) * size_of<ST>(), n_of(c), x);
  }
  // t, x -> h
  __device__ __forceinline__ void residual(int c, const float (&x)[8], float (&t)[8]) const {
    float g[8];
    if (a.gate) vec(a.gate, a.ld_gate, a.rows_per_gate, c, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = __fmaf_rn(a.gate ? g[i] : 1.0f, t[i], a.residual_scale * x[i]);
  }
  // h -> h stored; h -> y stored, or its codes
  __device__ __forceinline__ void finish(int c, float mean, float rstd, const float (&h)[8]) const {
    const int n = n_of(c);
    float y[8], f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (h[i] - mean) * rstd;
    if (a.norm_weight) {
      vec(a.norm_weight, 0, 0, c, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= f[i];
    }
    if (a.scale) {
      vec(a.scale, a.ld_scale, a.rows_per_scale, c, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __fmaf_rn(y[i], f[i], y[i]);
    }
    if (a.shift) {
      vec(a.shift, a.ld_shift, a.rows_per_shift, c, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += f[i];
    }
    store8<ST>(static_cast<uint8_t*>(a.h) + (row * a.ld_h + 8 * c) * size_of<ST>(), n, h);
    if (a.y) store8<DT>(static_cast<uint8_t*>(a.y) + (row * a.ld_y + 8 * c) * size_of<DT>(), n, y);
    if (a.codes) {
      const Mx8<DT> v = narrow8<DT>(y);
      if (n > 0) put_codes<DT>(a, row, c, v);
    }
  }
};

// Mean (0 for RMS) and 1 / sqrt(variance or mean square + eps) of a row; `piece(c, f)` gives its pieces. The squares
// are those of the values less the mean: no cancellation, whatever the row's offset.
template <class Piece, class Sum>
__device__ __forceinline__ void statistics(const Args& a, bool layer, Sum& sum, int first, int step, int pieces, Piece piece,
                                           float* mean, float* rstd) {
  const float inv_k = 1.0f / (float)a.K;
  float s = 0.0f;
  *mean = 0.0f;
  if (layer) {
    for (int c = first; c < pieces; c += step) {
      float f[8];
      piece(c, f);
      const int n = min((int)a.K - 8 * c, 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += i < n ? f[i] : 0.0f;
    }
    *mean = sum(s) * inv_k;
    s = 0.0f;
  }
  for (int c = first; c < pieces; c += step) {
    float f[8];
    piece(c, f);
    const int n = min((int)a.K - 8 * c, 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = i < n ? f[i] - *mean : 0.0f;
      s = __fmaf_rn(d, d, s);
    }
  }
  *rstd = 1.0f / __fsqrt_rn(sum(s) * inv_k + a.eps);
}

// A workgroup per row, the row read again in each pass, value by value: rows of less than 8 values, or of more than 16384. us, 4096 x
// 20000: bf16 1009 (0.65 TB/s), with an fp32 stream 1233 (0.8).
template <int ST, int DT>
__global__ __launch_bounds__(256) void gate_residual_norm_any(Args a) {
  __shared__ float slots[2][4];
  BlockSum<4> sum{slots, 0};
  const int pieces = (int)((a.K + 7) / 8);
  // (whole quads of lanes take part in a block's maximum, also behind the last piece)
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const Row<ST, DT> r{a, row};
    float pm = 0.0f, pr = 1.0f, mean, rstd;
    if (a.post_norm)
      statistics(a, a.post_norm == CDIT_NORM_LAYER, sum, threadIdx.x, 256, pieces,
                 [&](int c, float(&f)[8]) { r.branch(c, f); }, &pm, &pr);
    auto h_of = [&](int c, float(&f)[8]) {
      r.branch(c, f);
      if (a.post_norm) r.post(c, pm, pr, f);
      float x[8];
      r.stream(c, x);
      r.residual(c, x, f);
    };
    statistics(a, a.norm == CDIT_NORM_LAYER, sum, threadIdx.x, 256, pieces, h_of, &mean, &rstd);
    for (int c = threadIdx.x; c < pieces; c += 256) {
      float h[8];
      h_of(c, h);
      r.finish(c, mean, rstd, h);
    }
  }
}

// The row in registers: CH pieces per lane, WAVES wavefronts per row, 16-byte accesses. A workgroup takes a run of consecutive
// rows; the next row's loads are under way while a row is worked on, and the vectors, folded into one factor of the branch and a
// factor and an addend of the result, stay in registers until a row takes others (with one piece a lane; with two each row reads
// them again from the caches). us, 32760 x 5120, fp32 stream, one set of vectors: 604 with the vectors read for each row, 406 so
// (4.95 TB/s; a copy of 1 GiB runs at 5.1).
//
// Rows above 8192, two pieces a lane, spill nonetheless: the 128 registers of 16 wavefronts do not hold a row's h beside the next
// row's loads (16 to 18 registers to scratch with 16-bit streams, 46 to 60 with fp32 ones), nor do the 168 of 12 with an fp32 stream
// (6 to 14). us, bf16, and with an fp32 stream: 4096 x 8192 54 (4.96 TB/s) and 81 (4.98), x 12288 90 (4.5) and 145 (4.2), x 15360 112
// (4.5) and 200 (3.8); unaligned, bf16, x 8192 52, x 15360 138.
//
// ANY: rows of any length from 8 on, wherever they start. The last piece ends with the row and begins with values of the piece
// before it: these count once, and are stored twice, alike. us, bf16: 8192 x 5121 83 (5120: 70), 420 with the kernel above; 20000 x 71
// 13 and 98.
//
// ONCE: the 16-bit ones of x, branch and h are read and written non-temporally: they leave the caches to y or its codes, which the
// next kernel reads. bf16, us, without and with: 8192 x 4096 with vectors per token 109 and 85 (5.5 TB/s), 4096 x 15360 126 and 114,
// 32760 x 5120 291 and 290; below kOnceBytes, where the caches hold all of it, 2 x 4096 x 2560 36 and 42.
constexpr int64_t kOnceBytes = (int64_t)64 << 20;
template <int ST, int DT, int WAVES, int CH, bool ONCE, bool ANY>
__global__ __launch_bounds__(64 * WAVES) void gate_residual_norm_rows(Args a, int rows_per_wg) {
  __shared__ float slots[2][WAVES];
  BlockSum<WAVES> sum{slots, 0};
  const int64_t row0 = (int64_t)blockIdx.x * rows_per_wg, row_end = min(a.M, row0 + rows_per_wg);
  if (row0 >= row_end) return;
  const float inv_k = 1.0f / (float)a.K;
  const bool post_layer = a.post_norm == CDIT_NORM_LAYER, layer = a.norm == CDIT_NORM_LAYER;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int col[CH], skip[CH];  // first column of a piece, and how many of its values are the piece's before as well (ANY)
  bool in[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    col[c] = 8 * ((c * WAVES + wave) * 64 + lane);
    in[c] = col[c] < a.K;
    skip[c] = 0;
    if (ANY && in[c]) {
      skip[c] = max(col[c] - ((int)a.K - 8), 0);
      col[c] -= skip[c];
    }
  }
  auto fetch = [&](int64_t row, Mx8<DT>(&bb)[CH], Mx8<ST>(&xx)[CH]) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      bb[c] = {};
      xx[c] = {};
      if (in[c]) {
        bb[c] = mx_load8<DT, (ONCE && DT != CDIT_DT_F32), ANY>(static_cast<const uint8_t*>(a.branch) +
                                                               (row * a.ld_branch + col[c]) * size_of<DT>());
        xx[c] = mx_load8<ST, (ONCE && ST != CDIT_DT_F32), ANY>(static_cast<const uint8_t*>(a.x) +
                                                               (row * a.ld_x + col[c]) * size_of<ST>());
      }
    }
  };
  // gate * post_weight; norm_weight * (1 + scale); shift
  constexpr bool KEEP = CH == 1;
  constexpr int KEPT = KEEP ? CH : 1;
  float vg[KEPT][8], vm[KEPT][8], vs[KEPT][8];
  int64_t at_gate = -1, at_shift = -1, at_scale = -1;
  auto vector = [&](const void* p, int64_t at, int c, float(&f)[8]) {
    if (a.vec_f32) {
      Mx8<CDIT_DT_F32> v = {};
      if (in[c]) v = mx_load8<CDIT_DT_F32, false, ANY>(static_cast<const float*>(p) + at + col[c]);
      widen8<CDIT_DT_F32>(v, f);
    } else {
      Mx8<DT> v = {};
      if (in[c]) v = mx_load8<DT, false, ANY>(static_cast<const uint8_t*>(p) + (at + col[c]) * size_of<DT>());
      widen8<DT>(v, f);
    }
  };
  auto branch_factor = [&](int c, float(&f)[8]) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 1.0f;
    if (a.gate) vector(a.gate, at_gate * a.ld_gate, c, f);
    if (a.post_weight) {
      vector(a.post_weight, 0, c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= w[i];
    }
  };
  auto result_factor = [&](int c, float(&f)[8]) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 1.0f;
    if (a.norm_weight) vector(a.norm_weight, 0, c, f);
    if (a.scale) {
      vector(a.scale, at_scale * a.ld_scale, c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __fmaf_rn(f[i], w[i], f[i]);
    }
  };
  auto result_addend = [&](int c, float(&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.0f;
    if (a.shift) vector(a.shift, at_shift * a.ld_shift, c, f);
  };
  auto take_vectors = [&](int64_t row) {
    const int64_t ig = a.gate ? row / a.rows_per_gate : 0, ih = a.shift ? row / a.rows_per_shift : 0,
                  ic = a.scale ? row / a.rows_per_scale : 0;
    if (ig == at_gate && ih == at_shift && ic == at_scale) return;  // uniform
    at_gate = ig;
    at_shift = ih;
    at_scale = ic;
    if constexpr (KEEP) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        branch_factor(c, vg[c]);
        result_factor(c, vm[c]);
        result_addend(c, vs[c]);
      }
    }
  };
  // mean and 1 / sqrt(...) of the row whose pieces are f, as in statistics()
  auto stats = [&](const float(&f)[CH][8], bool centred, float* mean, float* rstd) {
    float s = 0.0f;
    *mean = 0.0f;
    if (centred) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += ANY && i < skip[c] ? 0.0f : f[c][i];  // (pieces behind the row are zeros)
      *mean = sum(s) * inv_k;
      s = 0.0f;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = in[c] && !(ANY && i < skip[c]) ? f[c][i] - *mean : 0.0f;
        s = __fmaf_rn(d, d, s);
      }
    *rstd = 1.0f / __fsqrt_rn(sum(s) * inv_k + a.eps);
  };
  auto one_row = [&](int64_t row, Mx8<DT>(&bb)[CH], Mx8<ST>(&xx)[CH], Mx8<DT>(&nb)[CH], Mx8<ST>(&nx)[CH]) {
    if (row + 1 < row_end) fetch(row + 1, nb, nx);
    take_vectors(row);
    float h[CH][8], mean = 0.0f, rstd = 1.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) widen8<DT>(bb[c], h[c]);
    if (a.post_norm) stats(h, post_layer, &mean, &rstd);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float x[8], f[8];
      widen8<ST>(xx[c], x);
      if constexpr (!KEEP) branch_factor(c, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float t = (h[c][i] - mean) * rstd;
        h[c][i] = in[c] ? __fmaf_rn(KEEP ? vg[KEEP ? c : 0][i] : f[i], t, a.residual_scale * x[i]) : 0.0f;
      }
    }
    stats(h, layer, &mean, &rstd);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (!in[c]) continue;
      float y[8], m[8], s[8];
      if constexpr (!KEEP) {
        result_factor(c, m);
        result_addend(c, s);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y[i] = __fmaf_rn((h[c][i] - mean) * rstd, KEEP ? vm[KEEP ? c : 0][i] : m[i], KEEP ? vs[KEEP ? c : 0][i] : s[i]);
      mx_store8<ST, (ONCE && ST != CDIT_DT_F32), ANY>(static_cast<uint8_t*>(a.h) + (row * a.ld_h + col[c]) * size_of<ST>(),
                                                 narrow8<ST>(h[c]));
      const Mx8<DT> v = narrow8<DT>(y);
      if (a.y) mx_store8<DT, false, ANY>(static_cast<uint8_t*>(a.y) + (row * a.ld_y + col[c]) * size_of<DT>(), v);
      if (a.codes) put_codes<DT>(a, row, col[c] / 8, v);
    }
  };
  Mx8<DT> b_raw[2][CH];
  Mx8<ST> x_raw[2][CH];
  fetch(row0, b_raw[0], x_raw[0]);
  for (int64_t row = row0; row < row_end; row += 2) {
    one_row(row, b_raw[0], x_raw[0], b_raw[1], x_raw[1]);
    if (row + 1 < row_end) one_row(row + 1, b_raw[1], x_raw[1], b_raw[0], x_raw[0]);
  }
}

// Whether every piece of 8 columns starts on 16 bytes.
template <int ST, int DT>
bool rows_aligned(const Args& a) {
  constexpr int SS = size_of<ST>(), DS = size_of<DT>();
  auto rows = [](const void* p, int64_t ld, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0;
  };
  const int vs = a.vec_f32 ? 4 : DS;
  auto vec = [&](const void* p, int64_t ld) { return !p || rows(p, ld, vs); };
  return a.K % 8 == 0 && rows(a.x, a.ld_x, SS) && rows(a.h, a.ld_h, SS) && rows(a.branch, a.ld_branch, DS) &&
         (!a.y || rows(a.y, a.ld_y, DS)) && vec(a.gate, a.ld_gate) && vec(a.shift, a.ld_shift) && vec(a.scale, a.ld_scale) &&
         vec(a.norm_weight, 0) && vec(a.post_weight, 0);
}

template <int ST, int DT>
int launch_types(const Args& a, hipStream_t stream) {
  if (a.K >= 8 && a.K <= 16384) {
    const int cus = cu_count();
    if (cus <= 0) {
      set_error("cannot query the CU count of the current device");
      return CDIT_EHIP;
    }
    const int pieces = (int)((a.K + 7) / 8);
    const bool once = DT != CDIT_DT_F32 && 2 * a.M * a.K >= kOnceBytes, aligned = rows_aligned<ST, DT>(a);
    auto launch = [&](auto kernel, int waves) {
      const int64_t target = (int64_t)cus * std::max(1, 24 / waves);
      const int per = (int)std::min<int64_t>((a.M + target - 1) / target, 1 << 20);
      hipLaunchKernelGGL(kernel, dim3((unsigned)((a.M + per - 1) / per)), dim3(64 * waves), 0, stream, a, per);
      return 0;
    };
    if (!aligned) {
#define CDIT_NORM_CASE(W, CH) \
  if (pieces <= 64 * W * CH) return launch(gate_residual_norm_rows<ST, DT, W, CH, false, true>, W);
      CDIT_NORM_CASE(1, 1)
      CDIT_NORM_CASE(2, 1)
      CDIT_NORM_CASE(4, 1)
      CDIT_NORM_CASE(8, 1)
      CDIT_NORM_CASE(12, 1)
      CDIT_NORM_CASE(16, 1)
      CDIT_NORM_CASE(16, 2)
#undef CDIT_NORM_CASE
    }
#define CDIT_NORM_CASE(W, CH)                                                                              \
  if (pieces <= 64 * W * CH) {                                                                             \
    if (once) return launch(gate_residual_norm_rows<ST, DT, W, CH, DT != CDIT_DT_F32, false>, W);          \
    return launch(gate_residual_norm_rows<ST, DT, W, CH, false, false>, W);                                \
  }
    CDIT_NORM_CASE(1, 1)
    CDIT_NORM_CASE(2, 1)
    CDIT_NORM_CASE(3, 1)
    CDIT_NORM_CASE(4, 1)
    CDIT_NORM_CASE(5, 1)
    CDIT_NORM_CASE(6, 1)
    CDIT_NORM_CASE(8, 1)
    CDIT_NORM_CASE(10, 1)
    CDIT_NORM_CASE(12, 1)
    CDIT_NORM_CASE(16, 1)
    CDIT_NORM_CASE(12, 2)
    CDIT_NORM_CASE(16, 2)
#undef CDIT_NORM_CASE
  }
  const dim3 grid((unsigned)std::min<int64_t>(a.M, 1 << 20));
  hipLaunchKernelGGL((gate_residual_norm_any<ST, DT>), grid, dim3(256), 0, stream, a);
  return 0;
}

}  // namespace

int launch_gate_residual_norm(const Args& a, hipStream_t stream) {
  if (a.dtype == CDIT_DT_F32) return launch_types<CDIT_DT_F32, CDIT_DT_F32>(a, stream);
  if (a.dtype == CDIT_DT_BF16)
    return a.x_dtype == CDIT_DT_F32 ? launch_types<CDIT_DT_F32, CDIT_DT_BF16>(a, stream)
                                    : launch_types<CDIT_DT_BF16, CDIT_DT_BF16>(a, stream);
  return a.x_dtype == CDIT_DT_F32 ? launch_types<CDIT_DT_F32, CDIT_DT_F16>(a, stream)
                                  : launch_types<CDIT_DT_F16, CDIT_DT_F16>(a, stream);
}

}  // namespace cdit
