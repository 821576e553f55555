// The 4-bit Linears for few rows (single tokens, conditioning vectors): a stream of weights.
//
// A workgroup takes 16 rows (or the less there are) and G times 16 output columns. The activation goes to LDS first (in pieces of K
// where it is long), and is quantized on the way where the caller has it in bf16. K is split between the W wavefronts in items of
// 512; a wavefront reads an item's weights straight from memory (every byte is used once, the next item's loads are under way meanwhile) and multiplies
// them with the activation's rows on the matrix core, and the W partial sums of 16 x 16 outputs meet in LDS. Bound by HBM, and
// by latency where N is small: 1 x 30720 x 5120 (M x N x K) 17.9 us for 84 MB, where a kernel that only reads them takes 14.8; 1 x
// 13824 x 5120 10.8 with the weight in the caches as far as it fits, 12.8 from HBM (8.2 to only read it).
//
// Lane l is row l & 15 (a column of the output; a row of the activation) and K block l >> 4 of a step of 128: 16 bytes of codes,
// 64 of each row in a request, and the scale in byte l >> 4 of the step's word. The scales go through LDS: 16 rows of them are
// a few KB in a row, fetched by the whole workgroup at once. (A word per lane and item straight from memory, whether 16
// bytes of each row or 256 in a row, held a loop of nothing but the loads to 4.1 TB/s where the codes alone ran at 5.2.)
#include <algorithm>

#include "gemm_common.h"
#include "mx_rows_plan.h"
#include "mxfp4_device.h"

namespace cdit {
namespace {

// Weight-only: bf16 activation. Codes: an activation in MXFP4. Quantize: a bf16 activation, quantized here.
enum Mode { kWeightOnly, kCodes, kQuantize };
constexpr int kMostRows = kMxRowsMost, kItem = kMxRowsItem;

template <int MODE, int OUT>
__global__ __launch_bounds__(64 * kMxRowsWaves) void gemm_mx_rows(Mx4Gemm g, int G, int chunk_items) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  {  // this workgroup's rows
    const int64_t m0 = kMostRows * (int64_t)blockIdx.y;
    g.a += m0 * g.lda * (MODE == kCodes ? 1 : 2);
    if (MODE == kCodes) g.a_scale += m0 * g.ldas;
    g.out = static_cast<uint8_t*>(g.out) + m0 * g.ldo * (OUT == CDIT_DT_F32 ? 4 : 2);
    g.M = min(g.M - (int)m0, kMostRows);
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, kg = lane >> 4;
  const int KB = g.K / kMxBlock, S = (g.K + 127) / 128 * 4, items = (g.K + kItem - 1) / kItem;
  const int pitch = mx_row_pitch(MODE == kWeightOnly, chunk_items), spitch = MODE == kWeightOnly ? 0 : mx_scale_pitch(chunk_items);
  float* const part = reinterpret_cast<float*>(smem);  // [G][waves][256]
  uint8_t* const wscale = smem + G * waves * 1024;  // [16 G][wpitch]
  const int wpitch = mx_scale_pitch(chunk_items);
  uint8_t* const xs = wscale + 16 * G * wpitch;
  uint8_t* const xe = xs + g.M * pitch;
  const int m = min(r, g.M - 1);  // (rows that do not exist repeat the last: their results are not stored)

  struct Weights {
    v4u c[4];
  };
  // (buffer accesses: what lies behind K, and rows behind the last, read as zeros without a branch around the load)
  auto load = [&](int group, int item, Weights& w) {
    const int n0 = 16 * (blockIdx.x * G + group), rows = min(g.N - n0, 16);
    const __amdgpu_buffer_rsrc_t codes = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(g.b + (int64_t)n0 * g.ldb), 0, rows > 0 ? (rows - 1) * (int)g.ldb + g.K / 2 : 0, 0x00020000);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int block = 16 * item + 4 * s + kg;
      const int at = (int)(block < KB ? (uint32_t)r * (uint32_t)g.ldb + 16u * block : 0x80000000u);
      w.c[s] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(codes, at, 0, 0));
    }
  };
  auto multiply = [&](const Weights& w, int group, int in_chunk, v4f (&acc)[2]) {
    const uint8_t* const ws = wscale + (16 * group + r) * wpitch + 16 * in_chunk + kg;
    const uint8_t* const x = xs + m * pitch + in_chunk * (MODE == kWeightOnly ? 1024 : 256) + kg * (MODE == kWeightOnly ? 64 : 16);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int e = ws[4 * s];
      if constexpr (MODE == kWeightOnly) {
        const float f = mx_scale_or_nan(e);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[q & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_to_bf16(w.c[s][q], f),
                                                               *reinterpret_cast<const v8bf*>(x + 256 * s + 16 * q), acc[q & 1], 0, 0, 0);
      } else {
        const v4i c = __builtin_bit_cast(v4i, w.c[s]), a = *reinterpret_cast<const v4i*>(x + 64 * s);
        const v8i w8 = __builtin_shufflevector(c, c, 0, 1, 2, 3, -1, -1, -1, -1);
        const v8i x8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
        const int xe_s = xe[m * spitch + 16 * in_chunk + 4 * s + kg];
        acc[s & 1] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc[s & 1], 4, 4, 0, e, 0, xe_s);
      }
    }
  };

  for (int i = threadIdx.x; i < G * waves * 256; i += blockDim.x) part[i] = 0.0f;
  for (int first = 0; first < items; first += chunk_items) {
    const int n_items = min(chunk_items, items - first), per = (n_items + waves - 1) / waves;
    // this wavefront's items of the chunk, for each group of columns; the first two items' weights go out before the activation
    const int mine = min(max(n_items - wave * per, 0), per), i0 = first + wave * per;
    Weights w[2];
    int lg = 0, li = 0;  // group and item to load next
    auto load_next = [&](Weights& into) {
      if (lg >= G || mine <= 0) return;
      load(lg, i0 + li, into);
      if (++li == mine) {
        li = 0;
        ++lg;
      }
    };
    // Blocks of the activation and words of the weight's scales, a thread's first of each before the weights: a wait for a load
    // is a wait for all before it.
    struct Block {
      Mx8<CDIT_DT_BF16> v[4];  // (codes: v[0], and the scale)
      int e;
    };
    const int n_blocks = 16 * n_items, n_words = 4 * n_items;
    auto fetch_block = [&](int t) -> Block {
      Block x = {};
      const int row = t / n_blocks, block = 16 * first + t - row * n_blocks;
      x.e = kMxPad;
      if (block >= KB) return x;
      if constexpr (MODE == kCodes) {
        x.v[0] = mx_load8<CDIT_DT_BF16>(g.a + (int64_t)row * g.lda + 16 * block);
        x.e = g.a_scale[(int64_t)row * g.ldas + block];
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) x.v[q] = mx_load8<CDIT_DT_BF16>(g.a + 2 * ((int64_t)row * g.lda + 32 * block + 8 * q));
      }
      return x;
    };
    auto put_block = [&](int t, const Block& x) {
      const int row = t / n_blocks, b = t - row * n_blocks;
      if constexpr (MODE == kWeightOnly) {
#pragma unroll
        for (int q = 0; q < 4; ++q) mx_store8<CDIT_DT_BF16>(xs + row * pitch + 64 * b + 16 * q, x.v[q]);
      } else if constexpr (MODE == kCodes) {
        mx_store8<CDIT_DT_BF16>(xs + row * pitch + 16 * b, x.v[0]);
        xe[row * spitch + b] = (uint8_t)x.e;
      } else {
        uint32_t top = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) top = max(top, mx_amax8<CDIT_DT_BF16>(x.v[q]));
        const int e = mx_exponent(top);
        v4u c;
#pragma unroll
        for (int q = 0; q < 4; ++q) c[q] = mx_codes8<CDIT_DT_BF16>(x.v[q], e);
        *reinterpret_cast<v4u*>(xs + row * pitch + 16 * b) = c;
        xe[row * spitch + b] = (uint8_t)e;
      }
    };
    auto fetch_word = [&](int t) -> uint32_t {  // words behind a row's last: the scales of zeros
      const int row = t / n_words, word = t - row * n_words, at = 16 * first + 4 * word;
      const int64_t n = min(16 * (int)blockIdx.x * G + row, g.N - 1);
      return at < S ? *reinterpret_cast<const uint32_t*>(g.b_scale + n * g.ldbs + at) : 0x7f7f7f7fu;
    };
    auto put_word = [&](int t, uint32_t v) {
      const int row = t / n_words;
      *reinterpret_cast<uint32_t*>(wscale + row * wpitch + 4 * (t - row * n_words)) = v;
    };
    const int blocks = g.M * n_blocks, words = 16 * G * n_words, t0 = threadIdx.x;
    Block x0 = {};
    uint32_t v0 = 0;
    if (t0 < blocks) x0 = fetch_block(t0);
    if (t0 < words) v0 = fetch_word(t0);
    load_next(w[0]);
    load_next(w[1]);
    if (first > 0) __syncthreads();  // the piece before has been read
    if (t0 < blocks) put_block(t0, x0);
    if (t0 < words) put_word(t0, v0);
    for (int t = t0 + blockDim.x; t < blocks; t += blockDim.x) put_block(t, fetch_block(t));
    for (int t = t0 + blockDim.x; t < words; t += blockDim.x) put_word(t, fetch_word(t));
    __syncthreads();
    v4f acc[2] = {};
    int group = 0, i = 0;  // of the item at hand
    auto one_item = [&](Weights& now) {
      const bool last = i + 1 == mine;
      multiply(now, group, i0 + i - first, acc);
      load_next(now);
      if (last) {  // (a lane's own place: what an earlier piece of K left there is its own)
        v4f* const p = reinterpret_cast<v4f*>(part + (group * waves + wave) * 256 + 4 * lane);
        *p = *p + (acc[0] + acc[1]);
        acc[0] = acc[1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        ++group;
        i = 0;
      } else {
        ++i;
      }
    };
    if (mine > 0) {
      while (true) {
        one_item(w[0]);
        if (group == G) break;
        one_item(w[1]);
        if (group == G) break;
      }
    }
  }
  __syncthreads();
  // element e of lane l: column 4 (l >> 4) + e, row l & 15
  for (int t = threadIdx.x; t < G * 16 * g.M; t += blockDim.x) {
    const int c = t % (16 * G), row = t / (16 * G), n = 16 * blockIdx.x * G + c;
    if (n >= g.N) continue;
    const float* const p = part + (c >> 4) * waves * 256 + 4 * (16 * ((c & 15) >> 2) + row) + (c & 3);
    float v = 0.0f;
    for (int k = 0; k < waves; ++k) v += p[256 * k];
    store_mx_one<OUT>(g, row, n, v);
  }
}

template <int MODE, int OUT>
int launch_rows(const Mx4Gemm& g, hipStream_t stream) {
  static bool lds_allowed[64];
  const int cus = cu_count();
  if (cus <= 0) {
    set_error("cannot query the CU count of the current device");
    return CDIT_EHIP;
  }
  const MxRowsPlan p = mx_rows_plan(MODE == kWeightOnly, g.M, g.N, g.K, cus);
  const int groups = (g.N + 15) / 16, blocks = (g.M + kMostRows - 1) / kMostRows;
  if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&gemm_mx_rows<MODE, OUT>), 160 * 1024, lds_allowed)) return rc;
  hipLaunchKernelGGL((gemm_mx_rows<MODE, OUT>), dim3((unsigned)((groups + p.groups - 1) / p.groups), (unsigned)blocks),
                     dim3(64 * p.waves), p.lds, stream, g, p.groups, p.chunk);
  return 0;
}
template <int MODE>
int launch_rows(const Mx4Gemm& g, hipStream_t stream) {
  switch (g.out_dtype) {
    case CDIT_DT_F16: return launch_rows<MODE, CDIT_DT_F16>(g, stream);
    case CDIT_DT_F32: return launch_rows<MODE, CDIT_DT_F32>(g, stream);
    default: return launch_rows<MODE, CDIT_DT_BF16>(g, stream);
  }
}

}  // namespace

// Whether this is the kernel for up to 16 rows and so many columns, and not a tile. Every workgroup handles the whole activation, so
// its time grows with rows times columns; us, this kernel and the best tile (w4a4 with its quantizer), M x N x K, weights from HBM:
// w4a4 4 x 13824 x 5120 14.9 and 18.1, 8: 17.1 and 18.5, 16: 21.2 and 18.2; 16 x 5120 x 5120 14.0 and 14.8; 16 x 30720 x 5120 38.8
// and 25.5. Weight-only 8 x 13824 x 5120 17.9 and 24.4, 16: 23.7 and 25.1; 16 x 30720 x 5120 45.9 and 32.4.
bool mx_rows_fit(bool weight_only, int64_t M, int64_t N, int64_t ldb) {
  return mx_rows_can(M, ldb) && M <= 16 && M * ((N + 15) / 16) < (weight_only ? 20000 : 10000);
}
// Its time for more than 16 rows, ns, next to the tiles': a workgroup per 16 x 16 outputs reads little for each of its steps along K
// and so is done first where the tiles leave CUs idle. us, this kernel and the best tile, M x N x K: w4a4 294 x 16 x 9248 8.9 and
// 13.8, 502 x 128 x 5856 7.0 and 10.0, 32 x 1024 x 15360 14.8 and 20.4, 17 x 5120 x 5120 10.5 and 9.4; w4a16 19.6 and 24.1, 16.8
// and 21.0, 30.0 and 53.2, 18.4 and 19.1.
int64_t mx_rows_ns(bool weight_only, int64_t M, int64_t N, int64_t K, int64_t cus) {
  const int64_t items = (K + kItem - 1) / kItem, blocks = (M + kMostRows - 1) / kMostRows * ((N + 15) / 16);
  return 4000 + (weight_only ? 870 : 270) * items + std::max<int64_t>(blocks - cus, 0) * items * (weight_only ? 240 : 115) / 100;
}
// Whether it can take them: 16 rows of the weight within 32-bit offsets.
bool mx_rows_can(int64_t M, int64_t ldb) { return M >= 1 && M <= 65535 * kMostRows && ldb < (int64_t)1 << 27; }

int launch_gemm_mxfp4_rows(const Mx4Gemm& g, hipStream_t stream) { return launch_rows<kCodes>(g, stream); }
int launch_linear_mxfp4_rows(const Mx4Gemm& g, hipStream_t stream) { return launch_rows<kQuantize, CDIT_DT_BF16>(g, stream); }
int launch_gemm_w4a16_rows(const Mx4Gemm& g, hipStream_t stream) { return launch_rows<kWeightOnly, CDIT_DT_BF16>(g, stream); }

}  // namespace cdit
