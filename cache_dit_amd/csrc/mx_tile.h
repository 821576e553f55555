// What the tiles of the two 4-bit GEMMs share: both hold their outputs as blocks of 32 x 32 in the layout of the 32-row matrix
// instructions, a lane (r32 = lane & 31, h = lane >> 5) TN consecutive columns n .. n + TN - 1 of the rows 32 i + 8 (e >> 2) + 4 h
// + (e & 3).
#ifndef CDIT_MX_TILE_H_
#define CDIT_MX_TILE_H_

#include <algorithm>
#include <type_traits>

#include "gemm_common.h"

namespace cdit {
namespace {

// A tile and its measured times, ns: of a launch, and per tile on the fullest CU; of a step of 256 along K, for a CU's only
// tile and for each of several (which run on the CU together, or one after the other).
struct MxTime {
  int variant, bm, bn, start, tile, lone, step;
};
// The tile with the least time, or the kernel for few rows where it takes less. Tiles beyond whole rounds of the CUs count half a
// round and half their share of one: fewer CUs share the memory and the power then.
inline int fastest_tile(const MxTime* t, int count, bool weight_only, const Mx4Gemm& g, int cus) {
  const int64_t steps = (g.K + 255) / 256;
  int best = -1;
  int64_t best_ns = 0;
  if (mx_rows_can(g.M, g.ldb) && g.M > 16) {
    best = kMxRows;
    best_ns = mx_rows_ns(weight_only, g.M, g.N, g.K, cus);
  }
  for (int i = 0; i < count; ++i) {
    const int64_t tiles = (int64_t)((g.M + t[i].bm - 1) / t[i].bm) * ((g.N + t[i].bn - 1) / t[i].bn);
    const int64_t permille = tiles <= cus ? 1000 : rounds_permille(tiles, cus, 500, 500);
    const int64_t ns = t[i].start + t[i].tile * permille / 1000 + steps * std::max<int64_t>(t[i].lone, t[i].step * permille / 1000);
    if (best < 0 || ns < best_ns) {
      best = t[i].variant;
      best_ns = ns;
    }
  }
  return best;
}
// Offsets inside a tile are 32 bits; tiles are counted in 32 bits.
inline bool tiles_fit(const Mx4Gemm& g, int a_bytes) {
  const int64_t widest = std::max({g.lda * a_bytes, g.ldas, g.ldb, g.ldbs, 4 * g.ldo, (int64_t)g.K * 2});
  return widest * 256 < INT32_MAX && ((int64_t)g.M / 32 + 1) * ((int64_t)g.N / 64 + 1) < INT32_MAX;
}

// The bias of a lane's columns in fp32; 0 for columns that do not exist, and without a bias.
template <int TN, int OUT>
__device__ __forceinline__ void mx_bias(const Mx4Gemm& g, int n, float (&bias)[TN]) {
  constexpr int OB = OUT == CDIT_DT_F32 ? 4 : 2;
  const __amdgpu_buffer_rsrc_t buf =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(g.bias), 0, g.bias ? g.N * OB : 0, 0x00020000);
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    if constexpr (OUT == CDIT_DT_F32)
      bias[j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buf, (n + j) * OB, 0, 0));
    else
      bias[j] = bias_to_f32<OUT>((uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(buf, (n + j) * OB, 0, 0));
  }
}

// Stores a wavefront's blocks from the registers they are in: a lane's TN columns are one store, 32 lanes a whole row of the
// wavefront's tile. The tile's rows are m0 .. m0 + bm - 1, row: this lane's first inside it. Rows of any alignment are stored so
// (the hardware takes such stores: 1357 x 4463 x 2208 (M x N x K) in tiles of 128 x 128 21.0 us column by column, 18.7 so); a
// lane whose columns the end of a row cuts stores them one by one.
template <int TM, int TN, int OUT>
__device__ __forceinline__ void store_mx_tile(v16f (&acc)[TM][TN], const Mx4Gemm& g, int m0, int bm, int row, int n) {
  constexpr int OB = OUT == CDIT_DT_F32 ? 4 : 2;
  const int rows = min(bm, g.M - m0);
  const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
      static_cast<uint8_t*>(g.out) + (int64_t)m0 * g.ldo * OB, 0, ((rows - 1) * (int)g.ldo + g.N) * OB, 0x00020000);
  const uint32_t row_bytes = (uint32_t)g.ldo * OB;
  const uint32_t off = (uint32_t)row * row_bytes + (uint32_t)n * OB;
  const bool cut = g.N % TN != 0 && __builtin_amdgcn_readfirstlane(n) + 32 * TN > g.N;  // (a wavefront's first lane: its first column)
  constexpr int kStoreOnce = 2;  // non-temporal: whole lines, written once
  // The 256 x 256 tile has its sums in accumulation registers. Left to itself the compiler copies them to others ahead of the
  // stores, many of them several times, and spills for it: here each is read where it is stored. The wait covers the last
  // matrix instruction, which the compiler does not see these reads depend on. us, without and with: w4a4 32760 x 13824 x 5120
  // 1160 and 1080, 8192 x 10240 x 2560 134 and 118, with GELU (and its steps in order, below) 166 and 128; w4a16 16384 x 5120 x
  // 5120 630 and 592. The tiles of half the size keep theirs where the compiler puts them: 1230 either way.
  constexpr bool IN_AGPRS = TM * TN >= 16;
  if constexpr (IN_AGPRS) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  }
  auto store = [&](auto gelu_tag, auto cut_tag) {
    const int at = (int)(n + TN <= g.N ? off : 0x80000000u);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t at_row = (uint32_t)(32 * i + 8 * (e >> 2) + (e & 3)) * row_bytes;
        float v[TN], ex[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if constexpr (IN_AGPRS)
            asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[j]) : "a"(acc[i][j][e]));
          else
            v[j] = acc[i][j][e];
        }
        if constexpr (decltype(gelu_tag)::value) {
          // (step by step: one wavefront a SIMD, and nothing but the other columns covers the latency of a step)
#pragma unroll
          for (int j = 0; j < TN; ++j) ex[j] = gelu_exp(v[j]);
          if constexpr (IN_AGPRS) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < TN; ++j) v[j] *= __builtin_amdgcn_rcpf(1.0f + ex[j]);
          if constexpr (IN_AGPRS) __builtin_amdgcn_sched_barrier(0);
        }
        auto pack = [](float lo, float hi) -> uint32_t {
          return OUT == CDIT_DT_F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
        };
        uint32_t w[TN];  // fp32, or pairs
#pragma unroll
        for (int j = 0; j < TN; ++j)
          w[j] = OUT == CDIT_DT_F32 ? __float_as_uint(v[j]) : j % 2 == 0 ? pack(v[j], j + 1 < TN ? v[j + 1 < TN ? j + 1 : 0] : 0.0f) : 0u;
        if constexpr (TN * OB == 16) {
          const v4u d = {w[0], w[1], w[2], w[TN - 1]};
          __builtin_amdgcn_raw_buffer_store_b128(d, out, at, at_row, kStoreOnce);
        } else if constexpr (TN * OB == 8) {
          const v2u d = {w[0], w[TN == 4 ? 2 : 1]};
          __builtin_amdgcn_raw_buffer_store_b64(d, out, at, at_row, kStoreOnce);
        } else if constexpr (TN * OB == 4) {
          const uint32_t d = w[0];
          __builtin_amdgcn_raw_buffer_store_b32(d, out, at, at_row, kStoreOnce);
        } else {
          const short d = (short)w[0];
          __builtin_amdgcn_raw_buffer_store_b16(d, out, at, at_row, kStoreOnce);
        }
        if constexpr (decltype(cut_tag)::value) {
#pragma unroll
          for (int j = 0; j < TN - 1; ++j) {
            const int one = (int)(n + TN > g.N && n + j < g.N ? off + j * OB : 0x80000000u);
            if constexpr (OUT == CDIT_DT_F32) {
              const uint32_t d = w[j];
              __builtin_amdgcn_raw_buffer_store_b32(d, out, one, at_row, 0);
            } else {
              const short d = (short)(w[j & ~1] >> (16 * (j & 1)));
              __builtin_amdgcn_raw_buffer_store_b16(d, out, one, at_row, 0);
            }
          }
        }
      }
  };
  // (a branch around all of the stores, not one in each of them)
  auto store_cut = [&](auto gelu_tag) {
    if constexpr (TN > 1) {
      if (cut) return store(gelu_tag, std::true_type{});
    }
    store(gelu_tag, std::false_type{});
  };
  if (g.epilogue & CDIT_EPI_GELU_TANH)
    store_cut(std::true_type{});
  else
    store_cut(std::false_type{});
}

}  // namespace
}  // namespace cdit
#endif
