// MXFP4 x MXFP4 GEMM (w4a4): out = epi(A W^T + bias) on codes of 4 bits with a scale per 32 of them along K.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands in this format: lane l holds the 32 codes (16 bytes) of
// row l & 15, K block l >> 4 of a step of 128, and the scale of that block in a byte of its own.
#include <algorithm>
#include <type_traits>

#include "gemm_common.h"
#include "mx_tile.h"
#include "mxfp4_device.h"

namespace cdit {
namespace {

__device__ __forceinline__ v4f mfma_mx(v4i w, v4i a, v4f acc, int w_scale, int a_scale) {
  const v8i w8 = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const v8i a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a8, acc, 4, 4, 0, w_scale, 0, a_scale);
}

// A wavefront per 32 x 32 outputs, operands straight from memory: any stride (the tiles below address with 32 bits).
template <int OUT>
__global__ __launch_bounds__(256) void gemm_mxfp4_direct(Mx4Gemm g) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kg = lane >> 4;
  const int n0 = blockIdx.x * 128 + wave * 32;
  if (n0 >= g.N) return;
  const int blocks = g.K / kMxBlock, steps = (g.K + 127) / 128;
  for (int m0 = blockIdx.y * 32; m0 < g.M; m0 += gridDim.y * 32) {
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
          if (m < g.M && n < g.N) store_mx_one<OUT>(g, m, n, acc[i][j][e]);
        }
  }
}

// ---------------------------------------------------------------------------
// Tiles through LDS, for more than a few rows. A workgroup of WGM x WGN wavefronts owns BM x BN outputs, a wavefront WM x WN
// of them as blocks of v_mfma_scale_f32_32x32x64_f8f6f4 (lane l: row l & 31, K block l >> 5 of 64). K advances in steps of 256:
// a 128-byte line of each panel row, four rounds of MFMAs. LDS-DMA fills rings of SA stages of A and SB of B.
//
//   round j = 0 .. 2 of step kt: MFMAs on fragments read before; meanwhile the fragments of round j + 1 are read
//   wait: own reads done, own DMA of step kt + 1 landed; barrier: so are everyone's, and the stages of step kt are free
//   round 3: MFMAs; meanwhile the first fragments of step kt + 1 are read; DMA of B's step kt + SB
//   rounds 0 and 1 of step kt + 1: DMA of A's step kt + SA
//
// A workgroup takes tiles blockIdx.x, blockIdx.x + gridDim.x, ... as one stream: the last steps of a tile fetch the first of the
// next, which land while the outputs are stored.
//
// LDS: a pass serves 16 lanes (lane bit 5 and the parity of bits 2..4 choose it); of the 8 chunks of 16 bytes of a panel row r, chunk
// c is stored at c ^ ((r >> 1) & 7), so that the lanes of a pass hit 16 different bank groups. The rows of B's panel are the
// columns n = TN p + j of a wavefront's tile at 32 j + p: a lane then holds TN consecutive columns of an output row, 32 lanes a
// whole row of the wavefront's tile, and the outputs are stored from the registers they are in.
//
// Scales: a lane needs bytes 2 j + (l >> 5) of its row for the rounds j = 0 .. 15 of 1024 along K. It loads 16 of those 32 bytes
// (those of its own half; a row's 32 are one request), and byte permutations and a swap between the halves of the
// wavefront bring them in order.
//
// Measured (M x N x K, weights and codes in HBM or caches as they come): 32760 x 13824 x 5120 in 256 x 256 tiles 1055 to 1080 us,
// 4.3 to 4.4 PFLOP/s, with GELU 1135, in fp32 (128 x 256 tiles) 1297; a loop of nothing but the instruction on random operands runs
// at 6.4 (the clock falls to 1.56 GHz), 725 us. Matrix cores busy 65 % of the cycles, no LDS conflicts. With a part left out: no
// scales after a tile's first 1050, no LDS-DMA after three steps 1110, no LDS reads 1045, no stores 1040, none of scales, DMA and
// reads 945 (of 1090): a wavefront a SIMD has nothing to cover a tile's end (2.8 us) and a step's changes with. Two a SIMD in tiles
// of 128 x 256 need 1.7 times the reads per product: 1225 us. Few tiles are bound by what a CU takes in, 50 to 60 GB/s: 512 x 5120 x
// 4096 in 128 x 128 tiles (160 of 256 CUs) 14 us.
template <int BM_, int BN_, int WGM_, int WGN_, int SA_, int SB_, int WPE_>
struct MxTile {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, SA = SA_, SB = SB_, WPE = WPE_;
  static constexpr int WAVES = WGM * WGN, THREADS = 64 * WAVES;
  static constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 32, TN = WN / 32;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, B_BASE = SA * A_BYTES, LDS = B_BASE + SB * B_BYTES;
  static constexpr int NDA = BM / 8 / WAVES, NDB = BN / 8 / WAVES, ND = NDA + NDB;  // DMA instructions per wavefront and step
  // instructions that may be in flight when step kt + 1 has to have landed: those behind its B, those behind its A
  static constexpr int BEHIND_B = NDA + (SB - 2) * ND, BEHIND_A = (SA - 2) * ND;
  static constexpr int FLY = BEHIND_A < BEHIND_B ? BEHIND_A : BEHIND_B;
  static constexpr int NS = TM + TN;  // loads of scales, in the first step of four
  static constexpr int GROUP_M = BM >= 256 ? 4 : 8;
  static constexpr int MIN_STEPS = SA > SB ? SA : SB;
  static_assert(WM % 32 == 0 && WN % 32 == 0 && NDA >= 1 && NDB >= 1 && (TN == 1 || TN == 2 || TN == 4), "whole fragments, whole instructions");
  static_assert(WAVES % 2 == 0, "the chunk that a lane fetches is the same in each of its wavefront's instructions");
  static_assert(SA >= 2 && SB >= 2 && FLY + ND + NS <= 63 && LDS <= 160 * 1024, "vmcnt has 6 bits; LDS");
};

template <int BYTE>
__device__ __forceinline__ v16f mfma_mx32(v4i a, v4i w, v16f acc, int a_scale, int w_scale) {
  const v8i w8 = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const v8i a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, w8, acc, 4, 4, BYTE, a_scale, BYTE, w_scale);
}

// The 16 bytes lane half h holds of a row's 32 scales (bytes 16 h ..) -> those of its blocks: byte j of the result is byte 2 j + h.
struct Scales {
  uint32_t w[4];
};
__device__ __forceinline__ Scales order_scales(v4u d) {
  auto even = [](uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x06040200u); };
  auto odd = [](uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07050301u); };
  // (the upper half of the lanes of the first operand and the lower half of the second change places)
  const auto p = __builtin_amdgcn_permlane32_swap(even(d[0], d[1]), odd(d[0], d[1]), false, false);
  const auto q = __builtin_amdgcn_permlane32_swap(even(d[2], d[3]), odd(d[2], d[3]), false, false);
  return {{(uint32_t)p[0], (uint32_t)q[0], (uint32_t)p[1], (uint32_t)q[1]}};
}

template <class C, int OUT>
__global__ __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(C::WPE, C::WPE))) void
gemm_mxfp4_tile(Mx4Gemm g, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  constexpr int TM = C::TM, TN = C::TN, MF = TM * TN, SA = C::SA, SB = C::SB, NDA = C::NDA, NDB = C::NDB;
  constexpr int WAVES = C::WAVES, WM = C::WM, WN = C::WN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WGN, wn = wave % C::WGN, r32 = lane & 31, h = lane >> 5;
  const int KB = g.K / kMxBlock, KT = max((g.K + 255) / 256, C::MIN_STEPS), S = (g.K + 127) / 128 * 4;
  const int ntiles = tiles_m * tiles_n;

  // Where the panels and scales of a tile are. Rows that do not exist lie beyond num_records: nothing is fetched for them and they
  // are zeros, codes and scales. No tile (behind the last): nothing at all.
  struct Source {
    const uint8_t *a, *b, *as, *bs;
    int na, nb, nas, nbs, m0, n0;
  };
  auto source_of = [&](int tile) -> Source {
    Source s = {};
    if (tile >= ntiles) return s;
    int tm, tn;
    tile_of_block<C::GROUP_M>(tile, ntiles, tiles_m, tiles_n, &tm, &tn);
    s.m0 = tm * C::BM;
    s.n0 = tn * C::BN;
    const int rm = min(C::BM, g.M - s.m0) - 1, rn = min(C::BN, g.N - s.n0) - 1;
    s.a = g.a + (int64_t)s.m0 * g.lda;
    s.b = g.b + (int64_t)s.n0 * g.ldb;
    s.as = g.a_scale + (int64_t)s.m0 * g.ldas;
    s.bs = g.b_scale + (int64_t)s.n0 * g.ldbs;
    s.na = rm * (int)g.lda + g.K / 2;
    s.nb = rn * (int)g.ldb + g.K / 2;
    s.nas = rm * (int)g.ldas + S;
    s.nbs = rn * (int)g.ldbs + S;
    return s;
  };
  auto buffer = [](const uint8_t* p, int bytes) -> __amdgpu_buffer_rsrc_t {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
  };

  // DMA instruction p of this wavefront fills panel rows 8 q .. 8 q + 7, q = wave + WAVES p: lane l lands on row l / 8, position
  // l % 8 and fetches the chunk that the swizzle stores there.
  const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  uint32_t off_a[NDA], off_b[NDB];
#pragma unroll
  for (int p = 0; p < NDA; ++p) {
    const int row = 8 * (wave + WAVES * p) + (lane >> 3);
    off_a[p] = (uint32_t)row * (uint32_t)g.lda + 16 * chunk;
  }
#pragma unroll
  for (int p = 0; p < NDB; ++p) {
    const int row = 8 * (wave + WAVES * p) + (lane >> 3), in = row % WN;
    off_b[p] = (uint32_t)(row - in + TN * (in % 32) + in / 32) * (uint32_t)g.ldb + 16 * chunk;
  }
  // Chunks behind K of a row go to an offset beyond the descriptor: zeros.
  auto dma_a = [&](const Source& s, int kt, int stage, int p) {
    const uint32_t beyond = 8 * kt + chunk < KB ? 0u : 0x80000000u;
    const __amdgpu_buffer_rsrc_t src = buffer(s.a, s.na);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        src, (__attribute__((address_space(3))) void*)(smem + stage + (wave + WAVES * p) * 1024), 16,
        (int)(off_a[p] | beyond), kt * 128, 0, 0);
  };
  auto dma_b = [&](const Source& s, int kt, int stage, int p) {
    const uint32_t beyond = 8 * kt + chunk < KB ? 0u : 0x80000000u;
    const __amdgpu_buffer_rsrc_t src = buffer(s.b, s.nb);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        src, (__attribute__((address_space(3))) void*)(smem + stage + (wave + WAVES * p) * 1024), 16,
        (int)(off_b[p] | beyond), kt * 128, 0, 0);
  };

  // operand read map: round j reads chunk 2 j + h; panel rows of a fragment are 32 in a row, A and B alike
  uint32_t rd_a[4], rd_b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t at = ((2 * j + h) ^ ((r32 >> 1) & 7)) << 4;
    rd_a[j] = (wm * WM + r32) * 128 + at;
    rd_b[j] = (wn * WN + r32) * 128 + at;
  }
  // (__restrict__ gives the loads alias information: without it the compiler puts a wait for every DMA in flight in front of
  // an LDS read. The stage read is never one that DMA fills; the waits before the barriers order the two.)
  auto read = [&](const uint8_t* __restrict__ st, uint32_t at, int i) -> v4i {
    return *reinterpret_cast<const v4i*>(st + at + i * 32 * 128);
  };

  uint32_t off_as[TM], off_bs[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) off_as[i] = (uint32_t)(wm * WM + 32 * i + r32) * (uint32_t)g.ldas + 16 * h;
#pragma unroll
  for (int j = 0; j < TN; ++j) off_bs[j] = (uint32_t)(wn * WN + TN * r32 + j) * (uint32_t)g.ldbs + 16 * h;
  v4u a_raw[TM], b_raw[TN];
  // the scales of steps kt .. kt + 3, kt a multiple of 4; words behind the row's last: 0, a scale of 2^-127 for codes that are 0
  auto load_scales = [&](const Source& s, int kt) {
    const int at = 8 * kt;
    const __amdgpu_buffer_rsrc_t as = buffer(s.as, s.nas), bs = buffer(s.bs, s.nbs);
    if (at + 32 <= S) {
#pragma unroll
      for (int i = 0; i < TM; ++i) a_raw[i] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(as, off_as[i], at, 0));
#pragma unroll
      for (int j = 0; j < TN; ++j) b_raw[j] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(bs, off_bs[j], at, 0));
    } else {
      uint32_t beyond[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) beyond[k] = at + 16 * h + 4 * k < S ? 0u : 0x80000000u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
          a_raw[i][k] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(as, (off_as[i] + 4 * k) | beyond[k], at, 0);
#pragma unroll
        for (int j = 0; j < TN; ++j)
          b_raw[j][k] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(bs, (off_bs[j] + 4 * k) | beyond[k], at, 0);
      }
    }
  };
  Scales sa[TM], sb[TN];
  auto order = [&]() {
#pragma unroll
    for (int i = 0; i < TM; ++i) sa[i] = order_scales(a_raw[i]);
#pragma unroll
    for (int j = 0; j < TN; ++j) sb[j] = order_scales(b_raw[j]);
  };
  float bias[TN];
  auto load_bias = [&](const Source& s) { mx_bias<TN, OUT>(g, s.n0 + wn * WN + TN * r32, bias); };

  Source cur = source_of(blockIdx.x), nxt = cur;
  load_scales(cur, 0);
  load_bias(cur);
  // windows before step 0: what the steps before would have fetched
#pragma unroll
  for (int w = -C::MIN_STEPS; w < 0; ++w) {
    if (w + SB >= 0) {
#pragma unroll
      for (int p = 0; p < NDB; ++p) dma_b(cur, w + SB, C::B_BASE + (w + SB) * C::B_BYTES, p);
    }
    if (w + SA >= 0 && w < -1) {  // (the last window's A goes out in step 0)
#pragma unroll
      for (int p = 0; p < NDA; ++p) dma_a(cur, w + SA, (w + SA) * C::A_BYTES, p);
    }
  }
  order();
  wait_and_barrier<C::FLY + NDB>();  // step 0 has landed

  int a_prev = (SA - 1) * C::A_BYTES, a_cur = 0, a_next = C::A_BYTES;
  int b_cur = C::B_BASE, b_next = C::B_BASE + C::B_BYTES;
  v4i a[2][TM], b[2][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) a[0][i] = read(smem + a_cur, rd_a[0], i);
#pragma unroll
  for (int j = 0; j < TN; ++j) b[0][j] = read(smem + b_cur, rd_b[0], j);

  for (int tile = blockIdx.x;; tile += gridDim.x) {
    nxt = source_of(tile + gridDim.x);
    v16f acc[TM][TN];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = bias[j];

    // T: step of four, which decides the words of the scales
    auto step = [&](int kt, auto t_tag) {
      constexpr int T = decltype(t_tag)::value;
      if (T == 0) {
        if (kt + 4 < KT)
          load_scales(cur, kt + 4);
        else
          load_scales(nxt, 0);
      }
      const bool a_here = kt - 1 + SA < KT, b_here = kt + SB < KT;  // else: the next tile's
      const Source a_src = a_here ? cur : nxt, b_src = b_here ? cur : nxt;
      const int a_kt = kt - 1 + SA - (a_here ? 0 : KT), b_kt = kt + SB - (b_here ? 0 : KT);
      auto round = [&](auto j_tag, auto items) {
        constexpr int J = decltype(j_tag)::value;
#pragma unroll
        for (int s = 0; s < MF; ++s) {
          items(s);
          const int i = s / TN, j = s % TN;
          acc[i][j] = mfma_mx32<J>(a[J & 1][i], b[J & 1][j], acc[i][j], sa[i].w[T], sb[j].w[T]);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // fragments of the round after J, over the first three quarters of the MFMAs
      auto reads = [&](int s, int j_next, int a_stage, int b_stage) {
        constexpr int NR = TM + TN;
#pragma unroll
        for (int q = 0; q < NR; ++q)
          if (q * MF * 3 / (4 * NR) == s) {
            if (q < TN)
              b[j_next & 1][q] = read(smem + b_stage, rd_b[j_next], q);
            else
              a[j_next & 1][q - TN] = read(smem + a_stage, rd_a[j_next], q - TN);
          }
      };
      round(std::integral_constant<int, 0>{}, [&](int s) {
        reads(s, 1, a_cur, b_cur);
#pragma unroll
        for (int p = 0; p < NDA; ++p)
          if (2 * p * MF / NDA == s) dma_a(a_src, a_kt, a_prev, p);
      });
      round(std::integral_constant<int, 1>{}, [&](int s) {
        reads(s, 2, a_cur, b_cur);
#pragma unroll
        for (int p = 0; p < NDA; ++p)
          if (2 * p * MF / NDA == MF + s) dma_a(a_src, a_kt, a_prev, p);
      });
      round(std::integral_constant<int, 2>{}, [&](int s) { reads(s, 3, a_cur, b_cur); });
      wait_and_barrier<C::FLY + (T == 0 ? C::NS : 0)>();
      round(std::integral_constant<int, 3>{}, [&](int s) {
        reads(s, 0, a_next, b_next);
#pragma unroll
        for (int p = 0; p < NDB; ++p)
          if (p * MF / NDB == s) dma_b(b_src, b_kt, b_cur, p);
      });
      a_prev = a_cur;
      a_cur = a_next;
      a_next = a_next + C::A_BYTES == C::B_BASE ? 0 : a_next + C::A_BYTES;
      b_cur = b_next;
      b_next = b_next + C::B_BYTES == C::LDS ? C::B_BASE : b_next + C::B_BYTES;
    };
    for (int kt = 0; kt < KT; kt += 4) {
      step(kt, std::integral_constant<int, 0>{});
      if (kt + 1 < KT) step(kt + 1, std::integral_constant<int, 1>{});
      if (kt + 2 < KT) step(kt + 2, std::integral_constant<int, 2>{});
      if (kt + 3 < KT) step(kt + 3, std::integral_constant<int, 3>{});
      order();
    }
    const bool more = tile + (int)gridDim.x < ntiles;
    if (more) load_bias(nxt);

    store_mx_tile<TM, TN, OUT>(acc, g, cur.m0, C::BM, wm * WM + 4 * h, cur.n0 + wn * WN + TN * r32);
    if (!more) break;
    cur = nxt;
  }
  wait_vm<0>();  // no DMA outlives the workgroup
}

template <class C, int OUT>
int launch_tile_out(const Mx4Gemm& g, hipStream_t stream) {
  static bool lds_allowed[64];
  if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&gemm_mxfp4_tile<C, OUT>), C::LDS, lds_allowed)) return rc;
  const int cus = cu_count();
  if (cus <= 0) {
    set_error("cannot query the CU count of the current device");
    return CDIT_EHIP;
  }
  const int tiles_m = (g.M + C::BM - 1) / C::BM, tiles_n = (g.N + C::BN - 1) / C::BN;
  hipLaunchKernelGGL((gemm_mxfp4_tile<C, OUT>), dim3((unsigned)std::min(tiles_m * tiles_n, cus * C::WPE)), dim3(C::THREADS),
                     C::LDS, stream, g, tiles_m, tiles_n);
  return 0;
}
template <class C>
int launch_tile(const Mx4Gemm& g, hipStream_t stream) {
  switch (g.out_dtype) {
    case CDIT_DT_F16: return launch_tile_out<C, CDIT_DT_F16>(g, stream);
    case CDIT_DT_F32: return launch_tile_out<C, CDIT_DT_F32>(g, stream);
    default: return launch_tile_out<C, CDIT_DT_BF16>(g, stream);
  }
}

}  // namespace

// Times from problems of a quarter of a round to eight rounds at K = 1024 and 5120.
static const MxTime kTimes[] = {
    {1, 256, 256, 8000, 2800, 1880, 1890}, {5, 128, 256, 3500, 2700, 1070, 1117}, {6, 256, 128, 3500, 2700, 1070, 1117},
    {2, 128, 128, 2700, 1000, 610, 579},    {3, 64, 128, 2700, 900, 430, 372},     {7, 128, 64, 2700, 1000, 412, 360},
    {4, 64, 64, 2500, 1060, 319, 235},      {8, 32, 64, 2500, 850, 294, 174}};

int choose_gemm_mxfp4(const Mx4Gemm& g) {
  if (mx_rows_fit(false, g.M, g.N, g.ldb)) return kMxRows;
  const int cus = cu_count();
  return tiles_fit(g, 1) ? fastest_tile(kTimes, sizeof(kTimes) / sizeof(kTimes[0]), false, g, cus > 0 ? cus : 256) : 0;
}

int launch_gemm_mxfp4(const Mx4Gemm& g, int variant, hipStream_t stream) {
  if (variant < 0) variant = choose_gemm_mxfp4(g);
  if (variant == kMxRows && mx_rows_can(g.M, g.ldb)) return launch_gemm_mxfp4_rows(g, stream);
  if (!tiles_fit(g, 1)) variant = 0;
  if (variant == 1 && g.out_dtype == CDIT_DT_F32) variant = 5;  // (no registers left for 16-byte stores of 256 x 256)
  switch (variant) {
    case 1: {
      using C = MxTile<256, 256, 2, 2, 3, 2, 1>;
      return g.out_dtype == CDIT_DT_F16 ? launch_tile_out<C, CDIT_DT_F16>(g, stream) : launch_tile_out<C, CDIT_DT_BF16>(g, stream);
    }
    case 2: return launch_tile<MxTile<128, 128, 2, 2, 3, 2, 2>>(g, stream);
    case 3: return launch_tile<MxTile<64, 128, 2, 2, 3, 3, 2>>(g, stream);
    case 4: return launch_tile<MxTile<64, 64, 2, 2, 4, 4, 2>>(g, stream);
    case 5: return launch_tile<MxTile<128, 256, 2, 2, 3, 3, 1>>(g, stream);
    case 6: return launch_tile<MxTile<256, 128, 2, 2, 3, 3, 1>>(g, stream);
    case 7: return launch_tile<MxTile<128, 64, 2, 2, 3, 3, 2>>(g, stream);
    case 8: return launch_tile<MxTile<32, 64, 1, 2, 4, 4, 3>>(g, stream);
  }
  const dim3 grid((unsigned)((g.N + 127) / 128), (unsigned)std::min((g.M + 31) / 32, 65535));
  switch (g.out_dtype) {
    case CDIT_DT_F16: hipLaunchKernelGGL(gemm_mxfp4_direct<CDIT_DT_F16>, grid, dim3(256), 0, stream, g); break;
    case CDIT_DT_F32: hipLaunchKernelGGL(gemm_mxfp4_direct<CDIT_DT_F32>, grid, dim3(256), 0, stream, g); break;
    default: hipLaunchKernelGGL(gemm_mxfp4_direct<CDIT_DT_BF16>, grid, dim3(256), 0, stream, g);
  }
  return 0;
}

}  // namespace cdit
