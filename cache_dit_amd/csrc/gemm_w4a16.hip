// Weight-only GEMM with an MXFP4 weight (w4a16): out = epi(X W^T + bias), X bf16.
//
// The weight's codes become bf16 with v_cvt_scalef32_pk_bf16_fp4, which applies the block's scale (exact: a code
// has two significant bits), and are multiplied with v_mfma_f32_16x16x32_bf16. Lane l holds row l & 15; of a step of
// 128 along K its 16 bytes of codes are block l >> 4, 32 consecutive k, which feed four instructions of 8 k each.
#include <algorithm>
#include <type_traits>

#include "gemm_common.h"
#include "mx_tile.h"
#include "mxfp4_device.h"

namespace cdit {
namespace {

// A wavefront per 32 x 32 outputs, operands straight from memory: any stride (the tiles below address with 32 bits).
__global__ __launch_bounds__(256) void gemm_w4a16_direct(Mx4Gemm g) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kg = lane >> 4;
  const int n0 = blockIdx.x * 128 + wave * 32;
  if (n0 >= g.N) return;
  const int blocks = g.K / kMxBlock, steps = (g.K + 127) / 128;
  for (int m0 = blockIdx.y * 32; m0 < g.M; m0 += gridDim.y * 32) {
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
        wsv[i] = in ? mx_scale_or_nan(ws[i][4 * s]) : 1.0f;
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
          if (m < g.M && n < g.N) store_mx_one<CDIT_DT_BF16>(g, m, n, acc[i][j][e]);
        }
  }
}

// ---------------------------------------------------------------------------
// Tiles through LDS, for more than a few rows: the frame of the w4a4 tiles (gemm_mxfp4.hip) with steps of 64 along K (a
// 128-byte line of each row of X), four of them to a line of the weight's codes. A wavefront's blocks are
// v_mfma_f32_32x32x16_bf16: lane l is row l & 31, and in instruction q of a step the elements 32 (l >> 5) + 8 q .. + 7: block
// 2 T + (l >> 5) of step T, so that a lane's 16 bytes of codes are the four instructions' operands under one scale.
//
//   instructions q = 0 .. 2 of step x: MFMAs; meanwhile X's fragments of q + 1 are read and the weight's converted
//   wait: own reads done, own DMA of step x + 1 landed; barrier: so are everyone's, and X's stage of step x is free
//   q = 3: MFMAs; meanwhile codes and first fragments of step x + 1 are read, and converted
//   DMA of X's step x + SA from here to the end of the next step's q = 2; of the weight's line k + SB in the first two steps of
//   line k + 1 (the codes of a line are read one step ahead)
//
// Measured: 4608 x 5120 x 5120 (M x N x K) 185 to 190 us, 1.27 to 1.30 PFLOP/s (256 x 128 tiles; 200 in 256 x 256, 191 in 128 x
// 256), 16384 x 5120 x 5120 592 us, 1.45 (256 x 256 tiles); the library's bf16 product reaches 1.36 on 16384 x 16384 x 16384. Bound
// by the matrix cores at the clock they run at.
template <int BM_, int BN_, int WGM_, int WGN_, int SA_, int WPE_>
struct W4Tile {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, SA = SA_, SB = 2, WPE = WPE_;
  static constexpr int WAVES = WGM * WGN, THREADS = 64 * WAVES;
  static constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 32, TN = WN / 32;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, B_BASE = SA * A_BYTES, LDS = B_BASE + SB * B_BYTES;
  static constexpr int NDA = BM / 8 / WAVES, NDB = BN / 8 / WAVES;  // DMA instructions per wavefront and step / line
  static constexpr int FLY = (SA - 2) * NDA;  // that may be in flight when step x + 1 has to have landed
  static constexpr int GROUP_M = BM >= 256 ? 4 : 8;
  static_assert(WM % 32 == 0 && WN % 32 == 0 && NDA >= 1 && NDB >= 1 && (TN == 1 || TN == 2 || TN == 4), "whole fragments, whole instructions");
  static_assert(WAVES % 2 == 0, "the chunk that a lane fetches is the same in each of its wavefront's instructions");
  static_assert(SA >= 3 && SA <= 8 && FLY + NDB + 2 * TN <= 63 && LDS <= 160 * 1024, "a tile has eight steps at least; vmcnt has 6 bits; LDS");
};

template <class C>
__global__ __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(C::WPE, C::WPE))) void
gemm_w4a16_tile(Mx4Gemm g, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  constexpr int TM = C::TM, TN = C::TN, MF = TM * TN, SA = C::SA, SB = C::SB, NDA = C::NDA, NDB = C::NDB;
  constexpr int WAVES = C::WAVES, WM = C::WM, WN = C::WN, OUT = CDIT_DT_BF16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WGN, wn = wave % C::WGN, r32 = lane & 31, h = lane >> 5;
  const int KB = g.K / kMxBlock, KL = max((g.K + 255) / 256, SB), S = (g.K + 127) / 128 * 4;  // KL: lines of codes
  const int ntiles = tiles_m * tiles_n;

  struct Source {  // as in the w4a4 tiles
    const uint8_t *a, *b, *bs;
    int na, nb, nbs, m0, n0;
  };
  auto source_of = [&](int tile) -> Source {
    Source s = {};
    if (tile >= ntiles) return s;
    int tm, tn;
    tile_of_block<C::GROUP_M>(tile, ntiles, tiles_m, tiles_n, &tm, &tn);
    s.m0 = tm * C::BM;
    s.n0 = tn * C::BN;
    const int rm = min(C::BM, g.M - s.m0) - 1, rn = min(C::BN, g.N - s.n0) - 1;
    s.a = g.a + 2 * (int64_t)s.m0 * g.lda;
    s.b = g.b + (int64_t)s.n0 * g.ldb;
    s.bs = g.b_scale + (int64_t)s.n0 * g.ldbs;
    s.na = 2 * (rm * (int)g.lda + g.K);
    s.nb = rn * (int)g.ldb + g.K / 2;
    s.nbs = rn * (int)g.ldbs + S;
    return s;
  };
  auto buffer = [](const uint8_t* p, int bytes) -> __amdgpu_buffer_rsrc_t {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
  };

  const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  uint32_t off_a[NDA], off_b[NDB];
#pragma unroll
  for (int p = 0; p < NDA; ++p)
    off_a[p] = (uint32_t)(8 * (wave + WAVES * p) + (lane >> 3)) * (uint32_t)g.lda * 2 + 16 * chunk;
#pragma unroll
  for (int p = 0; p < NDB; ++p) {
    const int row = 8 * (wave + WAVES * p) + (lane >> 3), in = row % WN;
    off_b[p] = (uint32_t)(row - in + TN * (in % 32) + in / 32) * (uint32_t)g.ldb + 16 * chunk;
  }
  auto dma_a = [&](const Source& s, int x, int stage, int p) {
    const uint32_t beyond = 8 * x + chunk < 4 * KB ? 0u : 0x80000000u;  // (8 elements a chunk)
    const __amdgpu_buffer_rsrc_t src = buffer(s.a, s.na);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        src, (__attribute__((address_space(3))) void*)(smem + stage + (wave + WAVES * p) * 1024), 16,
        (int)(off_a[p] | beyond), x * 128, 0, 0);
  };
  auto dma_b = [&](const Source& s, int k, int stage, int p) {
    const uint32_t beyond = 8 * k + chunk < KB ? 0u : 0x80000000u;
    const __amdgpu_buffer_rsrc_t src = buffer(s.b, s.nb);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        src, (__attribute__((address_space(3))) void*)(smem + stage + (wave + WAVES * p) * 1024), 16,
        (int)(off_b[p] | beyond), k * 128, 0, 0);
  };

  // X: chunk 4 h + q of a row; codes: chunk 2 T + h
  uint32_t rd_a[4], rd_b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    rd_a[j] = (wm * WM + r32) * 128 + (((4 * h + j) ^ ((r32 >> 1) & 7)) << 4);
    rd_b[j] = (wn * WN + r32) * 128 + (((2 * j + h) ^ ((r32 >> 1) & 7)) << 4);
  }
  auto read = [&](const uint8_t* __restrict__ st, uint32_t at, int i) -> v4u {
    return *reinterpret_cast<const v4u*>(st + at + i * 32 * 128);
  };

  // scales: the 8 bytes of a row for a line, of which a lane needs bytes 2 T + h; words behind the row's last: 0
  uint32_t off_bs[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) off_bs[j] = (uint32_t)(wn * WN + TN * r32 + j) * (uint32_t)g.ldbs;
  v2u raw[TN];
  auto load_scales = [&](const Source& s, int k) {
    const int at = 8 * k;
    const __amdgpu_buffer_rsrc_t bs = buffer(s.bs, s.nbs);
    if (at + 8 <= S) {
#pragma unroll
      for (int j = 0; j < TN; ++j) raw[j] = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(bs, off_bs[j], at, 0));
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        raw[j][0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(bs, off_bs[j] | (at < S ? 0u : 0x80000000u), at, 0);
        raw[j][1] = 0;
      }
    }
  };
  uint32_t sb[TN];
  auto order = [&]() {
#pragma unroll
    for (int j = 0; j < TN; ++j) sb[j] = __builtin_amdgcn_perm(raw[j][1], raw[j][0], h ? 0x07050301u : 0x06040200u);
  };

  float bias[TN];
  Source cur = source_of(blockIdx.x), nxt = cur;
  load_scales(cur, 0);
  mx_bias<TN, OUT>(g, cur.n0 + wn * WN + TN * r32, bias);
#pragma unroll
  for (int k = 0; k < SB; ++k)
#pragma unroll
    for (int p = 0; p < NDB; ++p) dma_b(cur, k, C::B_BASE + k * C::B_BYTES, p);
#pragma unroll
  for (int x = 0; x < SA - 1; ++x)
#pragma unroll
    for (int p = 0; p < NDA; ++p) dma_a(cur, x, x * C::A_BYTES, p);
  order();
  // X's step SA - 1 goes out in step 0 as a whole: its window's part in front of step 0 here
  constexpr int NDA3 = (NDA + 3) / 4;  // instructions of a window that go out in q = 3
#pragma unroll
  for (int p = 0; p < NDA3; ++p) dma_a(cur, SA - 1, (SA - 1) * C::A_BYTES, p);
  wait_and_barrier<C::FLY + NDA3>();  // step 0 and the lines have landed

  int a_prev = (SA - 1) * C::A_BYTES, a_cur = 0, a_next = C::A_BYTES;
  int b_prev = C::B_BASE + (SB - 1) * C::B_BYTES, b_cur = C::B_BASE, b_next = C::B_BASE + C::B_BYTES;
  v4u a[2][TM], wc[2][TN];  // X's fragments by q, codes by step
  v8bf wb[2][TN];           // converted, by q
  float fs[2][TN];          // scales by step
  auto scale_of = [&](uint32_t bytes, int t) -> float { return mx_scale_or_nan((bytes >> (8 * t)) & 255); };
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    wc[0][j] = read(smem + b_cur, rd_b[0], j);
    fs[0][j] = scale_of(sb[j], 0);
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) a[0][i] = read(smem + a_cur, rd_a[0], i);
#pragma unroll
  for (int j = 0; j < TN; ++j) wb[0][j] = mx_to_bf16(wc[0][j][0], fs[0][j]);

  for (int tile = blockIdx.x;; tile += gridDim.x) {
    nxt = source_of(tile + gridDim.x);
    v16f acc[TM][TN];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = bias[j];

    auto step = [&](int k, auto t_tag) {
      constexpr int T = decltype(t_tag)::value, P = T & 1, Q = P ^ 1;
      const int x = 4 * k + T;
      // the window of step x - 1 (X's step x - 1 + SA), and that of step x
      const bool here0 = x - 1 + SA < 4 * KL, here1 = x + SA < 4 * KL, b_here = k - 1 + SB < KL;
      const Source src0 = here0 ? cur : nxt, src1 = here1 ? cur : nxt, b_src = b_here ? cur : nxt;
      const int x0 = x - 1 + SA - (here0 ? 0 : 4 * KL), x1 = x + SA - (here1 ? 0 : 4 * KL), bk = k - 1 + SB - (b_here ? 0 : KL);
      // (T = 0, 1) half of line k - 1 + SB, into the stage of line k - 1; line SB - 1 of the first tile is there already
      const bool b_due = T < 2 && !(tile == (int)blockIdx.x && k == 0);
      if (T == 0) {
        if (k + 1 < KL)
          load_scales(cur, k + 1);
        else
          load_scales(nxt, 0);
      }
      auto quarter = [&](auto q_tag, auto items) {
        constexpr int QQ = decltype(q_tag)::value;
#pragma unroll
        for (int s = 0; s < MF; ++s) {
          items(s);
          const int i = s / TN, j = s % TN;
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a[QQ & 1][i]), wb[QQ & 1][j], acc[i][j], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // instructions of the window of step x - 1 that go out in q = 0 .. 2, evenly
      constexpr int REST = NDA - NDA3;
      auto window = [&](int slot) {
#pragma unroll
        for (int p = 0; p < REST; ++p)
          if (p * 3 * MF / (REST > 0 ? REST : 1) == slot) dma_a(src0, x0, a_prev, NDA3 + p);
      };
      auto reads_a = [&](int s, int q_next, int stage) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
          if (i * MF * 3 / (4 * TM) == s) a[q_next & 1][i] = read(smem + stage, rd_a[q_next], i);
      };
      auto convert = [&](int s, int q_next) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
          if (j * MF / TN == s) wb[q_next & 1][j] = mx_to_bf16(wc[P][j][q_next], fs[P][j]);
      };
      quarter(std::integral_constant<int, 0>{}, [&](int s) {
        reads_a(s, 1, a_cur);
        convert(s, 1);
        window(s);
      });
      quarter(std::integral_constant<int, 1>{}, [&](int s) {
        reads_a(s, 2, a_cur);
        convert(s, 2);
        window(MF + s);
#pragma unroll
        for (int p = 0; p < NDB; ++p)
          if (T < 2 && p % 2 == T && (p / 2) * MF / ((NDB + 1) / 2) == s) {
            if (b_due) dma_b(b_src, bk, b_prev, p);
          }
      });
      quarter(std::integral_constant<int, 2>{}, [&](int s) {
        reads_a(s, 3, a_cur);
        convert(s, 3);
        window(2 * MF + s);
      });
      // (this step's scales and line instructions are younger than what has to have landed; behind a line's last, two
      // windows go out before its codes are read)
      constexpr int YOUNG = T == 0 ? TN : 0, LINE = T == 0 ? (NDB + 1) / 2 : T == 1 ? NDB / 2 : 0;
      constexpr int FLY = T == 3 && C::FLY > 2 * NDA ? 2 * NDA : C::FLY;
      if (b_due)
        wait_and_barrier<FLY + YOUNG + LINE>();
      else
        wait_and_barrier<FLY + YOUNG>();
      if (T == 3) order();
      quarter(std::integral_constant<int, 3>{}, [&](int s) {
        // codes first: they are converted in the second half
#pragma unroll
        for (int j = 0; j < TN; ++j)
          if (j * (MF / 2) / (2 * TN) == s) {
            wc[Q][j] = read(smem + (T == 3 ? b_next : b_cur), rd_b[(T + 1) & 3], j);
            fs[Q][j] = scale_of(sb[j], (T + 1) & 3);
          }
        reads_a(s, 0, a_next);
#pragma unroll
        for (int p = 0; p < NDA3; ++p)
          if (p * MF / NDA3 == s) dma_a(src1, x1, a_cur, p);
#pragma unroll
        for (int j = 0; j < TN; ++j)
          if (MF / 2 + j * (MF / 2) / TN == s) wb[0][j] = mx_to_bf16(wc[Q][j][0], fs[Q][j]);
      });
      a_prev = a_cur;
      a_cur = a_next;
      a_next = a_next + C::A_BYTES == C::B_BASE ? 0 : a_next + C::A_BYTES;
      if (T == 3) {
        b_prev = b_cur;
        b_cur = b_next;
        b_next = b_next + C::B_BYTES == C::LDS ? C::B_BASE : b_next + C::B_BYTES;
      }
    };
    for (int k = 0; k < KL; ++k) {
      step(k, std::integral_constant<int, 0>{});
      step(k, std::integral_constant<int, 1>{});
      step(k, std::integral_constant<int, 2>{});
      step(k, std::integral_constant<int, 3>{});
    }
    const bool more = tile + (int)gridDim.x < ntiles;
    if (more) mx_bias<TN, OUT>(g, nxt.n0 + wn * WN + TN * r32, bias);
    store_mx_tile<TM, TN, OUT>(acc, g, cur.m0, C::BM, wm * WM + 4 * h, cur.n0 + wn * WN + TN * r32);
    if (!more) break;
    cur = nxt;
  }
  wait_vm<0>();  // no DMA outlives the workgroup
}

template <class C>
int launch_tile(const Mx4Gemm& g, hipStream_t stream) {
  static bool lds_allowed[64];
  if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&gemm_w4a16_tile<C>), C::LDS, lds_allowed)) return rc;
  const int cus = cu_count();
  if (cus <= 0) {
    set_error("cannot query the CU count of the current device");
    return CDIT_EHIP;
  }
  const int tiles_m = (g.M + C::BM - 1) / C::BM, tiles_n = (g.N + C::BN - 1) / C::BN;
  hipLaunchKernelGGL(gemm_w4a16_tile<C>, dim3((unsigned)std::min(tiles_m * tiles_n, cus * C::WPE)), dim3(C::THREADS), C::LDS,
                     stream, g, tiles_m, tiles_n);
  return 0;
}

// ---------------------------------------------------------------------------
// Few tiles (a prompt's rows): a workgroup per BM x BN outputs whose wavefronts split K as well. K advances in lines of 256; of
// each, wavefront group g = 0 .. 3 takes the elements 64 g .. 64 g + 63 of the same 32 x 32 blocks, and the four partial sums
// meet in LDS at the end. Such a problem has one workgroup a CU: with one wavefront per block, as in the tiles above, every
// step of 64 waited for LDS reads and conversions that a single MFMA cannot cover (64 x 64 tiles, 77 x 5120 x 4096 (M x N x K):
// 0.28 us a step of 64); four wavefronts per SIMD cover each other.
template <int BM_, int BN_, int D_>
struct W4Split {
  static constexpr int BM = BM_, BN = BN_, D = D_, RB = BM / 32, CB = BN / 32, WAVES = 4 * RB * CB, THREADS = 64 * WAVES;
  static constexpr int PANEL = BM * 128, A_BYTES = 4 * PANEL, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int JOIN = 3 * BM * BN * 4, LDS = D * STAGE > JOIN ? D * STAGE : JOIN;
  static constexpr int NDMA = STAGE / 1024, ND = (NDMA + WAVES - 1) / WAVES;  // DMA instructions of a line, of a wavefront
  static_assert(D >= 2 && (D - 1) * ND <= 63 && LDS <= 160 * 1024 && WAVES <= 16, "vmcnt has 6 bits; LDS");
};

template <class C>
__global__ __launch_bounds__(C::THREADS) void gemm_w4a16_split(Mx4Gemm g, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  constexpr int D = C::D, ND = C::ND, WAVES = C::WAVES, STAGE = C::STAGE, PANEL = C::PANEL, A_BYTES = C::A_BYTES;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = wave / (C::RB * C::CB), blk = wave % (C::RB * C::CB), rb = blk / C::CB, cb = blk % C::CB;
  const int r32 = lane & 31, h = lane >> 5;
  int tm, tn;
  tile_of_block<8>(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, &tm, &tn);
  const int m0 = tm * C::BM, n0 = tn * C::BN;
  const int KB = g.K / kMxBlock, KL = (g.K + 255) / 256, S = (g.K + 127) / 128 * 4;
  const int rm = min(C::BM, g.M - m0) - 1, rn = min(C::BN, g.N - n0) - 1;
  auto buffer = [](const uint8_t* p, int bytes) -> __amdgpu_buffer_rsrc_t {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t a_buf = buffer(g.a + 2 * (int64_t)m0 * g.lda, 2 * (rm * (int)g.lda + g.K));
  const __amdgpu_buffer_rsrc_t b_buf = buffer(g.b + (int64_t)n0 * g.ldb, rn * (int)g.ldb + g.K / 2);
  const __amdgpu_buffer_rsrc_t s_buf = buffer(g.b_scale + (int64_t)n0 * g.ldbs, rn * (int)g.ldbs + S);

  // DMA instruction q of a line fills 1 KiB: 8 rows of one of X's four panels, or of the codes; this wavefront's are wave +
  // WAVES p.
  auto dma = [&](int line, int stage) {
#pragma unroll
    for (int p = 0; p < ND; ++p) {
      const int q = wave + WAVES * p;
      if (q >= C::NDMA) continue;  // (uniform; the wait counts go by what this wavefront issues)
      const int byte = q * 1024, panel = byte / PANEL, row = (byte % PANEL) / 128 + (lane >> 3);
      const int chunk = (lane & 7) ^ ((row >> 1) & 7);
      if (byte < A_BYTES) {
        const int k = 256 * line + 64 * panel + 8 * chunk;
        const int at = (int)(k < g.K ? (uint32_t)row * (uint32_t)g.lda * 2 + 2 * k : 0x80000000u);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(a_buf, (__attribute__((address_space(3))) void*)(smem + stage + byte), 16, at, 0, 0, 0);
      } else {
        const int brow = (byte - A_BYTES) / 128 + (lane >> 3), c = (lane & 7) ^ ((brow >> 1) & 7), block = 8 * line + c;
        const int at = (int)(block < KB ? (uint32_t)brow * (uint32_t)g.ldb + 16 * block : 0x80000000u);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(b_buf, (__attribute__((address_space(3))) void*)(smem + stage + byte), 16, at, 0, 0, 0);
      }
    }
  };
  const int nd = C::NDMA / WAVES + (wave < C::NDMA % WAVES ? 1 : 0);  // instructions this wavefront issues for a line
  auto wait_lines = [&](int later) {  // at most `later` lines of this wavefront's DMA in flight
    if (nd == ND)
      wait_steps<ND, D - 1, true>(later);
    else
      wait_steps<ND - 1, D - 1, true>(later);
  };

  // fragment maps: X's chunk 4 h + q of this group's panel; codes' chunk 2 grp + h
  const int swz = (r32 >> 1) & 7;
  const uint32_t rd_a = grp * PANEL + (32 * rb + r32) * 128, rd_b = A_BYTES + (32 * cb + r32) * 128 + (((2 * grp + h) ^ swz) << 4);
  const uint32_t off_s = (uint32_t)(32 * cb + r32) * (uint32_t)g.ldbs + 4 * (grp >> 1);  // the word of this group's two bytes
  auto load_scale = [&](int line) -> uint32_t {
    const int at = (int)(8 * line + 4 * (grp >> 1) < S ? off_s + 8 * line : 0x80000000u);
    return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(s_buf, at, 0, 0);
  };
  auto read = [&](const uint8_t* __restrict__ st, uint32_t at) -> v4u { return *reinterpret_cast<const v4u*>(st + at); };

  v16f acc = {};
  uint32_t sc = load_scale(0), sc_next = 0;
#pragma unroll
  for (int l = 0; l < D - 1; ++l)
    if (l < KL) dma(l, l * STAGE);
  int stage = 0, free_stage = (D - 1) * STAGE;
  for (int l = 0; l < KL; ++l) {
    wait_lines(min(D - 2, KL - 1 - l));  // line l has landed; everyone is done with line l - 1
    if (l + 1 < KL) sc_next = load_scale(l + 1);
    if (l + D - 1 < KL) dma(l + D - 1, free_stage);
    const v4u c = read(smem + stage, rd_b);
    v4u a[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = read(smem + stage, rd_a + (((4 * h + q) ^ swz) << 4));
    const float f = mx_scale_or_nan((sc >> (8 * (2 * (grp & 1) + h))) & 255);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a[q]), mx_to_bf16(c[q], f), acc, 0, 0, 0);
    sc = sc_next;
    free_stage = stage;
    stage = stage + STAGE == D * STAGE ? 0 : stage + STAGE;
  }
  // join: groups 1 .. 3 leave their sums, group 0 adds them in turn
  wait_and_barrier<0>();
  float* const join = reinterpret_cast<float*>(smem);
  if (grp > 0) {
#pragma unroll
    for (int e = 0; e < 16; ++e) join[((grp - 1) * (C::RB * C::CB) + blk) * 1024 + 64 * e + lane] = acc[e];
  }
  __syncthreads();
  if (grp > 0) return;
  float bias[1];
  mx_bias<1, CDIT_DT_BF16>(g, n0 + 32 * cb + r32, bias);
  v16f out[1][1];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float v = acc[e];
#pragma unroll
    for (int k = 0; k < 3; ++k) v += join[(k * (C::RB * C::CB) + blk) * 1024 + 64 * e + lane];
    out[0][0][e] = v + bias[0];
  }
  store_mx_tile<1, 1, CDIT_DT_BF16>(out, g, m0, C::BM, 32 * rb + 4 * h, n0 + 32 * cb + r32);
}

template <class C>
int launch_split(const Mx4Gemm& g, hipStream_t stream) {
  static bool lds_allowed[64];
  if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&gemm_w4a16_split<C>), C::LDS, lds_allowed)) return rc;
  const int tiles_m = (g.M + C::BM - 1) / C::BM, tiles_n = (g.N + C::BN - 1) / C::BN;
  hipLaunchKernelGGL(gemm_w4a16_split<C>, dim3((unsigned)(tiles_m * tiles_n)), dim3(C::THREADS), C::LDS, stream, g, tiles_m,
                     tiles_n);
  return 0;
}

}  // namespace

// Times from problems of a quarter of a round to eight rounds at K = 1024 and 5120.
static const MxTime kTimes[] = {
    {1, 256, 256, 3500, 4400, 5880, 5580}, {5, 128, 256, 2700, 2750, 3575, 3190}, {6, 256, 128, 2700, 3000, 3510, 3040},
    {2, 128, 128, 2700, 900, 1940, 1750},   {3, 64, 128, 2700, 700, 1380, 1090},   {7, 128, 64, 2700, 700, 1220, 1150},
    {4, 64, 64, 2300, 900, 1000, 681},      {8, 32, 64, 1800, 1200, 780, 836}};

int choose_gemm_w4a16(const Mx4Gemm& g) {
  if (mx_rows_fit(true, g.M, g.N, g.ldb)) return kMxRows;
  const int cus = cu_count();
  return tiles_fit(g, 2) ? fastest_tile(kTimes, sizeof(kTimes) / sizeof(kTimes[0]), true, g, cus > 0 ? cus : 256) : 0;
}

int launch_gemm_w4a16(const Mx4Gemm& g, int variant, hipStream_t stream) {
  if (variant < 0) variant = choose_gemm_w4a16(g);
  if (variant == kMxRows && mx_rows_can(g.M, g.ldb)) return launch_gemm_w4a16_rows(g, stream);
  if (!tiles_fit(g, 2)) variant = 0;
  switch (variant) {
    case 1: return launch_tile<W4Tile<256, 256, 2, 2, 3, 1>>(g, stream);
    case 2: return launch_tile<W4Tile<128, 128, 2, 2, 3, 2>>(g, stream);
    case 3: return launch_tile<W4Tile<64, 128, 2, 2, 4, 2>>(g, stream);
    case 4: return launch_tile<W4Tile<64, 64, 2, 2, 4, 2>>(g, stream);
    case 5: return launch_tile<W4Tile<128, 256, 2, 2, 4, 1>>(g, stream);
    case 6: return launch_tile<W4Tile<256, 128, 2, 2, 4, 1>>(g, stream);
    case 7: return launch_tile<W4Tile<128, 64, 2, 2, 4, 2>>(g, stream);
    case 8: return launch_split<W4Split<32, 64, 4>>(g, stream);
  }
  const dim3 grid((unsigned)((g.N + 127) / 128), (unsigned)std::min((g.M + 31) / 32, 65535));
  hipLaunchKernelGGL(gemm_w4a16_direct, grid, dim3(256), 0, stream, g);
  return 0;
}

}  // namespace cdit
