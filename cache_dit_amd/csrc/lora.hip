// Low-rank adapters of many requests beside a shared projection (include/cdit_hip.h, cdit_lora_add):
//
//   t[m] = x[m] down[i]^T            i = ids[m], the adapter of row m; down[i] [R, K]
//   out[m] = base[m] + s[i] t[m] up[i]^T      up[i] [N, R]; rows without an adapter: base[m]
//
// Bound by HBM: x, base and the adapters in use are read once and out is written once; 2 M R (K + N) operations are few. Two
// kernels: the first multiplies tiles of rows by down and leaves t (fp32, a part for each of the pieces K is cut into, where rows
// alone are too few to fill the chip); the second adds the parts in their order, multiplies by up and adds to base. Rows need no
// order: a tile is multiplied by every adapter that its rows name, and each row keeps what its own gave. Rows of one request next to
// one another make tiles of one adapter; a tile of single tokens reads each of their adapters, which it has to.
//
// us, first and second product, the median of a kernel trace's passes (their fastest): one row, 5120 x 13824, rank 16: 4.5 (4.2) and 5.5
// (4.4), a launch and a step's latency each; 64 rows, 5120 x 5120, 24 adapters up to rank 64: 9.7 (8.0) and 11.2 (10.5), 9 MB of adapters
// each at 1 TB/s, reads that wait for one another: ids, ranks, x and down; ids, ranks, the parts of t; 16384 x 2560 x 10240, rank 32,
// GELU: 33 (24) and 158 (140), 671 MB at 4.2 TB/s (4.8); codes, 32760 x 5120 x 5120, ranks 128 and 64: 81 (67) and 190 (166), of which the
// second moves 671 MB at 3.5 TB/s (4.0).
//
// Sums are held in fp32. t enters the second product as the sum of two bf16 numbers: the upper 16 bits of the fp32 number and,
// rounded to bf16, what they leave out: 2^-16 of t. A single bf16 (2^-9) would cost as much as out's own rounding again.
#include <algorithm>

#include "gemm_common.h"
#include "mxfp4_device.h"
#include "quant_device.h"

namespace cdit {
namespace {

typedef cdit_lora_args Args;

constexpr int kStep = 64;  // k of a wavefront's step: 16 in a row for each lane, two matrix instructions

__device__ __forceinline__ int clamp8(int64_t n) { return n < 0 ? 0 : n > 8 ? 8 : (int)n; }
__device__ __forceinline__ int id_of(const Args& a, int64_t row) {
  if (row >= a.M) return -1;
  const int64_t at = a.rows_per_id == 1 ? row : (int64_t)((uint32_t)row / (uint32_t)a.rows_per_id);  // (M has 31 bits)
  const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[at] : (int64_t) static_cast<const int32_t*>(a.ids)[at];
  return id >= 0 && id < a.adapters ? (int)id : -1;
}
__device__ __forceinline__ int rank_of(const Args& a, int id) { return a.rank ? min(max(a.rank[id], 0), a.R) : a.R; }

// 16 bytes that start anywhere; and without the first `bytes` of them (0 to 15, the same for all lanes), zeros behind.
typedef mx_v4u Loose __attribute__((aligned(1)));
__device__ __forceinline__ v4u loose16(const void* p) { return *static_cast<const Loose*>(p); }
__device__ __forceinline__ v4u without_first(const v4u& v, int bytes) {
  uint32_t moved[5] = {v[0], v[1], v[2], v[3], 0};
#pragma unroll
  for (int step = 2; step >= 1; step /= 2)
    if (bytes / 4 & step) {
#pragma unroll
      for (int j = 0; j < 4; ++j) moved[j] = j + step < 4 ? moved[j + step] : 0u;
    }
  v4u out;
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = (uint32_t)((moved[j] | (uint64_t)moved[j + 1] << 32) >> (8 * (bytes & 3)));
  return out;
}

// What a lane of group g has of 64 k of a row: two operands of 8. Of bf16 elements 8 g to 8 g + 7 of each half, so that the four lanes
// of a row read 64 bytes next to one another (beside FP8, whose 16 bytes are 16 elements in a row, SIDE: 16 g to 16 g + 15).
template <bool FP8, bool ANY, bool SIDE = false>
struct Chunk {
  static constexpr int kWords = FP8 ? 4 : 8, XS = FP8 ? 1 : 2, kPieces = FP8 ? 1 : 2, kIn = 16 / XS;  // pieces of 16 bytes, kIn elements
  uint32_t w[kWords];
  static __device__ __forceinline__ int place(int piece, int g) { return FP8 || SIDE ? 16 * g + 8 * piece : 32 * piece + 8 * g; }
  __device__ __forceinline__ void load(const uint8_t* base, uint32_t at, int g) {  // base: the same for all lanes
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint8_t* const from = base + (at + place(i, g) * XS);
      const v4u v = ANY ? loose16(from) : *reinterpret_cast<const v4u*>(from);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
    }
  }
  // The same of a row of K that ends in these 64 k (k the first of them); what is behind it is zeros. A piece that the row ends in is
  // the row's last 16 bytes, moved up: by as many for all lanes. (Element by element, each behind its condition, waits 16 times:
  // 1357 rows of 2203 31 us in place of 11.)
  __device__ __forceinline__ void load_end(const uint8_t* base, uint32_t row_at, int k, int K, int g) {
    const uint8_t* const row = base + row_at;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int at = k + place(i, g);
      if (K < kIn) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * i + j] = 0;
#pragma unroll
        for (int e = 0; e < kIn; ++e)
          if (at + e < K)
            w[4 * i + e * XS / 4] |= (FP8 ? (uint32_t)row[at + e] : (uint32_t) reinterpret_cast<const uint16_t*>(row)[at + e]) << (8 * (e * XS % 4));
        continue;
      }
      const bool all = at + kIn <= K, some = at < K;
      const v4u v = loose16(row + (all ? at : K - kIn) * XS), part = without_first(v, (kIn - K % kIn) % kIn * XS);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = all ? v[j] : some ? part[j] : 0u;
    }
  }
  __device__ __forceinline__ v8bf half(int h) const {
    if constexpr (FP8)
      return e4m3x8_to_bf16(w[2 * h], w[2 * h + 1]);
    else
      return __builtin_bit_cast(v8bf, v4u{w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]});
  }
};

// A wavefront's view of 64 rows: lane l has row l's adapter, -1 for none, -2 for a row that does not exist.
__device__ __forceinline__ int row_id(const Args& a, int64_t row0) {
  const int64_t row = row0 + (threadIdx.x & 63);
  return row < a.M ? id_of(a, row) : -2;
}
// Rows of one adapter, wherever among 64 they are, 16 at a time: every slots-th such group, f(id, rows, first row's place in the list,
// how many). `list` (64 numbers of the wavefront's own in LDS) gets the rows in their order. The same in every wavefront.
template <class F>
__device__ __forceinline__ void for_groups(int mine, bool without, int slots, int slot, int* list, F f) {
  const int lane = threadIdx.x & 63;
  int index = 0;
  for (uint64_t pending = __ballot(without ? mine > -2 : mine > -1); pending;) {
    const int id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(pending));
    const uint64_t members = __ballot(mine == id);
    pending &= ~members;
    const int count = __builtin_popcountll(members), groups = (count + 15) / 16;
    int mine_next = slot >= index ? slot - index : slot - index + slots;  // groups of this adapter before one of this slot's
    index = (index + groups) % slots;
    if (mine_next >= groups) continue;
    if ((members >> lane) & 1) list[__builtin_popcountll(members & (((uint64_t)1 << lane) - 1))] = lane;
    for (; mine_next < groups; mine_next += slots) f(id, 16 * mine_next, min(count - 16 * mine_next, 16));
  }
}

// t of few rows: of 64, the rows of one adapter, 16 at a time, and, for each group of four wavefronts, 16 RT ranks; the four take
// every fourth step of the workgroup's piece of K and add up through LDS. A step's loads take a microsecond to come: an adapter's rows
// are read once for 64 rows, and K, ranks and adapters (slots) spread over all CUs, so that few steps follow one another.
// grid: 64 rows, pieces of K times slots, ranks.
template <bool FP8, bool ANY, int RT>
__global__ __launch_bounds__(512, RT == 4 ? 3 : 4) void lora_down(Args a, float* t, int steps_per_piece, int slots) {
  extern __shared__ v4f exchange[];  // [groups][2][RT][64]
  __shared__ int lists[8][64];
  constexpr int XS = FP8 ? 1 : 2;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, kw = wave & 3, rw = wave >> 2;
  const int64_t row0 = (int64_t)blockIdx.x * 64;
  const int r0 = (int)(blockIdx.z * (blockDim.x >> 8) + rw) * (16 * RT);
  const int piece = (int)blockIdx.y / slots, slot = (int)blockIdx.y % slots;
  // this wavefront's steps: first, first + 4, ... below last, all whole ones; and one that K ends in
  const int first = piece * steps_per_piece + kw, whole = (int)(a.K / kStep), last = min(whole, (piece + 1) * steps_per_piece);
  const bool ragged = a.K % kStep != 0 && whole >= first && whole < (piece + 1) * steps_per_piece && (whole - first) % 4 == 0;

  const uint8_t* const x_base = static_cast<const uint8_t*>(a.x) + row0 * a.ld_x * XS;

  for_groups(row_id(a, row0), false, slots, slot, lists[wave], [&](int id, int from, int count) {
    // (the compiler would keep all offsets that no adapter changes from one to the next: more than there are registers)
    int lane_now = lane;
    asm volatile("" : "+v"(lane_now));
    const int i16 = lane_now & 15, g = lane_now >> 4;
    const bool active = r0 < rank_of(a, id);
    const int row = lists[wave][from + min(i16, count - 1)];
    v4f acc[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[r] = v4f{0, 0, 0, 0};
    if (active) {
      typedef Chunk<FP8, ANY> X;
      typedef Chunk<false, ANY, FP8> W;
      const uint8_t* const w_base = static_cast<const uint8_t*>(a.down) + (int64_t)id * a.R * a.K * 2;
      const uint32_t x_at = (uint32_t)row * (uint32_t)a.ld_x * XS;
      uint32_t w_at[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) w_at[r] = (uint32_t)min(r0 + 16 * r + i16, a.R - 1) * (uint32_t)a.K * 2;
      auto load = [&](int s, X& x, W(&w)[RT]) {
        const uint32_t k = (uint32_t)s * kStep;
#pragma unroll
        for (int r = 0; r < RT; ++r) w[r].load(w_base, w_at[r] + 2 * k, g);
        x.load(x_base, x_at + XS * k, g);
      };
      auto multiply = [&](const X& x, const W(&w)[RT]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const v8bf b = x.half(h);
#pragma unroll
          for (int r = 0; r < RT; ++r) acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[r].half(h), b, acc[r], 0, 0, 0);
        }
      };
      if (first < last) {
        X x[2];
        W w[2][RT];
        load(first, x[0], w[0]);
        for (int s = first;;) {
          if (s + 4 < last) load(s + 4, x[1], w[1]);
          multiply(x[0], w[0]);
          s += 4;
          if (s >= last) break;
          if (s + 4 < last) load(s + 4, x[0], w[0]);
          multiply(x[1], w[1]);
          s += 4;
          if (s >= last) break;
        }
      }
      if (ragged) {
        X x;
        x.load_end(x_base, x_at, whole * kStep, (int)a.K, g);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          W w;
          w.load_end(w_base, w_at[r], whole * kStep, (int)a.K, g);
#pragma unroll
          for (int h = 0; h < 2; ++h) acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.half(h), x.half(h), acc[r], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);  // (not all at once: that takes 220 registers, or scratch, which takes 60 us)
        }
      }
    }
    // (3 -> 1, 2 -> 0), then 1 -> 0: a fixed order
    v4f* const place = exchange + (size_t)rw * 2 * RT * 64;
    auto put = [&](int which) {
#pragma unroll
      for (int r = 0; r < RT; ++r) place[(which * RT + r) * 64 + lane] = acc[r];
    };
    auto take = [&](int which) {
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[r] += place[(which * RT + r) * 64 + lane];
    };
    if (active && kw >= 2) put(kw - 2);
    __syncthreads();
    if (active && kw < 2) take(kw);
    __syncthreads();
    if (active && kw == 1) put(0);
    __syncthreads();
    if (active && kw == 0) {
      take(0);
      if (i16 < count) {
        float* const to = t + ((int64_t)piece * a.M + row0 + row) * a.R + r0 + 4 * g;
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if (r0 + 16 * r < a.R) *reinterpret_cast<v4f*>(to + 16 * r) = acc[r];
      }
    }
    __syncthreads();
  });
}

// A tile of 64 rows in the second product: its adapters, and its t (parts added, times the adapter's and the row's scale, in two bf16
// numbers) in LDS.
struct Tile {
  int id[64], rank[64];
  uint64_t members[64];
  int row_rank[64];
  float row_factor[64];
  // the 32-rank pieces of all adapters: adapter * 8 + piece (256 ranks are 8)
  int parts;
  uint16_t part[64 * 8];
};
// x as the sum of two bf16 numbers: its upper half, and, in fp32, what that leaves out.
__device__ __forceinline__ void split(float x, uint32_t* hi, float* lo) {
  const uint32_t u = __float_as_uint(x) & 0xffff0000u;
  // an infinity or NaN leaves nothing; a NaN whose bits are all below stays one
  *hi = x != x ? u >> 16 | 0x40u : u >> 16;
  *lo = (u & 0x7f800000u) != 0x7f800000u ? x - __uint_as_float(u) : 0.0f;
}
__device__ __forceinline__ void split4(const v4f& x, uint16_t* upper, uint16_t* lower) {
  uint32_t hi[4];
  float lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(x[i], &hi[i], &lo[i]);
  *reinterpret_cast<v2u*>(upper) = v2u{hi[0] | hi[1] << 16, hi[2] | hi[3] << 16};
  *reinterpret_cast<v2u*>(lower) = v2u{pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3])};
}
// The 8 places behind a row's R ranks, which are what an operand of 32 ranks finds where R ends in its middle. Zeros: up's operand is
// cut to zeros there as well, but zero times an infinity of another rank would be a NaN.
__device__ __forceinline__ void clear_behind(const Args& a, int rows, uint16_t* upper, uint16_t* lower) {
  const int m = (int)threadIdx.x % rows;
  if ((int)threadIdx.x < 2 * rows) *reinterpret_cast<v4u*>(((int)threadIdx.x < rows ? upper : lower) + m * (a.R + 8) + a.R) = v4u{0, 0, 0, 0};
}
__device__ __forceinline__ int stage_t(const Args& a, const float* t, int pieces, int64_t row0, int rows, Tile& tile, uint16_t* upper,
                                       uint16_t* lower) {
  const int lane = threadIdx.x & 63, ld = a.R + 8;
  const int mine = lane < rows ? id_of(a, row0 + lane) : -1;
  const int rank = mine >= 0 ? rank_of(a, mine) : 0;
  if (threadIdx.x < 64) {
    tile.row_rank[lane] = rank;
    tile.row_factor[lane] = mine < 0 ? 0.0f : (a.scale ? a.scale[mine] : 1.0f) * (a.x_scale ? a.x_scale[row0 + lane] : 1.0f);
  }
  int count = 0;
  for (uint64_t pending = __ballot(mine >= 0); pending; ++count) {
    const int leader = __builtin_ctzll(pending), id = __builtin_amdgcn_readlane(mine, leader);
    const uint64_t members = __ballot(mine == id);
    pending &= ~members;
    if (threadIdx.x == 0) {
      tile.id[count] = id;
      tile.rank[count] = __builtin_amdgcn_readlane(rank, leader);
      tile.members[count] = members;
    }
  }
  __syncthreads();
  if (threadIdx.x < 64 && threadIdx.x < count) {
    int at = 0, here = 0;
    for (int j = 0; j <= (int)threadIdx.x; ++j) {
      at += here;
      here = (tile.rank[j] + 31) / 32;
    }
    for (int k = 0; k < here; ++k) tile.part[at + k] = (uint16_t)(8 * threadIdx.x + k);
    if ((int)threadIdx.x == count - 1) tile.parts = at + here;
  }
  if (threadIdx.x == 0 && count == 0) tile.parts = 0;
  clear_behind(a, 64, upper, lower);
  // quads of a row are a multiple of 4: 16 threads of a wavefront and more are in one row, or rows next to one another
  const int quads = a.R / 4, all = 64 * quads;
  constexpr int kBatch = 4;
  for (int q0 = threadIdx.x; q0 < all; q0 += 256 * kBatch) {
    v4f v[kBatch];
    int m[kBatch], r[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int q = min(q0 + 256 * i, all - 1);
      m[i] = (int)((uint32_t)q / (uint32_t)quads);
      r[i] = 4 * (q - m[i] * quads);
      v[i] = v4f{0, 0, 0, 0};
      if (r[i] < tile.row_rank[m[i]]) v[i] = *reinterpret_cast<const v4f*>(t + (row0 + m[i]) * a.R + r[i]);
    }
    for (int s = 1; s < pieces; ++s)
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (r[i] < tile.row_rank[m[i]]) v[i] += *reinterpret_cast<const v4f*>(t + (s * a.M + row0 + m[i]) * a.R + r[i]);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (q0 + 256 * i >= all) break;
      const int have = tile.row_rank[m[i]] - r[i];
      const float f = tile.row_factor[m[i]];
      v4f x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = e < have ? v[i][e] * f : 0.0f;
      split4(x, upper + m[i] * ld + r[i], lower + m[i] * ld + r[i]);
    }
  }
  __syncthreads();
  return count;
}
// up for the 32 columns from n0 and the 32 ranks from k on, as two operands. Row i of an instruction's tile h is column 8 (i / 4) +
// 4 h + i % 4: a lane's results are 8 columns in a row.
__device__ __forceinline__ void load_up(const Args& a, int64_t n0, int id, int k, v4u (&w)[2]) {
  const int i16 = threadIdx.x & 15, r = k + 8 * (threadIdx.x >> 4 & 3);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t col = min(n0 + 8 * (i16 >> 2) + 4 * h + (i16 & 3), a.N - 1);
    w[h] = *reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(a.up) + ((int64_t)id * a.N + col) * a.R + min(r, a.R - 8));
  }
}
// Nothing of what lies behind the rank.
__device__ __forceinline__ void cut_up(int rank, int k, v4u (&w)[2]) {
  const int r = k + 8 * (threadIdx.x >> 4 & 3);
  if (r + 8 <= rank) return;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (r + i >= rank) w[h][i / 2] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
}
// have <= 8 columns of a row of base.
template <bool ANY>
__device__ __forceinline__ Mx8<CDIT_DT_BF16> load_base(const uint16_t* p, int have) {
  Mx8<CDIT_DT_BF16> b = {};
  if (have == 8) b = mx_load8<CDIT_DT_BF16, false, ANY>(p);
  if (!ANY || have == 8) return b;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < have) b.w[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
  return b;
}
__device__ __forceinline__ Mx8<CDIT_DT_BF16> sum_of(bool gelu, const Mx8<CDIT_DT_BF16>& b, const float (&add)[8]) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = (i & 1 ? bf16_hi(b.w[i / 2]) : bf16_lo(b.w[i / 2])) + add[i];
    if (gelu) y[i] = gelu_tanh(y[i]);
  }
  Mx8<CDIT_DT_BF16> v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.w[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
  return v;
}
template <bool ANY>
__device__ __forceinline__ void store_out(uint16_t* p, int have, const Mx8<CDIT_DT_BF16>& v) {
  if (have == 8) {
    mx_store8<CDIT_DT_BF16, false, ANY>(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < have) p[i] = (uint16_t)(v.w[i / 2] >> (16 * (i & 1)));
}

// base + t up^T for few rows: of 64, the rows of one adapter, or of none, 16 at a time, and `columns` columns; a wavefront takes 32
// columns at a time. grid: 64 rows, column pieces, slots.
template <bool ANY>
__global__ __launch_bounds__(256) void lora_up(Args a, const float* t, int pieces, int columns) {
  extern __shared__ uint16_t parts[];  // t's upper and lower halves [2][16][R + 8]
  __shared__ int lists[4][64];
  constexpr int kAhead = 4;
  const int ld = a.R + 8, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint16_t *const upper = parts, *const lower = parts + 16 * ld;
  const int64_t row0 = (int64_t)blockIdx.x * 64, begin = (int64_t)blockIdx.y * columns + 32 * wave;
  const int64_t end = min(a.N, ((int64_t)blockIdx.y + 1) * columns);
  const bool gelu = a.epilogue & CDIT_EPI_GELU_TANH;
  for_groups(row_id(a, row0), true, (int)gridDim.z, (int)blockIdx.z, lists[wave], [&](int id, int from, int count) {
    int lane = threadIdx.x & 63;  // (as in lora_down)
    asm volatile("" : "+v"(lane));
    const int i16 = lane & 15, g = lane >> 4;
    const int64_t row = row0 + lists[wave][from + min(i16, count - 1)];
    const uint16_t* const base = static_cast<const uint16_t*>(a.base) + row * a.ld_base;
    const int rank = id < 0 ? 0 : rank_of(a, id), steps = (rank + 31) / 32;
    auto fetch = [&](int64_t n0) { return load_base<ANY>(base + n0 + 8 * g, n0 + 8 * g < a.N ? clamp8(a.N - n0 - 8 * g) : 0); };
    auto finish = [&](int64_t n0, const Mx8<CDIT_DT_BF16>& b, const v4f(&acc)[2]) {
      const int64_t n = n0 + 8 * g;
      if (i16 >= count || n >= a.N) return;
      const float add[8] = {acc[0][0], acc[0][1], acc[0][2], acc[0][3], acc[1][0], acc[1][1], acc[1][2], acc[1][3]};
      store_out<ANY>(static_cast<uint16_t*>(a.out) + row * a.ld_out + n, clamp8(a.N - n), sum_of(gelu, b, add));
    };
    Mx8<CDIT_DT_BF16> next = {};
    if (begin < end) next = fetch(begin);
    // pieces of 32 columns and 32 ranks, one after the other, kAhead of them under way
    v4u w[kAhead][2];
    int64_t load_n = begin;
    int load_k = 0;
    auto load = [&](v4u(&to)[2]) {
      load_up(a, load_n, id, 32 * load_k, to);
      if (++load_k < steps) return;
      load_k = 0;
      load_n = load_n + 128 < end ? load_n + 128 : load_n;  // (behind the last one: that again)
    };
    if (steps > 0 && begin < end) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) load(w[i]);
    }
    if (steps > 0) {
      clear_behind(a, 16, upper, lower);
      const int quads = a.R / 4;
      for (int q = threadIdx.x; q < 16 * quads; q += 256) {
        const int m = (int)((uint32_t)q / (uint32_t)quads), r = 4 * (q - m * quads);
        v4f v = {0, 0, 0, 0};
        if (m < count && r < rank) {
          const int64_t at = row0 + lists[wave][from + m];
          const float f = (a.scale ? a.scale[id] : 1.0f) * (a.x_scale ? a.x_scale[at] : 1.0f);
          const float* const p = t + at * a.R + r;
          const int64_t next_piece = a.M * a.R;
          v = *reinterpret_cast<const v4f*>(p);
          int s = 1;
          for (; s < pieces; s += 8) {  // eight on their way at a time
            v4f u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = *reinterpret_cast<const v4f*>(p + min(s + i, pieces - 1) * next_piece);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (s + i < pieces) v += u[i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = r + i < rank ? v[i] * f : 0.0f;
        }
        split4(v, upper + m * ld + r, lower + m * ld + r);
      }
      __syncthreads();
    }
    if (steps == 0) {
      const v4f none[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      for (int64_t n0 = begin; n0 < end; n0 += 128) {
        const Mx8<CDIT_DT_BF16> b = next;
        if (n0 + 128 < end) next = fetch(n0 + 128);
        finish(n0, b, none);
      }
      return;
    }
    v4f acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    int64_t n0 = begin;
    int k = 0;
    while (n0 < end) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (n0 >= end) break;
        cut_up(rank, 32 * k, w[i]);
        const int at = i16 * ld + min(32 * k + 8 * g, a.R);  // (behind R: zeros)
        const v8bf hi = *reinterpret_cast<const v8bf*>(upper + at), lo = *reinterpret_cast<const v8bf*>(lower + at);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[i][h]), hi, acc[h], 0, 0, 0);
          acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[i][h]), lo, acc[h], 0, 0, 0);
        }
        load(w[i]);
        if (++k < steps) continue;
        const Mx8<CDIT_DT_BF16> b = next;
        if (n0 + 128 < end) next = fetch(n0 + 128);
        finish(n0, b, acc);
        acc[0] = acc[1] = v4f{0, 0, 0, 0};
        n0 += 128;
        k = 0;
      }
    }
    __syncthreads();  // (t's place is free for the next rows')
  });
}

// The same for 64 rows: each wavefront multiplies 64 rows by 32 of the workgroup's 128 columns, and adds 16 rows of all 128 to base;
// between the two the sums change hands in LDS, and memory is read and written in 256 bytes of a row (64 bytes, as the instruction
// leaves them, cost 15 % of the rate). t stays in registers (KS pieces of 32 ranks; beyond 128 one workgroup a CU has
// them); the next columns' base and up are under
// way meanwhile, loaded without branches, which would make the compiler wait for all of them: what does not exist is read where
// something does, and not used.
template <bool ANY, int KS>
__global__ __launch_bounds__(256, KS <= 4 ? 2 : 1) void lora_up_rows(Args a, const float* t, int pieces, int columns, int tiles_per_id, int64_t rows_per_id) {
  extern __shared__ uint16_t parts[];  // t's upper and lower halves [2][64][R + 8]
  __shared__ Tile tile;
  // sums [64][128] in quads: quad q of a row at place q / 2 + 16 (q & 1), its lower four bits turned by the row's
  __shared__ v4f sums[64][32];
  uint16_t *const upper = parts, *const lower = parts + 64 * (a.R + 8);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int64_t request = (int64_t)blockIdx.x / tiles_per_id * rows_per_id, row0 = request + (int64_t)(blockIdx.x % tiles_per_id) * 64;
  const int64_t rows_left = min(request + rows_per_id, a.M) - row0;
  if (rows_left <= 0) return;  // (the last request's rows may be fewer)
  const int rows = rows_left < 64 ? (int)rows_left : 64;
  const int count = stage_t(a, t, pieces, row0, rows, tile, upper, lower);
  const bool gelu = a.epilogue & CDIT_EPI_GELU_TANH;
  const int64_t begin = (int64_t)blockIdx.y * columns, end = min(a.N, begin + columns);

  // base and out: rows 16 wave + 4 j + g, columns n0 + 8 i16. Aligned (out_aligned) as buffers, whose rows end with the
  // tile's: what lies behind is zeros, and not stored. All of an offset is in its vector register, here and wherever this file reads
  // or writes through a buffer: that is what is compared with the buffer's size. A scalar offset is taken off the size first, and
  // the rows of a short tile, or the columns behind N, can lie further than the size is: nothing here depends on what a difference
  // below zero means.
  auto buffer = [&](const void* p, int64_t ld) -> __amdgpu_buffer_rsrc_t {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(static_cast<const uint16_t*>(p) + row0 * ld), 0,
                                             (int)(((rows - 1) * ld + a.N) * 2), 0x00020000);
  };
  // Rows that start anywhere (ANY) by address, 8 columns at a time all the same: where a row ends among them its last 8 are read and
  // moved, when they are needed. N is 8 or more.
  const uint32_t base_at = ANY ? 0 : (uint32_t)(((16 * wave + g) * a.ld_base + 8 * i16) * 2);
  const uint32_t out_at = ANY ? 0 : (uint32_t)(((16 * wave + g) * a.ld_out + 8 * i16) * 2);
  auto fetch = [&](int64_t n0, Mx8<CDIT_DT_BF16>(&b)[4]) {
    if constexpr (ANY) {
      const uint16_t* const from = static_cast<const uint16_t*>(a.base) + row0 * a.ld_base;
      const uint32_t n = (uint32_t)min((int)n0 + 8 * i16, (int)a.N - 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v4u v = loose16(from + ((uint32_t)min(16 * wave + 4 * j + g, rows - 1) * (uint32_t)a.ld_base + n));
#pragma unroll
        for (int i = 0; i < 4; ++i) b[j].w[i] = v[i];
      }
    } else {
      const __amdgpu_buffer_rsrc_t from = buffer(a.base, a.ld_base);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v4u v = __builtin_bit_cast(
            v4u, __builtin_amdgcn_raw_buffer_load_b128(from, (int)(base_at + (uint32_t)(n0 * 2 + 8 * j * a.ld_base)), 0, 0));
#pragma unroll
        for (int i = 0; i < 4; ++i) b[j].w[i] = v[i];
      }
    }
  };
  auto finish = [&](int64_t n0, const v4f(&acc)[4][2], const Mx8<CDIT_DT_BF16>(&b)[4]) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) sums[16 * m + i16][((4 * wave + g) ^ i16) + 16 * h] = acc[m][h];
    __syncthreads();
    const int64_t n = n0 + 8 * i16;
    const int have = clamp8(a.N - n);
    const bool ends = ANY && n0 + 128 > a.N && a.N % 8 != 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 16 * wave + 4 * j + g;
      const v4f lo = sums[r][i16 ^ (r & 15)], hi = sums[r][(i16 ^ (r & 15)) + 16];
      const float add[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      Mx8<CDIT_DT_BF16> old = b[j];
      if (ends) {
        const v4u part = without_first(v4u{old.w[0], old.w[1], old.w[2], old.w[3]}, (int)(8 - a.N % 8) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) old.w[i] = have < 8 ? part[i] : old.w[i];
      }
      const Mx8<CDIT_DT_BF16> y = sum_of(gelu, old, add);
      if constexpr (ANY) {
        uint16_t* const to = static_cast<uint16_t*>(a.out) + row0 * a.ld_out;
        if (r < rows && have > 0) store_out<true>(to + ((uint32_t)r * (uint32_t)a.ld_out + (uint32_t)n), have, y);
      } else {
        const v4u v = {y.w[0], y.w[1], y.w[2], y.w[3]};
        // (With a scalar offset the compiler also holds the store to have read its data when it is issued and lets the next
        // instruction write the first of these registers, which has reached memory: lanes 12 to 15 of each 16, where several
        // workgroups share a CU.)
        const uint32_t at = out_at + (uint32_t)(n0 * 2 + 8 * j * a.ld_out);
        __builtin_amdgcn_raw_buffer_store_b128(v, buffer(a.out, a.ld_out), (int)(have > 0 ? at : 0x80000000u), 0, 0);
      }
    }
    __syncthreads();
  };
  Mx8<CDIT_DT_BF16> next[4];
  fetch(begin, next);
  if (count != 1) {
    // Any number of adapters: one piece of 32 ranks after the other, whichever adapter's it is, and each row takes its own's. The sum
    // goes through the instructions as in a tile of one adapter: a row's result has the same bits whatever the rows beside it name.
    // kAhead pieces are under way, the next columns' among them.
    constexpr int kAhead = 4;
    const int pieces_of_up = __builtin_amdgcn_readfirstlane(tile.parts);
    v4f acc[4][2];
    auto clear = [&]() {
#pragma unroll
      for (int m = 0; m < 4; ++m) acc[m][0] = acc[m][1] = v4f{0, 0, 0, 0};
    };
    auto columns_done = [&](int64_t n0) {
      Mx8<CDIT_DT_BF16> b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = next[j];
      fetch(n0 + 128 < end ? n0 + 128 : begin, next);
      finish(n0, acc, b);
      clear();
    };
    clear();
    if (pieces_of_up == 0) {
      for (int64_t n0 = begin; n0 < end; n0 += 128) columns_done(n0);
      return;
    }
    v4u w[kAhead][2];
    int64_t load_n = begin;
    int load_e = 0;
    auto load = [&](v4u(&to)[2]) {
      const int part = __builtin_amdgcn_readfirstlane(tile.part[load_e]);
      load_up(a, load_n + 32 * wave, __builtin_amdgcn_readfirstlane(tile.id[part >> 3]), 32 * (part & 7), to);
      if (++load_e < pieces_of_up) return;
      load_e = 0;
      load_n = load_n + 128 < end ? load_n + 128 : load_n;  // (behind the last ones: those again)
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(w[i]);
    int e = 0;
    for (int64_t n0 = begin; n0 < end;) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (n0 >= end) break;
        const int part = __builtin_amdgcn_readfirstlane(tile.part[e]), j = part >> 3, k = 32 * (part & 7);
        const uint64_t members = tile.members[j];
        cut_up(__builtin_amdgcn_readfirstlane(tile.rank[j]), k, w[i]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (!(__builtin_amdgcn_readfirstlane((int)(members >> (16 * m))) & 0xffff)) continue;
          const int at = (16 * m + i16) * (a.R + 8) + min(k + 8 * g, a.R);  // (behind R: zeros)
          const v8bf hi = *reinterpret_cast<const v8bf*>(upper + at), lo = *reinterpret_cast<const v8bf*>(lower + at);
          const bool member = members >> (16 * m + i16) & 1;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            v4f d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[i][h]), hi, acc[m][h], 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[i][h]), lo, d, 0, 0, 0);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[m][h][q] = member ? d[q] : acc[m][h][q];
          }
        }
        load(w[i]);
        if (++e < pieces_of_up) continue;
        e = 0;
        columns_done(n0);
        n0 += 128;
      }
    }
    return;
  }
  const int id = __builtin_amdgcn_readfirstlane(tile.id[0]), rank = __builtin_amdgcn_readfirstlane(tile.rank[0]);
  const uint64_t members = tile.members[0];
  v8bf hi[4][KS], lo[4][KS];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int at = (16 * m + i16) * (a.R + 8) + min(32 * k + 8 * g, a.R);  // (behind R: zeros)
      hi[m][k] = *reinterpret_cast<const v8bf*>(upper + at);
      lo[m][k] = *reinterpret_cast<const v8bf*>(lower + at);
    }
  // (up's rows behind N are zeros, values behind the rank are cut)
  const uint16_t* const up = static_cast<const uint16_t*>(a.up) + (int64_t)id * a.N * a.R;
  const __amdgpu_buffer_rsrc_t up_buf =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(up), 0, (int)(a.N * a.R * 2), 0x00020000);
  const uint32_t up_at = (uint32_t)(((32 * wave + 8 * (i16 >> 2) + (i16 & 3)) * a.R + 8 * g) * 2);
  auto load = [&](int64_t n0, int k, v4u(&w)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(
                                         up_buf, (int)(up_at + (uint32_t)(((n0 + 4 * h) * a.R + (32 * k < rank ? 32 * k : 0)) * 2)), 0, 0));
  };
  // (with the addresses that ANY needs, four pieces leave no registers for two columns of base at a time)
  constexpr bool LATE = ANY && KS == 4;
  v4u w[KS][2];
#pragma unroll
  for (int k = 0; k < KS; ++k) load(begin, k, w[k]);
  for (int64_t n0 = begin; n0 < end; n0 += 128) {
    Mx8<CDIT_DT_BF16> b[4];
    const int64_t then = n0 + 128 < end ? n0 + 128 : begin;
    if constexpr (!LATE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = next[j];
      fetch(then, next);
    }
    v4f acc[4][2];
#pragma unroll
    for (int m = 0; m < 4; ++m) acc[m][0] = acc[m][1] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if (32 * k < rank) {
        if (32 * k + 32 > rank) cut_up(rank, 32 * k, w[k]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            acc[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[k][h]), hi[m][k], acc[m][h], 0, 0, 0);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            acc[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[k][h]), lo[m][k], acc[m][h], 0, 0, 0);
        }
      }
      load(then, k, w[k]);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const bool member = members >> (16 * m + i16) & 1;  // (no adapter: t is 0, but 0 times an infinity is none)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][h][i] = member ? acc[m][h][i] : 0.0f;
    }
    finish(n0, acc, LATE ? next : b);
    if constexpr (LATE) fetch(then, next);
  }
}

// t of 128 rows and 16 RT ranks, for many rows. Tiles of x and down come by DMA into a ring of STAGES steps in LDS, 128 bytes of each
// row of x a step: read into registers as the matrix instruction takes x, 64 bytes of 16 rows, memory gives 3.6 TB/s, in 128 bytes
// 5.5; and with less than four steps or so under way the wavefronts, which wait for one another at every step, wait for memory.
// us, 32760 x 5120, bf16: one step ahead in registers 98, three 93, six 66 (registers are enough for that up to 32 ranks).
// Where the rows of a request have one adapter, tiles end with the request. Elsewhere a tile has several, of which kSlots workgroups take
// each its share: one that took them one after the other would take as many times longer, and all would wait for it.
// Rows that do not start and end at 16 bytes (ANY) cannot come by DMA: they go through registers, two steps ahead, into two stages.
// K is 128 or more, offsets in a tile are below kTallBytes. grid: row tiles, pieces of K times slots, ranks.
constexpr int kSlots = 4, kTallRows = 128;
constexpr int64_t kTallBytes = (int64_t)1 << 30;
template <bool FP8, bool ANY, int RT>
struct Tall {
  static constexpr int XS = FP8 ? 1 : 2, HALVES = FP8 ? 2 : 1;  // of a step of 128 bytes of x, 64 k each
  static constexpr int STEP = 128 / XS;
  static constexpr int X_BYTES = kTallRows * 128, W_BYTES = 16 * RT * 128, STAGE = X_BYTES + HALVES * W_BYTES;
  static constexpr int STAGES = ANY ? 2 : 150 * 1024 / STAGE < 6 ? 150 * 1024 / STAGE : 6;
  static constexpr int NX = X_BYTES / 4096, NW = RT >= 2 ? RT / 2 : 1;  // DMA instructions of a wavefront (1 KB each)
  static constexpr int FLY = NX + HALVES * NW;
  static constexpr int RG = RT == 8 ? 2 : 1, MT = 2 * RG, RW = RT / RG;  // wavefronts side by side over ranks; 16-row and
                                                                        // 16-rank tiles of each
};
template <bool FP8, bool ANY, int RT>
__global__ __launch_bounds__(256) void lora_down_tall(Args a, float* t, int k_per_piece, int tiles_per_id, int64_t rows_per_id) {
  typedef Tall<FP8, ANY, RT> C;
  constexpr int MT = C::MT, RW = C::RW, RG = C::RG, S = C::STAGES;
  extern __shared__ __attribute__((aligned(1024))) uint8_t ring[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int64_t request = blockIdx.x / tiles_per_id, begin = request * rows_per_id,
                row0 = begin + (int64_t)(blockIdx.x % tiles_per_id) * kTallRows;
  const int rows = (int)min((int64_t)kTallRows, min(begin + rows_per_id, a.M) - row0);
  if (rows <= 0) return;  // (the last request's rows may be fewer)
  const int r0 = (int)blockIdx.z * (16 * RT), slot = (int)blockIdx.y % kSlots, piece = (int)blockIdx.y / kSlots;
  const int steps = (int)((a.K + C::STEP - 1) / C::STEP), first = piece * (k_per_piece / C::STEP),
            last = min(steps, first + k_per_piece / C::STEP);
  const int id0 = lane < rows ? id_of(a, row0 + lane) : -1, id1 = 64 + lane < rows ? id_of(a, row0 + 64 + lane) : -1;
  uint64_t pending0 = __ballot(id0 >= 0), pending1 = __ballot(id1 >= 0);

  // A row's 128 bytes are 8 pieces, piece p at place p ^ (row / 2 & 7): the 16 rows that a matrix instruction takes at once lie in
  // different banks. DMA instruction n writes rows 8 n to 8 n + 7, lane by lane.
  const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  const uint32_t x_ld = (uint32_t)a.ld_x * C::XS, x_end = (uint32_t)a.K * C::XS, w_ld = (uint32_t)a.K * 2;
  uint32_t x_at[C::NX], w_at[C::NW];
#pragma unroll
  for (int n = 0; n < C::NX; ++n) {
    const int row = 8 * (wave + 4 * n) + (lane >> 3);
    x_at[n] = ANY ? (uint32_t)min(row, rows - 1) * x_ld : (uint32_t)row * x_ld + 16 * chunk;
  }
  // (16 ranks are two instructions: wavefronts 2 and 3 write what 0 and 1 do)
  auto w_block = [&](int n) { return RT == 1 ? wave & 1 : wave + 4 * n; };
#pragma unroll
  for (int n = 0; n < C::NW; ++n) {
    const int r = 8 * w_block(n) + (lane >> 3);
    w_at[n] = ANY ? (uint32_t)min(r, a.R - r0 - 1) * w_ld : (uint32_t)r * w_ld + 16 * chunk;
  }
  // (rows that do not exist lie behind the buffer's end: zeros. By address they are the last one's, and their t is not kept)
  const uint8_t* const x_base = static_cast<const uint8_t*>(a.x) + row0 * a.ld_x * C::XS;
  const __amdgpu_buffer_rsrc_t x_buf =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(x_base), 0, (int)((rows - 1) * x_ld + x_end), 0x00020000);

  for (int index = 0; pending0 | pending1; ++index) {  // the same in every wavefront
    const int id = pending0 ? __builtin_amdgcn_readlane(id0, __builtin_ctzll(pending0))
                            : __builtin_amdgcn_readlane(id1, __builtin_ctzll(pending1));
    const uint64_t members0 = __ballot(id0 == id), members1 = __ballot(id1 == id);
    pending0 &= ~members0;
    pending1 &= ~members1;
    const int rank = __builtin_amdgcn_readfirstlane(rank_of(a, id));
    if (index % kSlots != slot || r0 >= rank) continue;
    const uint8_t* const w_base = static_cast<const uint8_t*>(a.down) + ((int64_t)id * a.R + r0) * a.K * 2;
    const __amdgpu_buffer_rsrc_t w_buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(w_base), 0, (int)((rank - r0) * w_ld),
                                                                           0x00020000);  // (nothing behind the rank is read)
    auto issue = [&](int s, int stage) {
      const uint32_t behind = (uint32_t)s * 128 + 16 * chunk < x_end ? 0u : 0x80000000u;
#pragma unroll
      for (int n = 0; n < C::NX; ++n)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(x_buf, (__attribute__((address_space(3))) void*)(ring + stage + (wave + 4 * n) * 1024), 16,
                                                 (int)((x_at[n] + (uint32_t)s * 128) | behind), 0, 0, 0);
#pragma unroll
      for (int half = 0; half < C::HALVES; ++half) {
        const uint32_t k = (uint32_t)(s * C::HALVES + half) * 128;  // bytes; of FP8's second half behind the row's end, maybe
        const uint32_t behind = k + 16 * chunk < w_ld ? 0u : 0x80000000u;
#pragma unroll
        for (int n = 0; n < C::NW; ++n)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              w_buf, (__attribute__((address_space(3))) void*)(ring + stage + C::X_BYTES + half * C::W_BYTES + w_block(n) * 1024), 16,
              (int)((w_at[n] + k) | behind), 0, 0, 0);
      }
    };
    v4f acc[MT][RW];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < RW; ++r) acc[m][r] = v4f{0, 0, 0, 0};
    const uint32_t x_read = (uint32_t)((wave / RG) * (16 * MT) + i16) * 128, w_read = (uint32_t)((wave % RG) * (16 * RW) + i16) * 128;
    const int bank = i16 >> 1 & 7;
    auto read = [](const uint8_t* __restrict__ st, uint32_t at) -> v4u { return *reinterpret_cast<const v4u*>(st + at); };
    auto multiply = [&](int stage) {
#pragma unroll
      for (int half = 0; half < C::HALVES; ++half) {
        v4u x[MT][FP8 ? 1 : 2], w[2][RW];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < (FP8 ? 1 : 2); ++h)
            x[m][h] = read(ring, stage + x_read + m * 2048 + (((FP8 ? 4 * half + g : 2 * g + h) ^ bank) << 4));
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < RW; ++r)
            w[h][r] = read(ring, stage + C::X_BYTES + half * C::W_BYTES + w_read + r * 2048 + (((2 * g + h) ^ bank) << 4));
        __builtin_amdgcn_sched_barrier(0);  // (all reads under way before the first product waits for its own)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            v8bf b;
            if constexpr (FP8)
              b = e4m3x8_to_bf16(x[m][0][2 * h], x[m][0][2 * h + 1]);
            else
              b = __builtin_bit_cast(v8bf, x[m][h]);
#pragma unroll
            for (int r = 0; r < RW; ++r)
              acc[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[h][r]), b, acc[m][r], 0, 0, 0);
          }
      }
    };
    __syncthreads();  // (the ring is free: an adapter before this one may still be read)
    if constexpr (ANY) {
      struct Held {
        v4u x[C::NX], w[C::HALVES][C::NW];
      };
      auto load = [&](int s, Held& h) {
        const uint32_t in_x = min((uint32_t)s * 128 + 16 * chunk, x_end - 16);
#pragma unroll
        for (int n = 0; n < C::NX; ++n) h.x[n] = loose16(x_base + (x_at[n] + in_x));
#pragma unroll
        for (int half = 0; half < C::HALVES; ++half) {
          const uint32_t in_w = min((uint32_t)(s * C::HALVES + half) * 128 + 16 * chunk, w_ld - 16);
#pragma unroll
          for (int n = 0; n < C::NW; ++n) h.w[half][n] = loose16(w_base + (w_at[n] + in_w));
        }
      };
      // the 16 bytes at `at` of a row that ends at `end`, of which `v` are the row's last 16 if it ends before theirs
      auto cut = [](const v4u& v, uint32_t at, uint32_t end) -> v4u {
        const v4u part = without_first(v, (int)(16 - end % 16) % 16);
        v4u out;
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = at + 16 <= end ? v[j] : at < end ? part[j] : 0u;
        return out;
      };
      auto put = [&](const Held& h, int stage) {
#pragma unroll
        for (int n = 0; n < C::NX; ++n) *reinterpret_cast<v4u*>(ring + stage + (wave + 4 * n) * 1024 + lane * 16) = h.x[n];
#pragma unroll
        for (int half = 0; half < C::HALVES; ++half)
#pragma unroll
          for (int n = 0; n < C::NW; ++n)
            *reinterpret_cast<v4u*>(ring + stage + C::X_BYTES + half * C::W_BYTES + w_block(n) * 1024 + lane * 16) = h.w[half][n];
      };
      auto step = [&](int s, Held& h, int stage) {
        if (s == steps - 1 && w_ld % (128 * C::HALVES) != 0) {
#pragma unroll
          for (int n = 0; n < C::NX; ++n) h.x[n] = cut(h.x[n], (uint32_t)s * 128 + 16 * chunk, x_end);
#pragma unroll
          for (int half = 0; half < C::HALVES; ++half)
#pragma unroll
            for (int n = 0; n < C::NW; ++n) h.w[half][n] = cut(h.w[half][n], (uint32_t)(s * C::HALVES + half) * 128 + 16 * chunk, w_ld);
        }
        put(h, stage);
        load(min(s + 2, last - 1), h);
        wait_and_barrier<63>();  // (for what is in LDS, not for what is on its way to registers)
        multiply(stage);
      };
      Held h[2];
      load(first, h[0]);
      load(min(first + 1, last - 1), h[1]);
      for (int s = first; s < last; s += 2) {
        step(s, h[0], 0);
        if (s + 1 < last) step(s + 1, h[1], C::STAGE);
      }
    } else {
      for (int i = 0; i < S - 1; ++i)
        if (first + i < last) issue(first + i, i * C::STAGE);
      int now = 0, free = (S - 1) * C::STAGE;  // the stage of a step, and the one before, which is free behind the step's barrier
      for (int s = first; s < last; ++s) {
        if (s + S - 2 < last)
          wait_and_barrier<C::FLY*(S - 2)>();
        else
          wait_steps<C::FLY, S - 2, true>(last - 1 - s);
        if (s + S - 1 < last) issue(s + S - 1, free);
        multiply(now);
        free = now;
        now = now + C::STAGE < S * C::STAGE ? now + C::STAGE : 0;
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = (wave / RG) * (16 * MT) + 16 * m + i16;
      if (!((row < 64 ? members0 : members1) >> (row & 63) & 1)) continue;
      float* const to = t + ((int64_t)piece * a.M + row0 + row) * a.R + r0 + (wave % RG) * (16 * RW) + 4 * g;
#pragma unroll
      for (int r = 0; r < RW; ++r)
        if (r0 + (wave % RG) * (16 * RW) + 16 * r < a.R) *reinterpret_cast<v4f*>(to + 16 * r) = acc[m][r];
    }
  }
}

// Up to 8 rows a CU count as few; in the first product with more than 32 ranks, or rows that cannot come by DMA, up to one. us, gathered
// and in tiles, of 300, 1000, 2000 and 4096 rows, 11 requests with 5 adapters, 5120 x 5120. First product: 32 ranks 6.2 and 7.1, 9.6 and
// 12.0, 13.7 and 12.6, 25 and 21; 64 ranks 8.9 and 8.4, 14.8 and 14.8, 21 and 16, 36 and 24; 128 ranks 14 and 10, 31 and 20, 43 and 21, 70
// and 30; 16 ranks of 5121 x 5121 8.4 and 8.2, 19 and 11, 28 and 16, 41 and 32. Second product: 32 ranks 7.9 and 16, 14 and 20, 18 and 24,
// 36 and 31; 64 ranks 11 and 20, 20 and 26, 28 and 32, 54 and 41; 128 ranks 16 and 34, 29 and 42, 40 and 50, 79 and 63; 16 ranks of 5121 x
// 5121 8.6 and 15, 18 and 20, 28 and 25, 52 and 37.
constexpr int64_t kFewRows = 8;
struct Plan {
  int rt, groups, pieces, steps_per_piece;
  int tall_rt, tall_pieces, k_per_piece;  // ranks / 16 of a workgroup of lora_down_tall (0: not for this problem), and its cuts of K
};
Plan plan_of(int64_t M, int64_t K, int64_t R, int64_t cus) {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  Plan p = {};
  p.rt = R > 32 ? 4 : R > 16 ? 2 : 1;
  p.groups = R > 64 ? 2 : 1;
  // 32 KB of down for a workgroup, where K has them; more where there are workgroups enough.
  const int64_t tiles = up(M, 16) * up(R, 16 * p.rt * p.groups), steps = std::max<int64_t>(up(K, kStep), 1);
  const int64_t pieces = std::min(std::max<int64_t>(4 * cus / tiles, 1), up(steps, 16 / p.rt));
  p.steps_per_piece = (int)up(steps, pieces);
  p.pieces = (int)up(steps, p.steps_per_piece);
  p.tall_rt = M <= cus || K < 128 ? 0 : R > 64 ? 8 : p.rt;
  if (p.tall_rt) {
    const int64_t steps = up(K, 128), pieces = std::min(std::max<int64_t>(cus / (up(M, 128) * up(R, 16 * p.tall_rt)), 1), up(steps, 4));
    p.k_per_piece = (int)up(steps, pieces) * 128;
    p.tall_pieces = (int)up(K, p.k_per_piece);
  }
  return p;
}
// Workgroups that share the groups of up to 16 rows that 64 rows fall into: as many as there can be, up to `most`.
int slots_of(const Args& a, int64_t most) {
  const int64_t rows = std::min<int64_t>(a.M, 64), ids = a.rows_per_id == 1 ? rows : (rows - 1) / a.rows_per_id + 2;
  return (int)std::min<int64_t>({(rows + 15) / 16 - 1 + std::min<int64_t>(ids, (int64_t)a.adapters + 1), rows, most});
}

bool x_aligned(const Args& a) {
  const int64_t es = a.x_fp8 ? 1 : 2;
  return reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ld_x * es % 16 == 0 && reinterpret_cast<uintptr_t>(a.down) % 16 == 0 &&
         a.K % 8 == 0;
}
bool out_aligned(const Args& a) {
  return reinterpret_cast<uintptr_t>(a.base) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.ld_base % 8 == 0 &&
         a.ld_out % 8 == 0 && a.N % 8 == 0;
}

template <bool FP8, bool ANY>
void launch_down(const Args& a, const Plan& p, float* t, hipStream_t stream) {
  const int slots = slots_of(a, 32);  // (fewer for many rows: 1000 of 200 requests 8.3 and 11.3 us, 128 tokens 14.0 and 12.6)
  const dim3 grid((unsigned)((a.M + 63) / 64), (unsigned)(p.pieces * slots),
                  (unsigned)((a.R + 16 * p.rt * p.groups - 1) / (16 * p.rt * p.groups)));
  const size_t lds = (size_t)p.groups * 2 * p.rt * 64 * sizeof(v4f);
#define CDIT_LORA_CASE(RT) \
  if (p.rt == RT) hipLaunchKernelGGL((lora_down<FP8, ANY, RT>), grid, dim3(256 * p.groups), lds, stream, a, t, p.steps_per_piece, slots);
  CDIT_LORA_CASE(1)
  CDIT_LORA_CASE(2)
  CDIT_LORA_CASE(4)
#undef CDIT_LORA_CASE
}

template <bool FP8, bool ANY>
int launch_down_tall(const Args& a, const Plan& p, float* t, hipStream_t stream) {
  const bool by_request = a.rows_per_id >= kTallRows;
  const int64_t rows = by_request ? std::min(a.rows_per_id, a.M) : a.M, tiles = (rows + kTallRows - 1) / kTallRows;
  const dim3 grid((unsigned)((a.M + rows - 1) / rows * tiles), (unsigned)(p.tall_pieces * kSlots),
                  (unsigned)((a.R + 16 * p.tall_rt - 1) / (16 * p.tall_rt)));
  auto launch = [&](auto kernel, int lds, bool* done) {
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, done)) return rc;
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, stream, a, t, p.k_per_piece, (int)tiles, rows);
    return 0;
  };
  static bool done[4][64];
#define CDIT_LORA_CASE(RT, I) \
  if (p.tall_rt == RT) return launch(lora_down_tall<FP8, ANY, RT>, Tall<FP8, ANY, RT>::STAGE * Tall<FP8, ANY, RT>::STAGES, done[I]);
  CDIT_LORA_CASE(1, 0)
  CDIT_LORA_CASE(2, 1)
  CDIT_LORA_CASE(4, 2)
  CDIT_LORA_CASE(8, 3)
#undef CDIT_LORA_CASE
  return 0;
}

template <bool ANY>
int launch_up(const Args& a, int pieces, const float* t, int64_t cus, hipStream_t stream) {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t blocks = up(a.N, 128);
  if (a.M <= kFewRows * cus || a.N < 8) {
    // As many workgroups as run at once; 32 slots in all, or 5 for 64 rows (rows that are next to one another fall into one group more
    // than four). us, with 32 for 64 rows and so: 128 tokens with 64 adapters 35 and 22, 200 with 24 41 and 23; 1244 rows of 53 requests
    // with 28 22 and 16.
    const int64_t tiles = up(a.M, 64), slots = slots_of(a, std::max<int64_t>(32 / tiles, 5));
    const int64_t cuts = std::min(blocks, std::max<int64_t>(1, 4 * cus / (tiles * slots)));
    const int columns = (int)(up(blocks, cuts) * 128);
    hipLaunchKernelGGL((lora_up<ANY>), dim3((unsigned)tiles, (unsigned)up(a.N, columns), (unsigned)slots), dim3(256),
                       (size_t)2 * 16 * (a.R + 8) * 2, stream, a, t, pieces, columns);
    return 0;
  }
  const int64_t rows = a.rows_per_id >= 64 ? std::min(a.rows_per_id, a.M) : a.M, tiles_per_id = up(rows, 64), tiles = up(a.M, rows) * tiles_per_id;
  // As many workgroups as run at once, each of which stages its t once.
  const int64_t cuts = std::min(blocks, std::max<int64_t>(1, 2 * cus / tiles));
  const int columns = (int)(up(blocks, cuts) * 128);
  const dim3 grid((unsigned)tiles, (unsigned)up(a.N, columns));
  auto launch = [&](auto kernel, bool* done) {
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), 2 * 64 * (256 + 8) * 2, done)) return rc;
    hipLaunchKernelGGL(kernel, grid, dim3(256), (size_t)2 * 64 * (a.R + 8) * 2, stream, a, t, pieces, columns, (int)tiles_per_id, rows);
    return 0;
  };
  static bool done[4][64];
  return a.R <= 32 ? launch(lora_up_rows<ANY, 1>, done[0]) : a.R <= 64 ? launch(lora_up_rows<ANY, 2>, done[1])
       : a.R <= 128 ? launch(lora_up_rows<ANY, 4>, done[2]) : launch(lora_up_rows<ANY, 8>, done[3]);
}

}  // namespace

int64_t lora_workspace(int64_t M, int64_t K, int64_t R, int64_t cus) {
  const Plan p = plan_of(M, K, R, cus);
  return (int64_t)std::max(p.pieces, p.tall_pieces) * M * R * (int64_t)sizeof(float);
}

int launch_lora(const cdit_lora_args& a, float* t, int64_t cus, hipStream_t stream) {
  const Plan p = plan_of(a.M, a.K, a.R, cus);
  const bool aligned = x_aligned(a), dma = aligned && a.K % (a.x_fp8 ? 16 : 8) == 0,
             tall = p.tall_rt && (a.M > kFewRows * cus || a.R > 32 || !dma) && 128 * a.ld_x * 2 < kTallBytes && 256 * a.K * 2 < kTallBytes;
  if (tall) {
    if (int rc = a.x_fp8 ? dma ? launch_down_tall<true, false>(a, p, t, stream) : launch_down_tall<true, true>(a, p, t, stream)
                         : dma ? launch_down_tall<false, false>(a, p, t, stream) : launch_down_tall<false, true>(a, p, t, stream))
      return rc;
  } else if (aligned) {
    a.x_fp8 ? launch_down<true, false>(a, p, t, stream) : launch_down<false, false>(a, p, t, stream);
  } else {
    a.x_fp8 ? launch_down<true, true>(a, p, t, stream) : launch_down<false, true>(a, p, t, stream);
  }
  const int pieces = tall ? p.tall_pieces : p.pieces;
  return out_aligned(a) ? launch_up<false>(a, pieces, t, cus, stream) : launch_up<true>(a, pieces, t, cus, stream);
}

}  // namespace cdit
