// How the 4-bit kernel for few rows (gemm_mx_rows.hip) lays out its workgroup's memory. Host arithmetic without HIP: it is
// tested on the CPU.
#ifndef CDIT_MX_ROWS_PLAN_H_
#define CDIT_MX_ROWS_PLAN_H_

#include <stdint.h>

#include <algorithm>

namespace cdit {

constexpr int kMxRowsMost = 16;          // rows of a workgroup
constexpr int kMxRowsItem = 512;         // along K
constexpr int kMxRowsWaves = 8;          // at most
constexpr int kMxRowsLds = 64 * 1024;    // of activation and scales: two workgroups fit a CU

// Bytes of a row of the activation in LDS for `items` items, and of a row of scales. 16 (4) more than a multiple of 256 (16): the
// 16 rows a pass reads start in different banks.
constexpr int mx_row_pitch(bool weight_only, int items) { return items * (weight_only ? 1024 : 256) + 16; }
constexpr int mx_scale_pitch(int items) { return items * 16 + 4; }

struct MxRowsPlan {
  int groups;  // of 16 columns, a workgroup
  int chunk;   // items of K in LDS at a time
  int waves;
  int lds;     // bytes
};
inline MxRowsPlan mx_rows_plan(bool weight_only, int M, int N, int K, int cus) {
  const int items = std::max(1, (int)(((int64_t)K + kMxRowsItem - 1) / kMxRowsItem)), rows = std::min(M, kMxRowsMost);
  MxRowsPlan p;
  // Two groups of columns a workgroup where there are more than two for each CU: 30720 columns, K 5120, one row 23.1 us with one,
  // 21.5 with two, 23.9 with four (5 wavefronts; 10 are slower throughout). 8 wavefronts at most: 13824 columns, K 5120
  // 12.8 us with 5 or 8, 15.6 with 10; K 16384 33.2 with 8, 41.1 with 16.
  p.groups = ((int64_t)N + 15) / 16 > 2 * (int64_t)cus ? 2 : 1;
  // As many items of the activation and of scales as fit; even shares of them for the wavefronts. (Sizes of all of K pass 32 bits
  // from K = 2^26 on: they are never formed.)
  const int more = rows * (mx_row_pitch(weight_only, 1) - mx_row_pitch(weight_only, 0) + 16) + 16 * p.groups * 16;  // of an item
  const int none = rows * (mx_row_pitch(weight_only, 0) + mx_scale_pitch(0)) + 16 * p.groups * mx_scale_pitch(0);
  p.chunk = std::min(items, std::max(1, (kMxRowsLds - none) / more));
  const int per = (p.chunk + kMxRowsWaves - 1) / kMxRowsWaves;
  p.waves = (p.chunk + per - 1) / per;
  p.lds = p.groups * p.waves * 1024 + none + p.chunk * more;
  return p;
}

}  // namespace cdit
#endif
