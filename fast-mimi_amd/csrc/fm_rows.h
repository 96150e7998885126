// What the row norms share: rows held in registers by the lanes that reduce them, and
// how a call's sizes choose those lanes.
#pragma once

#include "fm_common.h"

namespace {

template <typename T> FM_DEVICE float widen(T v) { return (float)v; }

// Sums over the LPR lanes of a row; with 256, a block's waves, through `waves`
// (of its own for each sum between two barriers).
template <int LPR>
FM_DEVICE float row_sum(float v, float* waves = nullptr) {
#pragma unroll
  for (int o = 1; o < (LPR < 64 ? LPR : 64); o <<= 1) v += __shfl_xor(v, o, 64);
  if constexpr (LPR == 256) {
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (waves[0] + waves[1]) + (waves[2] + waves[3]);
  }
  return v;
}
template <int LPR>
FM_DEVICE void row_sums(float& s1, float& s2, float (*waves)[4]) {
  s1 = row_sum<(LPR < 64 ? LPR : 64)>(s1), s2 = row_sum<(LPR < 64 ? LPR : 64)>(s2);
  if constexpr (LPR == 256) {
    if ((threadIdx.x & 63) == 0) waves[0][threadIdx.x >> 6] = s1, waves[1][threadIdx.x >> 6] = s2;
    __syncthreads();
    s1 = (waves[0][0] + waves[0][1]) + (waves[0][2] + waves[0][3]);
    s2 = (waves[1][0] + waves[1][1]) + (waves[1][2] + waves[1][3]);
  }
}

// How a call runs: elements per access, vectors per lane, lanes per row (0
// vectors: the kernels that take any size).  A wave a row up to four vectors a
// lane, then a block a row, so that a lane's columns (three FP32 values each in
// the backward) stay in registers with several blocks on a CU: 20000 x 4096
// bfloat16 backward, one wave / one block a row, 147 / 121 us; FP32, rows read again
// at each step / one block a row, 793 / 196 us.  (Up to four vectors a wave is as
// good: 20000 x 1024 FP32 forward 26 / 30 us, backward 47 / 45.)  Single elements,
// where 16 bytes do not fit: up to eight a lane (50000 x 257 bfloat16 forward, one
// wave / one block a row, 29 / 55 us).
struct Plan {
  int e, nv, lpr;
};

Plan plan(int C, int size, bool aligned) {
  const int full = 16 / size, e = aligned && C % full == 0 ? full : 1;
  const int n = C / e;
  if (n <= 16) return {e, 1, 16};
  for (int nv : {1, 2, 4, 8})
    if (nv <= (e == 1 ? 8 : 4) && n <= 64 * nv) return {e, nv, 64};
  for (int nv : {2, 4, 8, 32})
    if (nv <= 32 / e && n <= 256 * nv) return {e, nv, 256};
  return {e, 0, 64};
}

constexpr int ONE_BLOCK = 8;  // rows of a group that are left to one block

// Backward blocks: enough to fill the chip (four to a CU), each with at least two
// rows per group; one alone (no second launch) for a handful of rows.  A block's
// partial sums are two FP32 rows to write and to join: beyond two blocks a CU they
// are held to a quarter of an input (8191 x 2048 bfloat16 34 -> 27 us).
int backward_blocks(long rows, const Plan& p, int size) {
  const int groups = p.nv && p.lpr < 256 ? 256 / p.lpr : 1;
  if (p.nv && rows <= ONE_BLOCK * groups) return 1;
  const long most = std::min<long>(1024, std::max<long>(512, rows * size / 32));
  return (int)std::max<long>(1, std::min<long>(most, (rows + 2 * groups - 1) / (2 * groups)));
}

}  // namespace
