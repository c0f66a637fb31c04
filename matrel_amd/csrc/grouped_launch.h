// Tile choice and launch of grouped_k, one translation unit a type.
#pragma once
#include "grouped_core.h"
#include "grouped_skinny.h"

template <int TY, int BM, int BN, int WM, int WN, int D, bool AK, bool BK,
          bool WEIGHTS, RowsPath PATH>
static void grouped_go(const GroupedArgs& p, hipStream_t s) {
  const long ntn = (p.N + BN - 1) / BN;
  const long ntm = WEIGHTS ? (long)p.E * ((p.M + BM - 1) / BM)
                           : grouped_row_tiles(p, BM);
  const size_t lds =
      D * ((BM + BN) * 128 + (TY == GT_FP8 ? WM * WN * 256 : 0));
  auto k = grouped_k<TY, BM, BN, WM, WN, D, AK, BK, WEIGHTS, PATH>;
  hipLaunchKernelGGL(k, dim3((unsigned)(ntm * ntn), (unsigned)p.splits),
                     dim3(64 * WM * WN), lds, s, p);
}

template <int TY, bool AK, bool BK, bool WEIGHTS>
static void grouped_big_go(const GroupedArgs& p, hipStream_t s) {
  const long ntn = (p.N + 255) / 256;
  const long ntm = WEIGHTS ? (long)p.E * ((p.M + 255) / 256)
                           : grouped_row_tiles(p, 256);
  auto k = grouped_big_k<TY, AK, BK, WEIGHTS>;
  hipLaunchKernelGGL(k, dim3((unsigned)(ntm * ntn), (unsigned)p.splits),
                     dim3(512),
                     2 * (4 * 128 * 128 + (TY == GT_FP8 ? 2048 : 0)), s, p);
}

// Tile codes, as ext_grouped.cpp picks them.
//   -1, -2: 16, 32 rows, columns by 16 (b with k along its rows)
//   0: 32 x 128   1: 64 x 64   2: 128 x 128   3: 256 x 256 (not f32)
// Stages: as many as let two workgroups (64 x 64: three) share a CU's LDS.
// More stages for fewer workgroups lost: bf16 8192 rows, 8 groups, 4096 x 2048,
// 128 x 128 with 2 / 4 stages: 169 / 229 us; f32 4096 rows, 12 groups, 1024 x
// 1000, 64 x 64 with 3 / 4: 93 / 98 us.
template <int TY, bool BK>
static void launch_rows_tile(const GroupedArgs& p, int tile, int path,
                             hipStream_t s) {
  if constexpr (BK) {
    if (tile == -1) return grouped_skinny_go<TY, 1>(p, path == ALIGNED, s);
    if (tile == -2) return grouped_skinny_go<TY, 2>(p, path == ALIGNED, s);
  }
  if (path == SLOW)
    return grouped_go<TY, 64, 64, 2, 2, 1, true, BK, false, SLOW>(p, s);
  if (path == ANY) {
    if (tile == 2)
      return grouped_go<TY, 128, 128, 2, 2, 2, true, BK, false, ANY>(p, s);
    return grouped_go<TY, 64, 64, 2, 2, 2, true, BK, false, ANY>(p, s);
  }
  if constexpr (TY != GT_F32)
    if (tile == 3) return grouped_big_go<TY, true, BK, false>(p, s);
  if (tile >= 2)
    return grouped_go<TY, 128, 128, 2, 2, 2, true, BK, false, ALIGNED>(p, s);
  if (tile == 1)
    return grouped_go<TY, 64, 64, 2, 2, 3, true, BK, false, ALIGNED>(p, s);
  if constexpr (!BK)  // with k along b's rows, -1 and -2 take few rows
    grouped_go<TY, 32, 128, 1, 4, 3, true, BK, false, ALIGNED>(p, s);
}

template <int TY>
static void launch_weights_tile(const GroupedArgs& p, int tile, int path,
                                hipStream_t s) {
  if (path == SLOW)
    return grouped_go<TY, 64, 64, 2, 2, 1, false, false, true, SLOW>(p, s);
  if (path == ANY) {
    if (tile >= 2)
      return grouped_go<TY, 128, 128, 2, 2, 2, false, false, true, ANY>(p, s);
    return grouped_go<TY, 64, 64, 2, 2, 2, false, false, true, ANY>(p, s);
  }
  if constexpr (TY != GT_F32)
    if (tile == 3) return grouped_big_go<TY, false, false, true>(p, s);
  if (tile >= 2)
    return grouped_go<TY, 128, 128, 2, 2, 2, false, false, true, ALIGNED>(p, s);
  grouped_go<TY, 64, 64, 2, 2, 3, false, false, true, ALIGNED>(p, s);
}
