// Tile choice and launch of grouped_k, one translation unit a type.
#pragma once
#include "grouped_core.h"

template <int TY, int BM, int BN, int WM, int WN, int D, bool AK, bool BK,
          bool WEIGHTS, bool FAST>
static void grouped_go(const GroupedArgs& p, hipStream_t s) {
  const long ntn = (p.N + BN - 1) / BN;
  // every range of rows that is not empty can end inside one tile more
  const long ntm = WEIGHTS ? (long)p.E * ((p.M + BM - 1) / BM)
                           : p.T / BM + p.E + 2;
  const size_t lds =
      D * ((BM + BN) * 128 + (TY == GT_FP8 ? WM * WN * 256 : 0));
  auto k = grouped_k<TY, BM, BN, WM, WN, D, AK, BK, WEIGHTS, FAST>;
  hipLaunchKernelGGL(k, dim3((unsigned)(ntm * ntn), (unsigned)p.splits),
                     dim3(64 * WM * WN), lds, s, p);
}

template <int TY, bool AK, bool BK, bool WEIGHTS>
static void grouped_big_go(const GroupedArgs& p, hipStream_t s) {
  const long ntn = (p.N + 255) / 256;
  const long ntm = WEIGHTS ? (long)p.E * ((p.M + 255) / 256)
                           : p.T / 256 + p.E + 2;
  auto k = grouped_big_k<TY, AK, BK, WEIGHTS>;
  hipLaunchKernelGGL(k, dim3((unsigned)(ntm * ntn), (unsigned)p.splits),
                     dim3(512), 2 * 4 * 128 * 128, s, p);
}
