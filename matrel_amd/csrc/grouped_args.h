// What the host hands to the grouped products.
#pragma once

#include <algorithm>

enum GroupedType { GT_BF16 = 0, GT_F16 = 1, GT_F32 = 2, GT_FP8 = 3 };

struct GroupedArgs {
  const void* a;      // rows: [T][K]; weights: [T][M]
  const void* b;      // rows: [E] of (n, k); weights: [T][N]
  void* c;            // rows: [T][N]; weights: [E][M][N]
  float* part;        // f32 partial sums [splits][...], null if splits == 1
  const void* offs;   // E + 1 offsets, null: one group of all rows
  const float* asc;   // fp8: scales of a, [ceil(K/128)][T]
  const float* bsc;   // fp8: scales of b, [E][ceil(K/128)][ceil(N/128)]
  long lda, ldb;      // elements from one row (or one k) to the next
  long gsb;           // rows: elements from one group's b to the next
  int T, M, N, K, E;
  int off64;          // offsets are 64-bit
  int splits;
  int out;            // GroupedType of c
  int accum;          // add to c (f32, one split)
};

// Row tiles of T rows in E groups, a head and a tail, at most: each of these
// ranges that is not empty can end inside a tile, and no more than T are not.
inline long grouped_row_tiles(const GroupedArgs& p, int bm) {
  return p.T / bm + std::min((long)p.E + 2, (long)p.T);
}

// Few rows: a workgroup makes blocks of 16 columns from n0 on, one after
// another. The first column of block j; where fewer blocks are left, of the
// last one that holds a column.
constexpr int few_rows_block(int n, int n0, int j) {
  return n0 + 16 * std::min(j, (n - 1 - n0) / 16);
}

// Row i of the 16 rows of b that such a block reads, from its first one: a
// block that ends early reads its last row again.
constexpr int few_rows_row(int n, int block, int i) {
  return std::min(i, n - 1 - block);
}
