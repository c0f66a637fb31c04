// Grouped products of float32 operands (exact float32 matrix instructions),
// and the join of partial sums for all types.
#include "grouped_launch.h"
#include "grouped_skinny.h"
#define DM 2

#define TY GT_F32
extern "C" void launch_grouped_f32(const GroupedArgs* p, int tile, int bk,
                                   int weights, int fast, hipStream_t s) {
  if (weights) {
    if (!fast) grouped_go<TY, 128, 128, 2, 2, 2, false, false, true, false>(*p, s);
    else grouped_go<TY, 128, 128, 2, 2, DM, false, false, true, true>(*p, s);
  } else if (tile < 0) {
    if (tile == -1) grouped_skinny_go<TY, 1>(*p, fast, s);
    else grouped_skinny_go<TY, 2>(*p, fast, s);
  } else if (bk) {
    if (!fast) grouped_go<TY, 128, 128, 2, 2, 2, true, true, false, false>(*p, s);
    else if (tile >= 1) grouped_go<TY, 128, 128, 2, 2, DM, true, true, false, true>(*p, s);
    else grouped_go<TY, 32, 128, 1, 4, 3, true, true, false, true>(*p, s);
  } else {
    if (!fast) grouped_go<TY, 128, 128, 2, 2, 2, true, false, false, false>(*p, s);
    else if (tile >= 1) grouped_go<TY, 128, 128, 2, 2, DM, true, false, false, true>(*p, s);
    else grouped_go<TY, 32, 128, 1, 4, 3, true, false, false, true>(*p, s);
  }
}

// The partial sums of a split axis, added in the order of the axis.
__global__ void __launch_bounds__(256)
grouped_join_k(const float* __restrict__ part, void* __restrict__ c, long n,
               int splits, int ty) {
  const long at = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  const int have = (int)min(4L, n - at);
  const bool vec = n % 4 == 0;
  f32x4 sum = {0, 0, 0, 0};
  for (int s = 0; s < splits; ++s) {
    const float* x = part + s * n + at;
    if (vec) {
      sum += *(const f32x4*)x;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < have) sum[i] += x[i];
    }
  }
  store4(c, at, ty, sum, have, vec);
}

extern "C" void launch_grouped_join(const float* part, void* c, long n,
                                    int splits, int ty, hipStream_t s) {
  hipLaunchKernelGGL(grouped_join_k, dim3((unsigned)((n + 1023) / 1024)),
                     dim3(256), 0, s, part, c, n, splits, ty);
}
