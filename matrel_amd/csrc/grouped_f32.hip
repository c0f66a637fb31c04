// Grouped products of float32 operands (exact float32 matrix instructions),
// and the join of partial sums for all types.
#include "grouped_launch.h"

#define TY GT_F32
extern "C" void launch_grouped_f32(const GroupedArgs* p, int tile, int bk,
                                  int weights, int path, hipStream_t s) {
  if (weights) launch_weights_tile<TY>(*p, tile, path, s);
  else if (bk) launch_rows_tile<TY, true>(*p, tile, path, s);
  else launch_rows_tile<TY, false>(*p, tile, path, s);
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
