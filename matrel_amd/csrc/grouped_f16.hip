// Grouped products of float16 operands, sums in float32.
#include "grouped_launch.h"

#define TY GT_F16
extern "C" void launch_grouped_f16(const GroupedArgs* p, int tile, int bk,
                                  int weights, int path, hipStream_t s) {
  if (weights) launch_weights_tile<TY>(*p, tile, path, s);
  else if (bk) launch_rows_tile<TY, true>(*p, tile, path, s);
  else launch_rows_tile<TY, false>(*p, tile, path, s);
}
