// Grouped products of e4m3 operands with a float32 scale for each 128 of a
// row of a and each 128 x 128 tile of b.
#include "grouped_launch.h"

extern "C" void launch_grouped_fp8(const GroupedArgs* p, int tile, int path,
                                   hipStream_t s) {
  launch_rows_tile<GT_FP8, true>(*p, tile, path, s);
}
