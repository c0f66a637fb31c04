// Grouped products of e4m3 operands with a float32 scale for each 128 of a
// row of a and each 128 x 128 tile of b.
#include "grouped_launch.h"
#include "grouped_skinny.h"
#define DM 2

extern "C" void launch_grouped_fp8(const GroupedArgs* p, int tile, int fast,
                                   hipStream_t s) {
  if (tile == -1) grouped_skinny_go<GT_FP8, 1>(*p, fast, s);
  else if (tile == -2) grouped_skinny_go<GT_FP8, 2>(*p, fast, s);
    else if (!fast) grouped_go<GT_FP8, 128, 128, 2, 2, 2, true, true, false, false>(*p, s);
  else if (tile == 2) grouped_big_go<GT_FP8, true, true, false>(*p, s);
  else if (tile == 1) grouped_go<GT_FP8, 128, 128, 2, 2, DM, true, true, false, true>(*p, s);
  else grouped_go<GT_FP8, 32, 128, 1, 4, 3, true, true, false, true>(*p, s);
}
