// Grouped products of bfloat16 operands, sums in float32.
#include "grouped_launch.h"
#include "grouped_skinny.h"
#define DM 2

#define TY GT_BF16
extern "C" void launch_grouped_bf16(const GroupedArgs* p, int tile, int bk,
                                  int weights, int fast, hipStream_t s) {
  if (weights) {
    if (!fast) grouped_go<TY, 128, 128, 2, 2, 2, false, false, true, false>(*p, s);
    else if (tile == 2) grouped_big_go<TY, false, false, true>(*p, s);
    else grouped_go<TY, 128, 128, 2, 2, DM, false, false, true, true>(*p, s);
  } else if (tile < 0) {
    if (tile == -1) grouped_skinny_go<TY, 1>(*p, fast, s);
    else grouped_skinny_go<TY, 2>(*p, fast, s);
  } else if (bk) {
    if (!fast) grouped_go<TY, 128, 128, 2, 2, 2, true, true, false, false>(*p, s);
    else if (tile == 2) grouped_big_go<TY, true, true, false>(*p, s);
    else if (tile == 1) grouped_go<TY, 128, 128, 2, 2, DM, true, true, false, true>(*p, s);
    else grouped_go<TY, 32, 128, 1, 4, 3, true, true, false, true>(*p, s);
  } else {
    if (!fast) grouped_go<TY, 128, 128, 2, 2, 2, true, false, false, false>(*p, s);
    else if (tile == 2) grouped_big_go<TY, true, false, false>(*p, s);
    else if (tile == 1) grouped_go<TY, 128, 128, 2, 2, DM, true, false, false, true>(*p, s);
    else grouped_go<TY, 32, 128, 1, 4, 3, true, false, false, true>(*p, s);
  }
}
