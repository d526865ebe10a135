// mi_pieces.h - what the kernels of many rows (prefill and scoring) share beside mi_common.h: stores at the elements' own
// alignment, and maxima over the lanes of a column.
#pragma once
#include "mi_common.h"

namespace mi {

// outputs are stored in pieces of several elements at the elements' own alignment
typedef f4_t f4_any __attribute__((aligned(4)));
typedef uint32_t h2_any __attribute__((aligned(2)));
typedef u2_t h4_any __attribute__((aligned(2)));
typedef u4_t h8_any __attribute__((aligned(2)));

// (v_maximum3_f32: fmaxf would quieten each operand first, an instruction per operand)
__device__ __forceinline__ float max3(float x, float y, float z) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x, y), z);
}
// the max over the four lanes l % 16 + 16 k that hold one column's scores
__device__ __forceinline__ float col_max(float x) {
  float a0 = x, a1 = x;
  lane_swap16(a0, a1);
  float b0 = __builtin_elementwise_maximum(a0, a1), b1 = b0;
  lane_swap32(b0, b1);
  return __builtin_elementwise_maximum(b0, b1);
}

}  // namespace mi
