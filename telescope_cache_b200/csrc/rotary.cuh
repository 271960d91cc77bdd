// One rotated pair, shared by the rotary pass and the fused cache step.
#pragma once

#include <type_traits>

namespace tc {

// y1 = x1 c - x2 s, y2 = x2 c + x1 s; no contraction, so that every kernel that
// rotates gives the same bits.
__device__ __forceinline__ void rotate_pair(float x1, float x2, float c, float s, float* y1, float* y2) {
  *y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
  *y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
}

}  // namespace tc
