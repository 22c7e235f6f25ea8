// elem.cuh -- conversions between fp32 and the element types of the integer operators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sm100.cuh"

namespace srdit {

SRDIT_DEV float to_f(float v) { return v; }
SRDIT_DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
SRDIT_DEV float to_f(__half v) { return __half2float(v); }

// x and y rounded to nearest as one word, x in its low half
SRDIT_DEV uint32_t pack2(float x, float y, __nv_bfloat16) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(y), "f"(x));
  return d;
}
SRDIT_DEV uint32_t pack2(float x, float y, __half) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(y), "f"(x));
  return d;
}

}  // namespace srdit
