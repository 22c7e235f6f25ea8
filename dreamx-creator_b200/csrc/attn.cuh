// attn.cuh -- what the attention kernels over keys of any length share: the exponential in
// base 2, maxima that keep a NaN, divisions by products, and mma.sync with its operands' moves.
#pragma once
#include "elem.cuh"

namespace srdit {

constexpr float kLog2e = 1.4426950408889634f;

// n / d and n % d for 0 <= n < 2^31 by a product: mul = ceil(2^(31 + l) / d), 2^l >= d
struct Divisor {
  uint32_t mul, shift;
  int d;
  static Divisor of(int d) {
    uint32_t l = 0;
    while ((1ll << l) < d) ++l;
    const uint64_t two = 1ull << (31 + l);
    return {static_cast<uint32_t>((two + d - 1) / d), 31 + l, d};
  }
  SRDIT_DEV int div(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift);
  }
  SRDIT_DEV int mod(int n) const { return n - div(n) * d; }
};

SRDIT_DEV float neg_inf() { return -__int_as_float(0x7f800000); }
SRDIT_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the larger of two, the largest of three; NaN if one is
SRDIT_DEV float max2(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
SRDIT_DEV float max3(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
template <typename T>
SRDIT_DEV void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                        uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
SRDIT_DEV uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
SRDIT_DEV uint4 lds16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(src));
  return v;
}

}  // namespace srdit
