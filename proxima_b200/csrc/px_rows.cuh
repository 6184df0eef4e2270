// Device helpers shared by the operators on embedding rows.
#pragma once

#include "px_tc.cuh"

namespace px {

// A bounded wait whose outcome nobody acts on (drains before an exit).
__device__ __forceinline__ void quiet_wait(uint32_t bar, uint32_t parity) {
  int dummy = 0;
  tc::mbar_wait(bar, parity, &dummy);
}

// Packed pairs of fp32: one instruction, two results.
struct F2 {
  uint64_t w;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.w) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack(F2 a, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.w));
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.w) : "l"(a.w), "l"(b.w), "l"(c.w));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
  return r;
}

}  // namespace px
