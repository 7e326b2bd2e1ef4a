// fp32 arithmetic on two elements at a time (f32x2), and the square root made of it.
#pragma once

#include <cuda_runtime.h>

namespace coco {
namespace {

typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void unpair(Pair p, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
  return p;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(a), "l"(b), "l"(c));
  return p;
}
__device__ __forceinline__ Pair twice(float a) { return pair(a, a); }
// a + b of products that are to be rounded first.  One by one: the compiler fuses a
// packed multiply into a packed add whatever their rounding modifiers say, and a last
// bit of a moment is a whole step of its code now and then.
__device__ __forceinline__ void sum2(Pair a, Pair b, float &x, float &y) {
  float a0, a1, b0, b1;
  unpair(a, a0, a1);
  unpair(b, b0, b1);
  x = __fadd_rn(a0, b0), y = __fadd_rn(a1, b1);
}
// Of -v, the negative of the root as the state keeps it, rounded to nearest: with y
// the hardware's reciprocal root of v, one Newton step r + (v - r^2) y / 2 from
// r = v y.  The multiply-add leaves the residual exact for v from 2^-100 on; 0 gives +0.
// An estimate y that is a unit or two off could leave a few significands a unit off the
// nearest root; this GPU's leaves none: the test goes through every fp32 number.
// (Negative throughout, so that no operand has to be negated.)
__device__ __forceinline__ Pair neg_root(Pair neg_v) {
  float v0, v1, y0, y1;
  unpair(neg_v, v0, v1);
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y0) : "f"(fmaxf(-v0, 0x1p-100f)));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y1) : "f"(fmaxf(-v1, 0x1p-100f)));
  const Pair y = pair(y0, y1), r = mul2(neg_v, y);
  return fma2(fma2(r, r, neg_v), mul2(y, twice(0.5f)), r);
}
// The same for any v: small ones scaled up first; inf and nan are their own roots.
__device__ __forceinline__ float neg_root_any(float neg_v) {
  const bool small = -neg_v < 0x1p-64f;
  float r, other;
  unpair(neg_root(pair(small ? neg_v * 0x1p64f : neg_v, 0.f)), r, other);
  if (small) r *= 0x1p-32f;
  return -neg_v < __uint_as_float(0x7f800000u) ? r : neg_v;
}

}  // namespace
}  // namespace coco
