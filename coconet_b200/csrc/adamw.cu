// AdamW over a list of tensors, with fp32 moments or with moments in 8 bits.
//
// Per element, t = step + 1, d1 = 1 - beta1^t, d2 = 1 - beta2^t (from the host):
//   g <- (sum over ranks of g) * grad_scale * clip
//   m <- beta1 m + (1 - beta1) g        v <- beta2 v + (1 - beta2) g^2
//   w <- w (1 - lr decay) - (lr / d1) m / (sqrt(v) / sqrt(d2) + eps)
// All paths run the same roundings, so the results do not depend on the path an
// element takes; moments, codes and scales match a scalar evaluation bit for bit.
//
// 8-bit moments: m and r = sqrt(v) as e4m3 codes with one power-of-two scale
// per 256 elements (e8m0: the exponent byte of a float).  r and not v: the
// quotient needs the root, whose range (2^16 under a block's scale) covers
// twice as many binades of v.  A code step is 1/8 of the value while a step of
// training moves v by 1 - beta2 of itself, so rounding to nearest would freeze
// the moments; they are rounded up or down at random with the probability of
// the part cut off, which keeps them right on average.  The random bits are a
// hash of the element's place, the step and a seed: the same on every rank
// count, launch shape and path.  A positive r never becomes 0 (the step would
// be m / eps).
//
// What bounds it: HBM.  One pass, every byte moved once; nothing is reused.
#include "list_device.cuh"

#ifndef COCO_ADAMW_THREADS
#define COCO_ADAMW_THREADS 384
#endif
#ifndef COCO_ADAMW_PEER_THREADS
#define COCO_ADAMW_PEER_THREADS 256
#endif

namespace coco {
namespace {

// ---- where a tensor's elements are --------------------------------------------
template <int RB> struct View {   // several ranks: tables in device memory
  const void *const *g;
  void *const *out;
  float *w;
};
template <> struct View<1> {
  const void *g[1];
  float *w;
  void *lp;
};

template <int RB> __device__ __forceinline__ void put_lp4(const View<RB> &v, int R, int kind, size_t i,
                                                          const float (&x)[4]) {
  uint2 q;
  if (kind == kLpF16) {
    const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
    q = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    q = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
  }
  if constexpr (RB == 1) {
    *reinterpret_cast<uint2 *>((unsigned short *)v.lp + i) = q;
  } else {
#pragma unroll
    for (int p = 0; p < RB; ++p)
      if (RB == 2 || p < R) st_sys_8((unsigned short *)v.out[p] + i, q);
  }
}
template <int RB> __device__ __forceinline__ void put_lp1(const View<RB> &v, int R, int kind, size_t i,
                                                          float x) {
  const unsigned short h =
      kind == kLpF16 ? Bits16<__half>::from_f32(x) : Bits16<__nv_bfloat16>::from_f32(x);
  if constexpr (RB == 1) {
    ((unsigned short *)v.lp)[i] = h;
  } else {
    for (int p = 0; p < R; ++p) st_sys_2((unsigned short *)v.out[p] + i, h);
  }
}
// New weights: the own fp32 values and the copy for everybody, or, without a
// copy, the fp32 values for everybody.
template <int RB> __device__ __forceinline__ void put_w4(const View<RB> &v, int R, int kind, size_t i,
                                                         const float (&x)[4]) {
  if (RB == 1 || kind != kLpNone)
    *reinterpret_cast<float4 *>(v.w + i) = make_float4(x[0], x[1], x[2], x[3]);
  if (kind != kLpNone) {
    put_lp4<RB>(v, R, kind, i, x);
  } else if constexpr (RB > 1) {
    const uint4 q = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                               __float_as_uint(x[3]));
#pragma unroll
    for (int p = 0; p < RB; ++p)
      if (RB == 2 || p < R) st_sys_16((float *)v.out[p] + i, q);
  }
}
template <int RB> __device__ __forceinline__ void put_w1(const View<RB> &v, int R, int kind, size_t i,
                                                         float x) {
  if (RB == 1 || kind != kLpNone) v.w[i] = x;
  if (kind != kLpNone) {
    put_lp1<RB>(v, R, kind, i, x);
  } else if constexpr (RB > 1) {
    for (int p = 0; p < R; ++p) st_sys_4((float *)v.out[p] + i, __float_as_uint(x));
  }
}

// ---- the update ------------------------------------------------------------------
// The reciprocal is the hardware's, within 2^-23, and so is the root of fp32
// moments: the exact ones branch per element, which keeps the elements' chains
// from overlapping (104 us against 74 for 12.6 M elements), and the update they
// serve is small against the weight.
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// One element, fp32 moments; g: scaled gradient.  The divisor is 0 or at least
// the smallest normal number (the host checks eps).
__device__ __forceinline__ void update1(const AdamWArgs &a, float decay, float g, float &w, float &m,
                                        float &v) {
  m = __fadd_rn(__fmul_rn(m, a.beta1), __fmul_rn(g, a.omb1));
  v = __fadd_rn(__fmul_rn(v, a.beta2), __fmul_rn(__fmul_rn(g, g), a.omb2));
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  const float den = __fadd_rn(__fmul_rn(r, a.rs2), a.eps);
  w = __fadd_rn(__fmul_rn(w, decay), __fmul_rn(__fmul_rn(m, a.neg_c1), rcp_fast(den)));
}

// With 8-bit moments the instructions, not the bytes, bound the kernel: two
// elements per instruction (f32x2), sums of products as multiply-adds.  (The
// compiler fuses a packed multiply into a packed add whatever their rounding
// modifiers say, so the fused form is what is written.)
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
__device__ __forceinline__ Pair step_w(const AdamWArgs &a, float decay, Pair w, Pair m, Pair r) {
  float d0, d1;
  unpair(fma2(r, twice(a.rs2), twice(a.eps)), d0, d1);
  return fma2(w, twice(decay), mul2(mul2(m, twice(a.neg_c1)), pair(rcp_fast(d0), rcp_fast(d1))));
}
// The root as the state keeps it, rounded to nearest: the hardware's reciprocal
// root y of v and one Newton step r + (v - r^2) y / 2 from r = v y, whose residual
// the multiply-add leaves exact.  Small v are scaled by 2^64 to keep it so; 0, inf
// and nan are their own results.
__device__ __forceinline__ Pair root_near(Pair v) {
  float v0, v1;
  unpair(v, v0, v1);
  const bool s0 = v0 < 0x1p-64f, s1 = v1 < 0x1p-64f;
  const float x0 = s0 ? v0 * 0x1p64f : v0, x1 = s1 ? v1 * 0x1p64f : v1;
  float y0, y1, r0, r1;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y0) : "f"(x0));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y1) : "f"(x1));
  const Pair x = pair(x0, x1), y = pair(y0, y1);
  const Pair r = mul2(x, y);
  unpair(r, r0, r1);
  const Pair left = fma2(pair(-r0, -r1), r, x);
  unpair(fma2(left, mul2(y, twice(0.5f)), r), r0, r1);
  r0 = s0 ? r0 * 0x1p-32f : r0, r1 = s1 ? r1 * 0x1p-32f : r1;
  r0 = __float_as_uint(v0) - 1u < 0x7f7fffffu ? r0 : v0;
  r1 = __float_as_uint(v1) - 1u < 0x7f7fffffu ? r1 : v1;
  return pair(r0, r1);
}
// ---- 8-bit codes -----------------------------------------------------------------
// Multiply and xor-shift rounds; the multipliers are binary fractions of the
// golden ratio and of the roots of 2, 3 and 5.  Any well-mixed function would do.
constexpr unsigned kPlaceMul = 0x9E3779B1u, kHighMul = 0x3C6EF373u;
__host__ __device__ __forceinline__ unsigned mix_bits(unsigned x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
// Two code bytes (the low 16 bits) as numbers.
__device__ __forceinline__ Pair decode2(unsigned codes) {
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)codes));
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
  return pair(f.x, f.y);
}
__device__ __forceinline__ float scale_of(unsigned byte) {
  return byte == 0 ? 0x1p-127f : __uint_as_float(byte == 255 ? 0x7fc00000u : byte << 23);
}
// A block's scale byte and what to multiply its values by before `encode`, from
// the largest magnitude (as bits) of the block: the largest code lies in [128, 256),
// which leaves room to round up below 448.  255 (not a number): the block holds inf
// or nan.  The factor, 2^(7 - e - 120), is no float for the largest e: `big` says
// that the values are to be multiplied by 2^-100 first.
struct BlockScale {
  unsigned byte;
  bool big;
  float factor;
};
__device__ __forceinline__ BlockScale block_scale(unsigned max_bits) {
  unsigned e = max_bits >> 23;
  e = e < 8u ? 8u : e > 254u ? 254u : e;
  BlockScale b;
  b.byte = max_bits >= 0x7f800000u ? 255u : e - 7u;
  b.big = e > 140u;
  b.factor = __uint_as_float((141u - (b.big ? e - 100u : e)) << 23);
  return b;
}
// The code's magnitude in the low 7 bits of x times the block's factor: its bits lead
// the float's, subnormal ones included; 20 random bits below them are added: 16 of the
// hash, then a one that centres them, then zeros.
__device__ __forceinline__ unsigned encode(float scaled, unsigned bits16) {
  return (__float_as_uint(scaled) + ((bits16 << 4) | 8u)) >> 20;
}

// ---- one unit: eight elements per lane ---------------------------------------------
// Vector form: elements i + 4 lane .. + 3 and i + 128 + 4 lane .. + 3, so that
// every 16-byte access of the warp is one run of memory.
template <int RB, typename GT>
__device__ __forceinline__ void unit_vec(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                         float decay, size_t i, float *m_, float *v_) {
  const int lane = threadIdx.x & 31;
  float g[2][4];
  float4 w[2], m[2], v[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int o = 4 * lane + 128 * q;
    sum_grad4<RB, GT>(t.g, R, i + o, g[q]);
    w[q] = *reinterpret_cast<const float4 *>(t.w + i + o);
    m[q] = *reinterpret_cast<const float4 *>(m_ + o);
    v[q] = *reinterpret_cast<const float4 *>(v_ + o);
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int o = 4 * lane + 128 * q;
    float w4[4] = {w[q].x, w[q].y, w[q].z, w[q].w}, m4[4] = {m[q].x, m[q].y, m[q].z, m[q].w},
          v4[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) update1(a, decay, __fmul_rn(g[q][e], s), w4[e], m4[e], v4[e]);
    *reinterpret_cast<float4 *>(m_ + o) = make_float4(m4[0], m4[1], m4[2], m4[3]);
    *reinterpret_cast<float4 *>(v_ + o) = make_float4(v4[0], v4[1], v4[2], v4[3]);
    put_w4<RB>(t, R, a.lp_kind, i + o, w4);
  }
}
// Scalar form: nv (0..8) elements of this lane, STRIDE apart, four at a time.
template <int RB, typename GT, int STRIDE>
__device__ __forceinline__ void unit_scalar(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                            float decay, size_t i, int nv, float *m_, float *v_) {
#pragma unroll 1
  for (int q = 0; q < nv; q += 4, i += 4 * STRIDE, m_ += 4 * STRIDE, v_ += 4 * STRIDE) {
    float g[4], w[4], m[4], v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (q + e < nv) {
        g[e] = sum_grad1<RB, GT>(t.g, R, i + e * STRIDE);
        w[e] = t.w[i + e * STRIDE];
        m[e] = m_[e * STRIDE];
        v[e] = v_[e * STRIDE];
      }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (q + e < nv) {
        update1(a, decay, __fmul_rn(g[e], s), w[e], m[e], v[e]);
        m_[e * STRIDE] = m[e];
        v_[e * STRIDE] = v[e];
        put_w1<RB>(t, R, a.lp_kind, i + e * STRIDE, w[e]);
      }
  }
}

// 8-bit state.  VEC: elements as in unit_vec, codes read and written four at a
// time; else elements lane, lane + 32, ... below `avail`.
template <int RB, typename GT, bool VEC>
__device__ __forceinline__ void unit_quant(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                           float decay, size_t i, int avail, unsigned long long place,
                                           unsigned char *m_, unsigned char *r_,
                                           unsigned char *scale) {
  const int lane = threadIdx.x & 31;
  auto at = [&](int e) { return VEC ? 4 * lane + (e & 3) + 128 * (e >> 2) : lane + 32 * e; };
  auto have = [&](int e) { return VEC || at(e) < avail; };
  float g[8], w[8], m[8], r[8];
  unsigned mc[4], rc[4];  // two codes each
  const unsigned sc = *reinterpret_cast<const unsigned short *>(scale);
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int o = 4 * lane + 128 * q;
      float g4[4];
      sum_grad4<RB, GT>(t.g, R, i + o, g4);
      const float4 w4 = *reinterpret_cast<const float4 *>(t.w + i + o);
      const unsigned m4 = *reinterpret_cast<const unsigned *>(m_ + o);
      const unsigned r4 = *reinterpret_cast<const unsigned *>(r_ + o);
      mc[2 * q] = m4 & 0xffffu, mc[2 * q + 1] = m4 >> 16;
      rc[2 * q] = r4 & 0xffffu, rc[2 * q + 1] = r4 >> 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) g[4 * q + e] = g4[e];
      w[4 * q] = w4.x, w[4 * q + 1] = w4.y, w[4 * q + 2] = w4.z, w[4 * q + 3] = w4.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      g[e] = have(e) ? sum_grad1<RB, GT>(t.g, R, i + at(e)) : 0.f;
      w[e] = have(e) ? t.w[i + at(e)] : 0.f;
      const unsigned cm = have(e) ? m_[at(e)] : 0u, cr = have(e) ? r_[at(e)] : 0u;
      mc[e >> 1] = e & 1 ? mc[e >> 1] | (cm << 8) : cm;
      rc[e >> 1] = e & 1 ? rc[e >> 1] | (cr << 8) : cr;
    }
  }
  const float m_scale = scale_of(sc & 0xffu), r_scale = scale_of(sc >> 8);
  unsigned m_max = 0, r_max = 0;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    Pair pm = mul2(decode2(mc[e >> 1]), twice(m_scale));
    const Pair r0 = mul2(decode2(rc[e >> 1]), twice(r_scale));
    const Pair pg = mul2(pair(g[e], g[e + 1]), twice(s));
    pm = fma2(pm, twice(a.beta1), mul2(pg, twice(a.omb1)));
    const Pair pr = root_near(fma2(mul2(r0, r0), twice(a.beta2), mul2(mul2(pg, pg), twice(a.omb2))));
    unpair(step_w(a, decay, pair(w[e], w[e + 1]), pm, pr), w[e], w[e + 1]);
    unpair(pm, m[e], m[e + 1]);
    unpair(pr, r[e], r[e + 1]);
#pragma unroll
    for (int k = e; k < e + 2; ++k)
      if (have(k)) {
        m_max = max(m_max, __float_as_uint(m[k]) & 0x7fffffffu);
        r_max = max(r_max, __float_as_uint(r[k]) & 0x7fffffffu);
      }
  }
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float w4[4] = {w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
      put_w4<RB>(t, R, a.lp_kind, i + 4 * lane + 128 * q, w4);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (have(e)) put_w1<RB>(t, R, a.lp_kind, i + at(e), w[e]);
  }
  const BlockScale mb = block_scale(__reduce_max_sync(0xffffffffu, m_max));
  const BlockScale rb = block_scale(__reduce_max_sync(0xffffffffu, r_max));
  if (mb.big) {
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] *= 0x1p-100f;
  }
  if (rb.big) {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = r[e] > 0.f ? fmaxf(r[e] * 0x1p-100f, 0x1p-126f) : r[e];  // stays positive
  }
  // place * multiplier + key, stepped from element to element
  const unsigned first = (unsigned)(place + at(0)) * kPlaceMul + (unsigned)((place + at(0)) >> 32) * kHighMul + a.key;
  unsigned cm[8], cr[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float y[2], z[2];
    unpair(mul2(pair(fabsf(m[e]), fabsf(m[e + 1])), twice(mb.factor)), y[0], y[1]);
    unpair(mul2(pair(r[e], r[e + 1]), twice(rb.factor)), z[0], z[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const unsigned bits = mix_bits(first + (unsigned)(at(e + k) - at(0)) * kPlaceMul);
      cm[e + k] = encode(y[k], bits & 0xffffu) | ((__float_as_uint(m[e + k]) >> 24) & 0x80u);
      const unsigned c = encode(z[k], bits >> 16);
      cr[e + k] = r[e + k] > 0.f ? max(c, 1u) : c;
    }
  }
  if (mb.byte == 255u || rb.byte == 255u) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (mb.byte == 255u) cm[e] = 0u;
      if (rb.byte == 255u) cr[e] = 0u;
    }
  }
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int o = 4 * lane + 128 * q;
      *reinterpret_cast<unsigned *>(m_ + o) =
          cm[4 * q] | (cm[4 * q + 1] << 8) | (cm[4 * q + 2] << 16) | (cm[4 * q + 3] << 24);
      *reinterpret_cast<unsigned *>(r_ + o) =
          cr[4 * q] | (cr[4 * q + 1] << 8) | (cr[4 * q + 2] << 16) | (cr[4 * q + 3] << 24);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (have(e)) m_[at(e)] = (unsigned char)cm[e], r_[at(e)] = (unsigned char)cr[e];
  }
  if (lane == 0) *reinterpret_cast<unsigned short *>(scale) = (unsigned short)(mb.byte | (rb.byte << 8));
}

// A unit inside one tensor: `avail` (1..256) elements from element i of the
// tensor and group e of the state on.
template <int RB, bool QUANT, typename GT>
__device__ __forceinline__ void unit_inside(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                            float decay, size_t i, int avail, bool vec, size_t e) {
  const int lane = threadIdx.x & 31;
  if constexpr (QUANT) {
    unsigned char *m = (unsigned char *)a.m + e * kListGroup, *r = (unsigned char *)a.v + e * kListGroup;
    unsigned char *scale = a.scale + e / kListUnitGroups * 2;
    const unsigned long long place = a.flat0 + e * kListGroup;
    if (vec && avail == kListUnit)
      unit_quant<RB, GT, true>(t, a, R, s, decay, i, avail, place, m, r, scale);
    else
      unit_quant<RB, GT, false>(t, a, R, s, decay, i, avail, place, m, r, scale);
  } else {
    float *m = (float *)a.m + e * kListGroup, *v = (float *)a.v + e * kListGroup;
    if (vec && avail == kListUnit)
      unit_vec<RB, GT>(t, a, R, s, decay, i, m, v);
    else
      unit_scalar<RB, GT, 32>(t, a, R, s, decay, i + lane, avail > lane ? (avail - lane + 31) / 32 : 0,
                              m + lane, v + lane);
  }
}

// 16-byte accesses of fp32 weights and gradients, 8-byte ones of 16-bit types.
template <typename GT> __device__ __forceinline__ bool vec_ok(const void *g, const float *w, const void *lp) {
  return ((uintptr_t)g & (sizeof(GT) == 4 ? 15u : 7u)) == 0 && ((uintptr_t)w & 15u) == 0 &&
         ((uintptr_t)lp & 7u) == 0;
}

// ---- the kernels -----------------------------------------------------------------
template <bool QUANT, typename GT, int CAP>
__global__ void __launch_bounds__(COCO_ADAMW_THREADS, 2)
    adamw_kernel(const __grid_constant__ ListTable<CAP> tab, const __grid_constant__ AdamWArgs a) {
  __shared__ unsigned s_off[CAP + 1];
  for (int k = threadIdx.x; k <= a.n; k += blockDim.x) s_off[k] = tab.off[k];
  float s = a.grad_scale;
  if (a.norm) {
    if (!is_finite(a.norm[0])) return;  // the gradients are not usable: the step is skipped
    s = __fmul_rn(a.norm[1], s);
  }
  __syncthreads();
  const int n = a.n, lane = threadIdx.x & 31;
  const unsigned total = s_off[n];
  const unsigned units = (total + kListUnitGroups - 1) / kListUnitGroups;
  const unsigned nw = blockDim.x >> 5;
  unsigned begin = 1, end = 0;  // the tensor at hand
  unsigned missing = 0;
  View<1> t = {};
  float decay = 1.f;
  bool vec = false;
  for (unsigned u = blockIdx.x * nw + (threadIdx.x >> 5); u < units; u += gridDim.x * nw) {
    const unsigned e = u * kListUnitGroups;
    if (e < begin || e >= end) {
      const int k = find_tensor(s_off, n, e);
      begin = s_off[k], end = s_off[k + 1];
      missing = tab.missing[k];
      t.g[0] = tab.g[k], t.w = tab.w[k], t.lp = tab.lp[k];
      decay = tab.decays[k] ? a.decay : 1.f;
      vec = a.state_aligned && vec_ok<GT>(t.g[0], t.w, t.lp);
    }
    if (QUANT || end - e >= kListUnitGroups || end == total) {
      const size_t left = (size_t)(end - e) * kListGroup - missing;
      unit_inside<1, QUANT, GT>(t, a, 1, s, decay, (size_t)(e - begin) * kListGroup,
                                left < kListUnit ? (int)left : kListUnit, vec, e);
    } else {
      // several tensors in one unit: every lane looks up its own group
      const unsigned el = e + lane;
      if (el < total) {
        const int k = bisect(0, n - 1, el, [&](int x) { return s_off[x]; });
        View<1> tl;
        tl.g[0] = tab.g[k], tl.w = tab.w[k], tl.lp = tab.lp[k];
        const int nv = el + 1 < s_off[k + 1] ? kListGroup : kListGroup - tab.missing[k];
        unit_scalar<1, GT, 1>(tl, a, 1, s, tab.decays[k] ? a.decay : 1.f,
                              (size_t)(el - s_off[k]) * kListGroup, nv,
                              (float *)a.m + (size_t)el * kListGroup, (float *)a.v + (size_t)el * kListGroup);
      }
      __syncwarp();
    }
  }
}

template <bool QUANT, typename GT, int RB>
__global__ void __launch_bounds__(COCO_ADAMW_PEER_THREADS, 2)
    adamw_peer_kernel(const __grid_constant__ PeerArgs pa, const __grid_constant__ AdamWArgs a0) {
  __shared__ int s_ok;
  const PeerRank &pr = pa.ranks[blockIdx.y];
  const int R = pa.world, lane = threadIdx.x & 31;
  const bool started = list_start_barrier(pr, pa, &s_ok);
  AdamWArgs a = a0;
  a.m = pr.m, a.v = pr.v, a.scale = pr.scale, a.flat0 = pr.flat0;
  float s = a.grad_scale;
  bool ok = started;
  if (pr.norm) {
    if (!is_finite(pr.norm[0])) ok = false;  // the same value on every rank
    s = __fmul_rn(pr.norm[1], s);
  }
  const PeerPiece *pieces = pr.pieces;
  const int n = pr.n;
  const unsigned units = ok ? (pr.groups + kListUnitGroups - 1) / kListUnitGroups : 0;
  const unsigned nw = blockDim.x >> 5;
  for (unsigned u = blockIdx.x * nw + (threadIdx.x >> 5); u < units; u += gridDim.x * nw) {
    const unsigned e = u * kListUnitGroups;
    const int k = bisect(0, n - 1, e, [&](int x) { return pieces[x].off; });
    const PeerPiece &pc = pieces[k];
    if (QUANT || pc.end - e >= kListUnitGroups || pc.end == pr.groups) {
      const size_t done = (size_t)(e - pc.off) * kListGroup, left = (size_t)pc.len - done;
      const View<RB> t = {pc.g, pc.out, pc.w};
      unit_inside<RB, QUANT, GT>(t, a, R, s, pc.decays ? a.decay : 1.f, (size_t)pc.begin + done,
                                 left < kListUnit ? (int)left : kListUnit,
                                 pc.aligned16 && pr.state_aligned, e);
    } else {
      const unsigned el = e + lane;
      if (el < pr.groups) {
        const PeerPiece &pl = pieces[bisect(k, n - 1, el, [&](int x) { return pieces[x].off; })];
        const size_t done = (size_t)(el - pl.off) * kListGroup, left = (size_t)pl.len - done;
        const View<RB> t = {pl.g, pl.out, pl.w};
        unit_scalar<RB, GT, 1>(t, a, R, s, pl.decays ? a.decay : 1.f, (size_t)pl.begin + done,
                               left < kListGroup ? (int)left : kListGroup,
                               (float *)a.m + (size_t)el * kListGroup,
                               (float *)a.v + (size_t)el * kListGroup);
      }
      __syncwarp();
    }
  }
  list_end_barrier(pr, pa, started);
}

// ---- launches --------------------------------------------------------------------
template <int CAP> using Kernel = void (*)(const ListTable<CAP>, const AdamWArgs);
template <int CAP> Kernel<CAP> pick(bool quant, cocoDataType_t g) {
  switch (g) {
    case cocoFloat32: return quant ? adamw_kernel<true, float, CAP> : adamw_kernel<false, float, CAP>;
    case cocoFloat16: return quant ? adamw_kernel<true, __half, CAP> : adamw_kernel<false, __half, CAP>;
    case cocoBfloat16:
      return quant ? adamw_kernel<true, __nv_bfloat16, CAP> : adamw_kernel<false, __nv_bfloat16, CAP>;
  }
  return nullptr;
}
typedef void (*PeerKernel)(const PeerArgs, const AdamWArgs);
template <bool QUANT, typename GT> PeerKernel pick_world(int world) {
  return world <= 2 ? adamw_peer_kernel<QUANT, GT, 2>
         : world <= 4 ? adamw_peer_kernel<QUANT, GT, 4> : adamw_peer_kernel<QUANT, GT, 8>;
}
PeerKernel pick_peer(bool quant, cocoDataType_t g, int world) {
  switch (g) {
    case cocoFloat32: return quant ? pick_world<true, float>(world) : pick_world<false, float>(world);
    case cocoFloat16: return quant ? pick_world<true, __half>(world) : pick_world<false, __half>(world);
    case cocoBfloat16:
      return quant ? pick_world<true, __nv_bfloat16>(world) : pick_world<false, __nv_bfloat16>(world);
  }
  return nullptr;
}

}  // namespace

unsigned adamw_rounding_key(uint64_t seed, int step) {
  return mix_bits(mix_bits((unsigned)seed) + (unsigned)(seed >> 32) * kHighMul +
                  (unsigned)step * kPlaceMul);
}

int adamw_threads(bool, cocoDataType_t) { return COCO_ADAMW_THREADS; }
int adamw_ctas_per_sm(bool, cocoDataType_t) { return 2; }

template <int CAP>
cudaError_t launch_adamw(bool quant, cocoDataType_t g_type, const ListTable<CAP> &table,
                         const AdamWArgs &args, int ctas, cudaStream_t stream) {
  const Kernel<CAP> k = pick<CAP>(quant, g_type);
  if (!k) return cudaErrorInvalidValue;
  void *params[] = {(void *)&table, (void *)&args};
  return cudaLaunchKernel((const void *)k, dim3(ctas), dim3(COCO_ADAMW_THREADS), params, 0, stream);
}
template cudaError_t launch_adamw<kListCapSmall>(bool, cocoDataType_t, const ListTable<kListCapSmall> &,
                                                 const AdamWArgs &, int, cudaStream_t);
template cudaError_t launch_adamw<kListCapLarge>(bool, cocoDataType_t, const ListTable<kListCapLarge> &,
                                                 const AdamWArgs &, int, cudaStream_t);

cudaError_t launch_adamw_peers(bool quant, cocoDataType_t g_type, const PeerArgs &peers,
                               const AdamWArgs &args, const ListLaunch &cfg, cudaStream_t stream) {
  const PeerKernel k = pick_peer(quant, g_type, peers.world);
  if (!k) return cudaErrorInvalidValue;
  void *params[] = {(void *)&peers, (void *)&args};
  const dim3 grid(cfg.ctas, cfg.nvirt);
  if (cfg.cooperative)
    return cudaLaunchCooperativeKernel((const void *)k, grid, dim3(cfg.threads), params, 0, stream);
  return cudaLaunchKernel((const void *)k, grid, dim3(cfg.threads), params, 0, stream);
}
cudaError_t adamw_peers_occupancy(bool quant, cocoDataType_t g_type, int world, int threads,
                                  int *ctas_per_sm) {
  const PeerKernel k = pick_peer(quant, g_type, world);
  if (!k) return cudaErrorInvalidValue;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(ctas_per_sm, (const void *)k, threads, 0);
}

}  // namespace coco
