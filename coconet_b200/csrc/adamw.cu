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
// What bounds it: HBM with fp32 moments, instruction issue with 8-bit ones.  One pass,
// every byte moved once; nothing is reused.
#include "list_device.cuh"
#include "pair_math.cuh"

#include <atomic>

// Threads of a CTA where an SM holds two, and tiles in flight of the staged kernels.
#ifndef COCO_ADAMW_THREADS
#define COCO_ADAMW_THREADS 352
#endif
#ifndef COCO_ADAMW_PACKED_THREADS
#define COCO_ADAMW_PACKED_THREADS 320
#endif
#ifndef COCO_ADAMW_QUANT_THREADS
#define COCO_ADAMW_QUANT_THREADS 384
#endif
#ifndef COCO_ADAMW_STAGES
#define COCO_ADAMW_STAGES 3
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

// Two values as 16-bit numbers in one word.
__device__ __forceinline__ unsigned lp_pair(int kind, float x, float y) {
  if (kind == kLpF16) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const unsigned *>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const unsigned *>(&h);
}
template <int RB, typename Index> __device__ __forceinline__ void put_lp4(const View<RB> &v, int R, int kind, Index i,
                                                          const float (&x)[4]) {
  uint2 q;
  if (kind == kLpF16) q = make_uint2(lp_pair(kLpF16, x[0], x[1]), lp_pair(kLpF16, x[2], x[3]));
  else q = make_uint2(lp_pair(kLpBf16, x[0], x[1]), lp_pair(kLpBf16, x[2], x[3]));
  if constexpr (RB == 1) {
    *reinterpret_cast<uint2 *>((unsigned short *)v.lp + i) = q;
  } else {
#pragma unroll
    for (int p = 0; p < RB; ++p)
      if (RB == 2 || p < R) st_sys_8((unsigned short *)v.out[p] + i, q);
  }
}
template <int RB, typename Index> __device__ __forceinline__ void put_lp1(const View<RB> &v, int R, int kind, Index i,
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
template <int RB, typename Index> __device__ __forceinline__ void put_w4(const View<RB> &v, int R, int kind, Index i,
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
template <int RB, typename Index> __device__ __forceinline__ void put_w1(const View<RB> &v, int R, int kind, Index i,
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
// from overlapping (74 us against 60 for 12.6 M elements), and the update they
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


// ---- 8-bit codes -----------------------------------------------------------------
// With 8-bit moments the instructions, not the bytes, bound the kernel (156 per
// element in the first form, 66 now; 88 would fill every issue slot at the copy rate):
// two elements per instruction (f32x2) where there is a form for it.

// Multiply and xor-shift rounds; the multipliers are binary fractions of the
// golden ratio and of the roots of 2, 3 and 5.  Any well-mixed function would do.
constexpr unsigned kPlaceMul = 0x9E3779B1u, kHighMul = 0x3C6EF373u;
__host__ __device__ __forceinline__ unsigned mix_most(unsigned x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  return (x ^ (x >> 15)) * 0xBB67AE85u;
}
__host__ __device__ __forceinline__ unsigned mix_bits(unsigned x) {
  x = mix_most(x);
  return x ^ (x >> 16);
}
// Two code bytes (the low 16 bits) as numbers.
__device__ __forceinline__ Pair decode2(unsigned codes) {
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)codes));
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
  return pair(f.x, f.y);
}
// Two scale bytes (the low 16 bits) as numbers.
__device__ __forceinline__ void scales_of(unsigned bytes, float &lo, float &hi) {
  unsigned b;
  asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(b) : "h"((unsigned short)bytes));
  lo = __uint_as_float(b << 16), hi = __uint_as_float(b & 0xffff0000u);
}
// A block's scale byte and what to multiply its values by before they are rounded,
// from the largest magnitude (as bits) of the block: the largest code lies in
// [128, 256), which leaves room to round up below 448.  255 (not a number): the block
// holds inf or nan.  The product of the two factors, 2^(14 - e) for a largest exponent
// field of e, is no float for the largest e; the first leaves the largest value in
// [2^7, 2^8) and costs nothing but what is far below the smallest code.
struct BlockScale {
  unsigned byte;
  float before, factor;
};
__device__ __forceinline__ BlockScale block_scale(unsigned max_bits) {
  unsigned e = max_bits >> 23;
  e = e < 8u ? 8u : e > 254u ? 254u : e;
  return {max_bits >= 0x7f800000u ? 255u : e - 7u, __uint_as_float((261u - e) << 23), 0x1p-120f};
}
// The same where the largest magnitude lies in [2^-119, 2^14): one factor does.
__device__ __forceinline__ bool is_usual(unsigned max_bits) { return max_bits - 0x04000000u < 0x46800000u - 0x04000000u; }
__device__ __forceinline__ BlockScale usual_scale(unsigned max_bits) {
  return {(max_bits >> 23) - 7u, 1.f, __uint_as_float(0x46800000u - (max_bits & 0x7f800000u))};
}
// x times the block's factor has the code's 7 magnitude bits in bits 20..26, subnormal
// codes included; adding 20 random bits (16 of the hash, a one that centres them, zeros)
// and cutting 20 off rounds up with the probability of the part cut off.  Here both are
// 4 bits further up, so that a multiply-add leaves the code in the top byte.  The hash's
// low half (m) and high half (r) in place, from the hash before its last x ^ (x >> 16):
__device__ __forceinline__ void rounding(unsigned x, unsigned &for_m, unsigned &for_r) {
  for_r = __byte_perm(x, 0x80u, 0x5324);                       // {0x80, x2, x3, 0}
  for_m = __byte_perm(x, 0x80u, 0x5104) ^ for_r ^ 0x80u;       // {0x80, x0 ^ x2, x1 ^ x3, 0}
}
__device__ __forceinline__ unsigned code_r(float scaled, unsigned random) {
  return __float_as_uint(scaled) * 16u + random;
}
__device__ __forceinline__ unsigned code_m(float scaled, unsigned random) {  // with its sign
  return (code_r(scaled, random) & 0x7fffffffu) | (__float_as_uint(scaled) & 0x80000000u);
}
__device__ __forceinline__ unsigned top_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
// Largest magnitude of three, nan if one is.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// ---- one unit: eight elements per lane ---------------------------------------------
// Vector form: elements i + 4 lane .. + 3 and i + 128 + 4 lane .. + 3, so that
// every 16-byte access of the warp is one run of memory.
// im: of the state.
template <int RB, typename GT, typename Index>
__device__ __forceinline__ void unit_vec(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                         float decay, Index i, float *m_, float *v_, Index im) {
  const unsigned lane = threadIdx.x & 31;
  float g[2][4];
  float4 w[2], m[2], v[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const Index o = 4 * lane + 128 * q;
    sum_grad4<RB, GT>(t.g, R, i + o, g[q]);
    w[q] = *reinterpret_cast<const float4 *>(t.w + (i + o));
    m[q] = *reinterpret_cast<const float4 *>(m_ + (im + o));
    v[q] = *reinterpret_cast<const float4 *>(v_ + (im + o));
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const Index o = 4 * lane + 128 * q;
    float w4[4] = {w[q].x, w[q].y, w[q].z, w[q].w}, m4[4] = {m[q].x, m[q].y, m[q].z, m[q].w},
          v4[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) update1(a, decay, __fmul_rn(g[q][e], s), w4[e], m4[e], v4[e]);
    *reinterpret_cast<float4 *>(m_ + (im + o)) = make_float4(m4[0], m4[1], m4[2], m4[3]);
    *reinterpret_cast<float4 *>(v_ + (im + o)) = make_float4(v4[0], v4[1], v4[2], v4[3]);
    put_w4<RB>(t, R, a.lp_kind, i + o, w4);
  }
}
// Scalar form: nv (0..8) elements of this lane, STRIDE apart, four at a time.
template <int RB, typename GT, int STRIDE, typename Index>
__device__ __forceinline__ void unit_scalar(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                            float decay, Index i, int nv, float *m_, float *v_, Index im) {
#pragma unroll 1
  for (int q = 0; q < nv; q += 4, i += 4 * STRIDE, im += 4 * STRIDE) {
    float g[4], w[4], m[4], v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (q + e < nv) {
        g[e] = sum_grad1<RB, GT>(t.g, R, i + e * STRIDE);
        w[e] = t.w[i + e * STRIDE];
        m[e] = m_[im + e * STRIDE];
        v[e] = v_[im + e * STRIDE];
      }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (q + e < nv) {
        update1(a, decay, __fmul_rn(g[e], s), w[e], m[e], v[e]);
        m_[im + e * STRIDE] = m[e];
        v_[im + e * STRIDE] = v[e];
        put_w1<RB>(t, R, a.lp_kind, i + e * STRIDE, w[e]);
      }
  }
}

// 8-bit state.  VEC: elements as in unit_vec, codes read and written four at a
// time; else elements lane, lane + 32, ... below `avail`.
template <bool VEC> __device__ __forceinline__ int quant_at(int e) {
  const int lane = threadIdx.x & 31;
  return VEC ? 4 * lane + (e & 3) + 128 * (e >> 2) : lane + 32 * e;
}
struct QuantUnit {      // what is read of a unit
  float g[8], w[8];
  unsigned m[2], r[2];  // four codes each, in the order of the elements
  unsigned scale;
};
template <int RB, typename GT, bool VEC, typename Index>
__device__ __forceinline__ void quant_load(QuantUnit &x, const View<RB> &t, int R, Index i, int avail,
                                           const unsigned char *m_, const unsigned char *r_, Index im,
                                           const unsigned char *scale) {
  x.scale = *reinterpret_cast<const unsigned short *>(scale);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    if constexpr (VEC) {
      const Index o = quant_at<true>(4 * q);
      float g4[4];
      sum_grad4<RB, GT>(t.g, R, i + o, g4);
      const float4 w4 = *reinterpret_cast<const float4 *>(t.w + (i + o));
      x.m[q] = *reinterpret_cast<const unsigned *>(m_ + (im + o));
      x.r[q] = *reinterpret_cast<const unsigned *>(r_ + (im + o));
#pragma unroll
      for (int e = 0; e < 4; ++e) x.g[4 * q + e] = g4[e];
      x.w[4 * q] = w4.x, x.w[4 * q + 1] = w4.y, x.w[4 * q + 2] = w4.z, x.w[4 * q + 3] = w4.w;
    } else {
      unsigned cm[4], cr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Index o = quant_at<false>(4 * q + e);
        const bool have = (int)o < avail;
        x.g[4 * q + e] = have ? sum_grad1<RB, GT>(t.g, R, i + o) : 0.f;
        x.w[4 * q + e] = have ? t.w[i + o] : 0.f;
        cm[e] = have ? m_[im + o] : 0u, cr[e] = have ? r_[im + o] : 0u;
      }
      auto word = [](const unsigned (&c)[4]) {
        return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
      };
      x.m[q] = word(cm), x.r[q] = word(cr);
    }
  }
}
// What the hash of an element mixes; it grows by kPlaceMul from one to the next (a unit
// does not cross a multiple of 2^32).
__device__ __forceinline__ unsigned hash_start(unsigned long long place, unsigned key) {
  return (unsigned)place * kPlaceMul + (unsigned)(place >> 32) * kHighMul + key;
}
// From what was read of a unit to its new weights (x.w, handed to put_w as soon as
// they are there), codes and scale bytes.  Elements that do not exist are zeros in x.
// first: hash_start of this lane's first element.
template <bool VEC, typename PutW>
__device__ __forceinline__ void quant_step(QuantUnit &x, const AdamWArgs &a, float s, float decay,
                                           unsigned first, PutW put_w) {
  float m_scale, r_scale;
  scales_of(x.scale, m_scale, r_scale);
  float m[8], r[8];  // r: -v, then -sqrt(v)
  float m_max = 0.f, v_max = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const int q = e >> 2, half = e & 2 ? 16 : 0;
    const Pair pm = mul2(decode2(x.m[q] >> half), twice(m_scale));
    const Pair r0 = mul2(decode2(x.r[q] >> half), twice(r_scale));
    const Pair g = mul2(pair(x.g[e], x.g[e + 1]), twice(s));
    sum2(mul2(pm, twice(a.beta1)), mul2(g, twice(a.omb1)), m[e], m[e + 1]);
    sum2(mul2(mul2(r0, r0), twice(a.neg_beta2)), mul2(mul2(g, g), twice(a.neg_omb2)), r[e], r[e + 1]);
    m_max = max_abs(m_max, m[e], m[e + 1]);
    v_max = max_abs(v_max, r[e], r[e + 1]);
  }
  bool rare = !(v_max < __uint_as_float(0x7f800000u));  // inf or nan
  // no v is below 2^-100 if no root was 0 and the scale is 2^-40 or more (and beta2 1/4)
  auto has_zero = [](unsigned codes) { return ((codes & 0x7f7f7f7fu) + 0x7f7f7f7fu & 0x80808080u) != 0x80808080u; };
  if (has_zero(x.r[0]) || has_zero(x.r[1]) || !(r_scale >= 0x1p-40f) || a.beta2 < 0.25f) {
    unsigned low = 0xffffffffu;  // distance above -0, the smallest of those that are not 0
#pragma unroll
    for (int e = 0; e < 8; ++e) low = min(low, __float_as_uint(r[e]) - 0x80000001u);
    rare = rare || low < 0x0d800000u;
  }
  if (rare) {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = neg_root_any(r[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) unpair(neg_root(pair(r[e], r[e + 1])), r[e], r[e + 1]);
  }
  float r_max = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float d0, d1;
    unpair(fma2(pair(r[e], r[e + 1]), twice(a.neg_rs2), twice(a.eps)), d0, d1);
    unpair(fma2(pair(x.w[e], x.w[e + 1]), twice(decay),
                mul2(mul2(pair(m[e], m[e + 1]), twice(a.neg_c1)), pair(rcp_fast(d0), rcp_fast(d1)))),
           x.w[e], x.w[e + 1]);
    r_max = max_abs(r_max, r[e], r[e + 1]);
  }
  put_w();
  const unsigned m_top = __reduce_max_sync(0xffffffffu, __float_as_uint(m_max) & 0x7fffffffu);
  const unsigned r_top = __reduce_max_sync(0xffffffffu, __float_as_uint(r_max) & 0x7fffffffu);
  BlockScale mb = usual_scale(m_top), rb = usual_scale(r_top);
  const bool unusual = !is_usual(m_top) || !is_usual(r_top);
  if (unusual) {
    mb = block_scale(m_top), rb = block_scale(r_top);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m[e] *= mb.before;
      r[e] = r[e] < 0.f ? fminf(r[e] * rb.before, -0x1p-126f) : r[e];  // stays below 0
    }
  }
  x.scale = mb.byte | (rb.byte << 8);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    unsigned cm[4], cr[4];
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const int k = 4 * q + e;
      float y[2], z[2];
      unpair(mul2(pair(m[k], m[k + 1]), twice(mb.factor)), y[0], y[1]);
      unpair(mul2(pair(r[k], r[k + 1]), twice(-rb.factor)), z[0], z[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        unsigned for_m, for_r;
        rounding(mix_most(first + (unsigned)(quant_at<VEC>(k + j) - quant_at<VEC>(0)) * kPlaceMul), for_m, for_r);
        cm[e + j] = code_m(y[j], for_m);
        cr[e + j] = code_r(z[j], for_r);
      }
    }
    unsigned mw = top_bytes(cm[0], cm[1], cm[2], cm[3]), rw = top_bytes(cr[0], cr[1], cr[2], cr[3]);
    const unsigned zero = ~(rw + 0x7f7f7f7fu) & 0x80808080u;  // roots rounded to 0: 1 unless they are 0,
    if (zero != 0u)                                           // which has lost its sign
      rw |= (zero & top_bytes(__float_as_uint(r[4 * q]), __float_as_uint(r[4 * q + 1]), __float_as_uint(r[4 * q + 2]),
                              __float_as_uint(r[4 * q + 3]))) >> 7;
    x.m[q] = mw, x.r[q] = rw;
  }
  if (unusual) {
    if (mb.byte == 255u) x.m[0] = x.m[1] = 0u;
    if (rb.byte == 255u) x.r[0] = x.r[1] = 0u;
  }
}
__device__ __forceinline__ void put_scale(const QuantUnit &x, unsigned char *scale) {
  if ((threadIdx.x & 31) == 0) *reinterpret_cast<unsigned short *>(scale) = (unsigned short)x.scale;
}
template <int RB, typename GT, bool VEC, typename Index>
__device__ __forceinline__ void unit_quant(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                           float decay, Index i, int avail, unsigned long long place,
                                           unsigned char *m_, unsigned char *r_, Index im,
                                           unsigned char *scale) {
  QuantUnit x;
  quant_load<RB, GT, VEC>(x, t, R, i, avail, m_, r_, im, scale);
  quant_step<VEC>(x, a, s, decay, hash_start(place + quant_at<VEC>(0), a.key), [&] {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if constexpr (VEC) {
        const float w4[4] = {x.w[4 * q], x.w[4 * q + 1], x.w[4 * q + 2], x.w[4 * q + 3]};
        put_w4<RB>(t, R, a.lp_kind, i + (Index)quant_at<true>(4 * q), w4);
      } else {
#pragma unroll
        for (int e = 4 * q; e < 4 * q + 4; ++e)
          if (quant_at<false>(e) < avail) put_w1<RB>(t, R, a.lp_kind, i + (Index)quant_at<false>(e), x.w[e]);
      }
    }
  });
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    if constexpr (VEC) {
      *reinterpret_cast<unsigned *>(m_ + (im + quant_at<true>(4 * q))) = x.m[q];
      *reinterpret_cast<unsigned *>(r_ + (im + quant_at<true>(4 * q))) = x.r[q];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Index o = quant_at<false>(4 * q + e);
        if ((int)o < avail) m_[im + o] = (unsigned char)(x.m[q] >> (8 * e)), r_[im + o] = (unsigned char)(x.r[q] >> (8 * e));
      }
    }
  }
  put_scale(x, scale);
}

// A unit inside one tensor: `avail` (1..256) elements from element i of the
// tensor and group e of the state on.
template <int RB, bool QUANT, typename GT>
__device__ __forceinline__ void unit_inside(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                            float decay, size_t i, int avail, bool vec, size_t e) {
  const int lane = threadIdx.x & 31;
  const size_t im = e * kListGroup;
  if constexpr (QUANT) {
    unsigned char *m = (unsigned char *)a.m, *r = (unsigned char *)a.v;
    unsigned char *scale = a.scale + e / kListUnitGroups * 2;
    if (vec && avail == kListUnit)
      unit_quant<RB, GT, true>(t, a, R, s, decay, i, avail, a.flat0 + im, m, r, im, scale);
    else
      unit_quant<RB, GT, false>(t, a, R, s, decay, i, avail, a.flat0 + im, m, r, im, scale);
  } else {
    float *m = (float *)a.m, *v = (float *)a.v;
    if (vec && avail == kListUnit)
      unit_vec<RB, GT>(t, a, R, s, decay, i, m, v, im);
    else
      unit_scalar<RB, GT, 32>(t, a, R, s, decay, i + lane, avail > lane ? (avail - lane + 31) / 32 : 0, m, v,
                                     im + lane);
  }
}

// ---- the kernels -----------------------------------------------------------------
// A unit that holds several tensors or the end of one, by one warp.  Kept apart from the
// kernels' loops, whose registers decide their speed.
template <bool QUANT, typename GT, int CAP>
__device__ __noinline__ void unit_general(const ListTable<CAP> *tab, const AdamWArgs &a, const unsigned *s_off,
                                          float s, unsigned unit) {
  const int n = a.n, lane = threadIdx.x & 31;
  const unsigned total = s_off[n], e = unit * kListUnitGroups;
  if (e >= total) return;
  const int k = find_tensor(s_off, n, e);
  const unsigned end = s_off[k + 1];
  View<1> t;
  if (QUANT || end - e >= kListUnitGroups || end == total) {
    t.g[0] = tab->g[k], t.w = tab->w[k], t.lp = tab->lp[k];
    const size_t left = (size_t)(end - e) * kListGroup - tab->missing[k];
    unit_inside<1, QUANT, GT>(t, a, 1, s, tab->flags[k] & kListDecays ? a.decay : 1.f,
                              (size_t)(e - s_off[k]) * kListGroup, left < kListUnit ? (int)left : kListUnit,
                              (tab->flags[k] & kListAligned) != 0, e);
  } else {
    // several tensors in one unit: every lane looks up its own group
    const unsigned el = e + lane;
    if (el >= total) return;
    const int kl = bisect(k, n - 1, el, [&](int x) { return s_off[x]; });
    t.g[0] = tab->g[kl], t.w = tab->w[kl], t.lp = tab->lp[kl];
    const int nv = el + 1 < s_off[kl + 1] ? kListGroup : kListGroup - tab->missing[kl];
    const size_t im = (size_t)el * kListGroup;
    unit_scalar<1, GT, 1>(t, a, 1, s, tab->flags[kl] & kListDecays ? a.decay : 1.f,
                          (size_t)(el - s_off[kl]) * kListGroup, nv, (float *)a.m, (float *)a.v, im);
  }
}

// fp32 moments, tensors that are aligned.  A CTA takes tiles of one unit per warp.
// Where a tile lies in one tensor, which and where is the same for all threads: it costs
// no vector registers, and an element's address is a common base and a 32-bit offset.
// HBM-bound: 336 M elements in 398 tensors 1.46 ms with fp32 gradients, 1.49 ms with bf16
// gradients and copies (28 bytes per element: 0.986 and 0.966 of the measured copy rate).
// Eleven warps: with bf16 gradients 8, 10, 12 and 16 warps measured 1.53, 1.56, 1.51 and
// 1.64 ms.
template <typename GT, int CAP>
__global__ void __launch_bounds__(COCO_ADAMW_THREADS, 2)
    adamw_kernel(const __grid_constant__ ListTable<CAP> tab, const __grid_constant__ AdamWArgs a) {
  __shared__ unsigned s_off[CAP + 1];
  const ListTable<CAP> *tp = &tab;
  hide(tp);  // for lookups that differ from thread to thread
  copy_offsets(s_off, tp->off, a.n);
  float s = a.grad_scale;
  if (a.norm) {
    if (!is_finite(a.norm[0])) return;  // the gradients are not usable: the step is skipped
    s = __fmul_rn(a.norm[1], s);
  }
  __syncthreads();
  constexpr unsigned kTile = COCO_ADAMW_THREADS / 32 * kListUnitGroups;
  const int n = a.n;
  const unsigned tiles = (tab.off[n] + kTile - 1) / kTile;
  const unsigned mine = (threadIdx.x & ~31u) * 8;  // elements before this warp's in the tile
  int k = 0;  // the tensor in which the tile begins
  for (unsigned tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const unsigned e = tile * kTile;
    int jump = 1;  // it lies at or behind the last one: double the steps, then halve them
    while (k + jump < n && tab.off[k + jump] <= e) k += jump, jump *= 2;
    for (; jump > 0; jump >>= 1)
      if (k + jump < n && tab.off[k + jump] <= e) k += jump;
    // the last group of a tensor may be short
    if (e + kTile < tab.off[k + 1] + (tab.missing[k] == 0) && (tab.flags[k] & kListAligned)) {
      const size_t i = (size_t)(e - tab.off[k]) * kListGroup, im = (size_t)e * kListGroup;
      View<1> t;
      t.g[0] = (const GT *)tab.g[k] + i;
      t.w = tab.w[k] + i;
      t.lp = (unsigned short *)tab.lp[k] + i;
      unit_vec<1, GT>(t, a, 1, s, tab.flags[k] & kListDecays ? a.decay : 1.f, mine, (float *)a.m + im,
                      (float *)a.v + im, mine);
    } else {
      unit_general<false, GT, CAP>(tp, a, s_off, s, tile * (COCO_ADAMW_THREADS / 32) + (threadIdx.x >> 5));
    }
  }
}

// ---- tiles staged in shared memory -----------------------------------------------------
// The same walk with the loads in the hands of the copy engine: one warp asks for whole
// tiles (bulk copies of the gradients, weights, moments and scales) ahead of time, so
// that a warp finds its unit in shared memory and neither waits for HBM nor holds
// registers for what is on its way.  8-bit moments, whose arithmetic leaves little room,
// and tensors that are not aligned: a tile of those is copied from the 16-byte boundary
// below its start to the one above its end (memory of the same allocation), and its new
// weights leave through shared memory, in 16-byte stores but for the ends of a unit.
// Where a tile holds several tensors its units are copied one by one.
//  (Times of the kernel alone, from a captured graph.)
//  8-bit moments, 336 M elements (16 bytes each): 0.84 ms, 0.98 of the copy rate, in a
//  burst, 0.92 ms at the clocks of a long run; with four tiles in flight in place of three
//  0.92.  With two CTAs per SM 0.88 ms in a burst, and beside that: loads by the threads
//  themselves 0.94 ms, asynchronous copies by every warp for itself 1.20 ms (102
//  instructions per element), L2 prefetches one to three units ahead 1.02 to 1.07 ms; two
//  tiles in flight 1.01, four 0.91 ms; 16, 14, 11, 10 warps 0.91, 0.91, 0.98, 0.91 ms.
//  8-bit moments, 900 tensors, 29 M elements: 80 us aligned, 96 packed (0.73).  Those are
//  read and written in shared memory element by element, up to four lanes to a bank: four
//  times the wavefronts of the aligned ones, 60 % of the shared memory's cycles, while the
//  issue slots are busy for 66 % (aligned: 72 %).
//  fp32 moments, 900 tensors, 29 M elements, hardly one aligned: 138 us (0.90) against
//  146 us with element by element loads and stores; 30 such tensors of fp32 gradients,
//  21 M elements: 101 us (0.94).  8 and 9 warps with three tiles in flight 141 and 146 us,
//  10 and 12 warps, which leave room for two, 138 and 142 us.
template <bool QUANT, bool WIDE, typename GT> struct Pipe {
  static constexpr int kThreads = !QUANT ? COCO_ADAMW_PACKED_THREADS : WIDE ? 2 * COCO_ADAMW_QUANT_THREADS : COCO_ADAMW_QUANT_THREADS;
  static constexpr int kCtas = WIDE ? 1 : 2;  // of an SM
  static constexpr int kWarps = kThreads / 32, kTile = kWarps * kListUnit;
  static constexpr int kState = kTile * (QUANT ? 1 : 4);  // bytes of m and of v
  // the gradients and weights of a tile, or of its units one by one
  static constexpr int kGUnit = kListUnit * (int)sizeof(GT) + 16, kWUnit = kListUnit * 4 + 16;
  static constexpr int kG = 0, kW = kG + kWarps * kGUnit, kM = kW + kWarps * kWUnit;
  static constexpr int kV = kM + kState, kScale = kV + kState;
  static constexpr int kBytes = kScale + (QUANT ? (kWarps * 2 + 15) / 16 * 16 + 16 : 0);
  static constexpr int kLp = kWarps * (kListUnit * 2 + 16);  // copies on their way out
  // of an SM's 228 KB: 1 KB per CTA is reserved, up to 9 KB are the kernel's other tables
  static constexpr int kFit = ((228 * 1024) / kCtas - 10 * 1024 - kLp) / kBytes;
  static constexpr int kStages = kFit < COCO_ADAMW_STAGES ? kFit : COCO_ADAMW_STAGES;
  static_assert(kStages >= 2 && kBytes % 16 == 0, "a tile is loaded while another is worked on");
  static constexpr int kSmem = kStages * kBytes + kLp;
};
// The aligned 16-byte pieces that hold bytes [p, p + n).
__device__ __forceinline__ unsigned window(const void *p, unsigned n) {
  return ((unsigned)((uintptr_t)p & 15u) + n + 15u) & ~15u;
}
__device__ __forceinline__ const void *floor16(const void *p) { return (const void *)((uintptr_t)p & ~(uintptr_t)15u); }
// A unit of T that lies in shared memory at the offset that p has within its 16 bytes,
// to p: whole 16-byte pieces at once, what is left at the two ends one by one.
template <typename T> __device__ __forceinline__ void store_unit(T *p, const unsigned char *src) {
  constexpr int kN = 16 / (int)sizeof(T), kPieces = kListUnit / kN;
  const int lane = threadIdx.x & 31, head = (int)((uintptr_t)p & 15u) / (int)sizeof(T);
  T *first = p - head;
  const T *from = reinterpret_cast<const T *>(src);
#pragma unroll
  for (int c = 0; c < kPieces; c += 32)
    if (c + lane > 0 || head == 0)
      reinterpret_cast<uint4 *>(first)[c + lane] = reinterpret_cast<const uint4 *>(from)[c + lane];
  if (head != 0 && lane < kN) {
    const int e = lane >= head ? lane : kListUnit + lane;
    first[e] = from[e];
  }
}

// What the asker of a tile has found out about one of its units.
struct __align__(16) UnitInfo {
  float *w;
  unsigned short *lp;
  void *m, *v;
  unsigned char *scale;
  unsigned g_at, w_at, m_at, scale_at;  // where they are in shared memory, in bytes
  unsigned staged;                      // elements that are asked for, 0: the unit is not staged; kDecays
  unsigned hash;                        // 8-bit moments: hash_start of its first element
  static constexpr unsigned kDecays = 1u << 16;
};

template <bool QUANT, bool WIDE, typename GT, int CAP>
__global__ void __launch_bounds__((Pipe<QUANT, WIDE, GT>::kThreads), (Pipe<QUANT, WIDE, GT>::kCtas))
    adamw_staged_kernel(const __grid_constant__ ListTable<CAP> tab, const __grid_constant__ AdamWArgs a) {
  typedef Pipe<QUANT, WIDE, GT> P;
  static_assert(P::kWarps <= 32, "a lane of the asking warp looks after each unit");
  constexpr unsigned S = P::kStages, kTileGroups = P::kTile / kListGroup;
  extern __shared__ __align__(128) unsigned char s_stage[];
  __shared__ unsigned s_off[CAP + 1];
  __shared__ __align__(8) unsigned long long s_full[S], s_empty[S];
  __shared__ UnitInfo s_info[S][P::kWarps];
  __shared__ int s_tensor[S];  // the tensor in which a stage's tile begins
  const ListTable<CAP> *tp = &tab;
  hide(tp);
  copy_offsets(s_off, tp->off, a.n);
  if (threadIdx.x == 0) {
#pragma unroll
    for (unsigned k = 0; k < S; ++k) mbar_init(&s_full[k], 1), mbar_init(&s_empty[k], P::kWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  float s = a.grad_scale;
  if (a.norm) {
    if (!is_finite(a.norm[0])) return;  // the gradients are not usable: the step is skipped
    s = __fmul_rn(a.norm[1], s);
  }
  __syncthreads();
  const unsigned tiles = (s_off[a.n] + kTileGroups - 1) / kTileGroups;
  const unsigned lane = threadIdx.x & 31, wid = threadIdx.x >> 5;

  // Asks for a tile into a free stage; by one warp, k: a tensor at or before the tile's.
  // Lane l looks after unit l.
  auto ask = [&](unsigned tile, unsigned st, int k) {
    const unsigned e = tile * kTileGroups, el = e + lane * kListUnitGroups, total = s_off[a.n];
    k += find_tensor(s_off + k, a.n - k, e);
    const bool mine_too = lane < P::kWarps && el < total;
    int kl = k;
    if (mine_too && el >= s_off[k + 1]) kl = bisect(k, a.n - 1, el, [&](int x) { return s_off[x]; });
    const unsigned char flags = tab.flags[kl];  // mostly one tensor: the constant bank answers at once
    unsigned staged = 0;
    if (mine_too && a.state_aligned) {
      const size_t left = (size_t)(s_off[kl + 1] - el) * kListGroup - tab.missing[kl];
      // fp32 moments: a unit that a tensor ends in may hold others
      staged = left >= kListUnit ? kListUnit : QUANT ? (unsigned)left : 0;
    }
    const size_t i = mine_too ? (size_t)(el - s_off[kl]) * kListGroup : 0;
    const GT *g = (const GT *)tab.g[kl] + i;
    float *w = tab.w[kl] + i;
    const unsigned g_head = (unsigned)((uintptr_t)g & 15u), w_head = (unsigned)((uintptr_t)w & 15u);
    // all units of one tensor: they follow one another in memory, and in the stage
    const bool run = __all_sync(0xffffffffu, lane >= P::kWarps || (staged == kListUnit && kl == k));
    if (lane < P::kWarps) {
      UnitInfo &info = s_info[st][lane];
      constexpr unsigned kUnitState = P::kState / P::kWarps;
      const size_t unit = (size_t)tile * P::kWarps + lane;
      const unsigned char *scale = a.scale + unit * 2;
      info.w = w, info.lp = (unsigned short *)tab.lp[kl] + i;
      info.m = (unsigned char *)a.m + unit * kUnitState, info.v = (unsigned char *)a.v + unit * kUnitState;
      info.scale = const_cast<unsigned char *>(scale);
      info.g_at = st * P::kBytes + P::kG + lane * (run ? kListUnit * (unsigned)sizeof(GT) : P::kGUnit) + g_head;
      info.w_at = st * P::kBytes + P::kW + lane * (run ? kListUnit * 4u : P::kWUnit) + w_head;
      info.m_at = st * P::kBytes + P::kM + lane * kUnitState;
      info.scale_at = st * P::kBytes + P::kScale + lane * 2 + (unsigned)((uintptr_t)(scale - lane * 2) & 15u);
      info.staged = staged | (flags & kListDecays ? UnitInfo::kDecays : 0u);
      info.hash = hash_start(a.flat0 + unit * kListUnit, a.key);
    }
    const unsigned many = run ? P::kTile : staged;
    const unsigned gb = window(g, many * (unsigned)sizeof(GT)), wb = window(w, many * 4);
    const bool copies = run ? lane == 0 : staged != 0;
    const unsigned bytes = __reduce_add_sync(0xffffffffu, copies ? gb + wb : 0u);
    unsigned char *dst = s_stage + st * P::kBytes;
    __syncwarp();  // the units' records, before the arrival that makes them visible
    if (lane == 0) {
      s_tensor[st] = k;
      if (bytes != 0) {
        const size_t im = (size_t)tile * P::kState;
        // of the last tile, the groups that there are
        const unsigned groups = total - e < kTileGroups ? total - e : kTileGroups;
        const unsigned state = groups * (P::kState / kTileGroups);
        const unsigned char *scale = a.scale + (size_t)tile * P::kWarps * 2;
        const unsigned sb = QUANT ? window(scale, groups / kListUnitGroups * 2) : 0;
        mbar_expect_tx(&s_full[st], bytes + state * 2 + sb);
        bulk_load(dst + P::kM, (const unsigned char *)a.m + im, state, &s_full[st]);
        bulk_load(dst + P::kV, (const unsigned char *)a.v + im, state, &s_full[st]);
        if (QUANT) bulk_load(dst + P::kScale, floor16(scale), sb, &s_full[st]);
      }
    }
    __syncwarp();
    if (copies) {
      bulk_load(dst + P::kG + (run ? 0 : lane * P::kGUnit), floor16(g), gb, &s_full[st]);
      bulk_load(dst + P::kW + (run ? 0 : lane * P::kWUnit), floor16(w), wb, &s_full[st]);
    }
    if (lane == 0 && bytes == 0) mbar_arrive(&s_full[st]);
    __syncwarp();
  };

  if (wid == 0)
    for (unsigned d = 0; d < S - 1; ++d)
      if (blockIdx.x + d * gridDim.x < tiles) ask(blockIdx.x + d * gridDim.x, d, 0);
  unsigned st = 0, phase = 0, turn = 0;  // the stage at hand, its round, the warp whose turn it is to ask
  bool ok = true;
#pragma unroll 1
  for (unsigned tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    ok = __all_sync(0xffffffffu, mbar_wait(&s_full[st], phase, a.timeout_ns));
    if (!ok) break;
    // the warps take turns at asking for the tile S - 1 ahead, into the stage that the
    // tile before this one has left
    if (turn == wid) {
      const unsigned ahead = tile + (S - 1) * gridDim.x, to = st == 0 ? S - 1 : st - 1;
      if (ahead < tiles) {
        // the stage's first use needs no wait; its tile before was number j - 1 of this CTA
        if (tile != blockIdx.x)
          ok = __all_sync(0xffffffffu, mbar_wait(&s_empty[to], st == 0 ? phase ^ 1u : phase, a.timeout_ns));
        if (!ok) break;
        ask(ahead, to, s_tensor[st]);
      }
    }
    turn = turn + 1 == P::kWarps ? 0 : turn + 1;
    const UnitInfo info = s_info[st][wid];
    if (info.staged & ~UnitInfo::kDecays) {
      float *w = info.w;
      unsigned short *lp = info.lp;
      const float decay = info.staged & UnitInfo::kDecays ? a.decay : 1.f;
      const unsigned char *gs = s_stage + info.g_at;
      unsigned char *ws = s_stage + info.w_at;
      const unsigned char *ms = s_stage + info.m_at;  // and the second moments P::kState behind
      const int avail = QUANT ? info.staged & ~UnitInfo::kDecays : kListUnit;
      const bool whole = !QUANT || avail == kListUnit;
      const bool aligned = (((info.g_at | info.w_at) & 15u) | ((uintptr_t)lp & 15u)) == 0;
      auto take = [&](int q, float (&g4)[4], float (&w4)[4]) {
        const unsigned o = 4 * lane + 128 * q;
        if (aligned) {
          widen4<GT>(*reinterpret_cast<const typename Raw<GT>::Four *>(gs + o * sizeof(GT)), g4);
          widen4<float>(*reinterpret_cast<const uint4 *>(ws + o * 4), w4);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            g4[j] = Raw<GT>::widen1(reinterpret_cast<const typename Raw<GT>::One *>(gs)[o + j]);
            w4[j] = reinterpret_cast<const float *>(ws)[o + j];
          }
        }
      };
      // this lane has taken all that it reads of the stage
      auto taken = [&] {
        __syncwarp();
        if ((aligned || !whole) && lane == 0) mbar_arrive(&s_empty[st]);
      };
      auto give = [&](const float (&x)[8]) {
        View<1> t;
        t.w = w, t.lp = lp;
        if (!whole) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (quant_at<true>(k) < avail) put_w1<1>(t, 1, a.lp_kind, (unsigned)quant_at<true>(k), x[k]);
          return;
        }
        if (aligned) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float w4[4] = {x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
            put_w4<1>(t, 1, a.lp_kind, 4 * lane + 128 * q, w4);
          }
          return;
        }
        unsigned char *ls = s_stage + S * P::kBytes + wid * (kListUnit * 2 + 16);
        float *wo = reinterpret_cast<float *>(ws);
        unsigned short *lo = reinterpret_cast<unsigned short *>(ls + ((uintptr_t)lp & 15u));
#pragma unroll
        for (int k = 0; k < 8; ++k) wo[quant_at<true>(k)] = x[k];
        if (a.lp_kind != kLpNone) {
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            const unsigned two = lp_pair(a.lp_kind, x[k], x[k + 1]);
            lo[quant_at<true>(k)] = (unsigned short)two;
            lo[quant_at<true>(k + 1)] = (unsigned short)(two >> 16);
          }
        }
        __syncwarp();
        store_unit(w, ws - ((uintptr_t)w & 15u));
        if (a.lp_kind != kLpNone) store_unit(lp, ls);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into this stage
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[st]);
      };
      if constexpr (QUANT) {
        QuantUnit x;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const unsigned o = 4 * lane + 128 * q;
          float g4[4], w4[4];
          take(q, g4, w4);
          x.m[q] = *reinterpret_cast<const unsigned *>(ms + o);
          x.r[q] = *reinterpret_cast<const unsigned *>(ms + P::kState + o);
#pragma unroll
          for (int j = 0; j < 4; ++j) x.g[4 * q + j] = g4[j], x.w[4 * q + j] = w4[j];
        }
        if (!whole) {  // what lies behind the tensor's end is no part of it
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (quant_at<true>(k) >= avail) {
              x.g[k] = 0.f, x.w[k] = 0.f;
              x.m[k >> 2] &= ~(0xffu << (8 * (k & 3))), x.r[k >> 2] &= ~(0xffu << (8 * (k & 3)));
            }
        }
        x.scale = *reinterpret_cast<const unsigned short *>(s_stage + info.scale_at);
        taken();
        quant_step<true>(x, a, s, decay, info.hash + 4 * lane * kPlaceMul, [&] { give(x.w); });
        unsigned char *m = (unsigned char *)info.m, *r = (unsigned char *)info.v;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const unsigned o = 4 * lane + 128 * q;
          if (whole || quant_at<true>(4 * q + 3) < avail) {
            *reinterpret_cast<unsigned *>(m + o) = x.m[q];
            *reinterpret_cast<unsigned *>(r + o) = x.r[q];
          } else {
            for (int j = 0; quant_at<true>(4 * q) + j < avail; ++j)
              m[o + j] = (unsigned char)(x.m[q] >> (8 * j)), r[o + j] = (unsigned char)(x.r[q] >> (8 * j));
          }
        }
        put_scale(x, info.scale);
      } else {
        float g[8], x[8], m[8], v[8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const unsigned o = 4 * lane + 128 * q;
          float g4[4], w4[4], m4[4], v4[4];
          take(q, g4, w4);
          widen4<float>(*reinterpret_cast<const uint4 *>(ms + o * 4), m4);
          widen4<float>(*reinterpret_cast<const uint4 *>(ms + P::kState + o * 4), v4);
#pragma unroll
          for (int j = 0; j < 4; ++j) g[4 * q + j] = g4[j], x[4 * q + j] = w4[j], m[4 * q + j] = m4[j], v[4 * q + j] = v4[j];
        }
        taken();
#pragma unroll
        for (int k = 0; k < 8; ++k) update1(a, decay, __fmul_rn(g[k], s), x[k], m[k], v[k]);
        float *mo = (float *)info.m, *vo = (float *)info.v;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const unsigned o = 4 * lane + 128 * q;
          *reinterpret_cast<float4 *>(mo + o) = make_float4(m[4 * q], m[4 * q + 1], m[4 * q + 2], m[4 * q + 3]);
          *reinterpret_cast<float4 *>(vo + o) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        }
        give(x);
      }
    } else {
      if (lane == 0) mbar_arrive(&s_empty[st]);
      unit_general<QUANT, GT, CAP>(tp, a, s_off, s, tile * P::kWarps + wid);
    }
    if (++st == S) st = 0, phase ^= 1u;
  }
  if (!ok) {
    // a copy or a warp of this CTA was not there in time: say so, and give the copies in
    // flight one more bounded wait before the shared memory is given up
    if (lane == 0) {
      record_status(a.page, cocoTimeout, 0, kPhaseCopy, -1, 0);
      for (unsigned d = 0; d < S; ++d, st = st + 1 == S ? 0 : st + 1, phase ^= st == 0)
        mbar_wait(&s_full[st], phase, a.timeout_ns);
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
                                      left < kListGroup ? (int)left : kListGroup, (float *)a.m, (float *)a.v,
                                      (size_t)el * kListGroup);
      }
      __syncwarp();
    }
  }
  list_end_barrier(pr, pa, started);
}

// ---- launches --------------------------------------------------------------------
template <int CAP> using Kernel = void (*)(const ListTable<CAP>, const AdamWArgs);
struct LaunchShape {
  int threads, ctas_per_sm, smem;
};
template <bool QUANT, bool WIDE, typename GT, int CAP> Kernel<CAP> pick_staged(LaunchShape *sh) {
  typedef Pipe<QUANT, WIDE, GT> P;
  *sh = {P::kThreads, P::kCtas, P::kSmem};
  return adamw_staged_kernel<QUANT, WIDE, GT, CAP>;
}
// 8-bit moments: staged tiles, which measured better for aligned tensors too.  `wide`,
// one CTA of 24 warps per SM in place of two of 12, has half as many tiles: better where
// they lie in one tensor mostly (398 tensors, 336 M elements: 0.84 against 0.88 ms; 30
// tensors, 21 M: 56.5 against 57.5 us), worse where many hold several (900 tensors, 29 M:
// 84 against 80 us, packed 102 against 96) and on few tiles (one tensor of 256 Ki elements
// 5.0 against 3.8 us, of 1 Mi 7.4 against 6.0; of 4 Mi the same, of 16 Mi 46.6 against 47.1).
// fp32 moments: staged tiles where tensors are not aligned, which the direct kernel would
// walk element by element; else the direct kernel (12.6 M elements 58 against 61 us,
// 336 M 1.49 against 1.51 ms).
template <int CAP> Kernel<CAP> pick(bool quant, bool packed, bool wide, cocoDataType_t g, LaunchShape *sh) {
  auto of = [&](auto type) -> Kernel<CAP> {
    typedef decltype(type) GT;
    if (quant) return wide ? pick_staged<true, true, GT, CAP>(sh) : pick_staged<true, false, GT, CAP>(sh);
    if (packed) return pick_staged<false, false, GT, CAP>(sh);
    *sh = {COCO_ADAMW_THREADS, 2, 0};
    return adamw_kernel<GT, CAP>;
  };
  switch (g) {
    case cocoFloat32: return of(float());
    case cocoFloat16: return of(__half());
    case cocoBfloat16: return of(__nv_bfloat16());
  }
  return nullptr;
}
// From how many units per tensor, on average, and per SM `wide` is taken: 256 Ki elements
// a tensor, 8 tiles a CTA.
constexpr size_t kWideUnits = 1024, kWideUnitsPerSm = 8 * 2 * COCO_ADAMW_QUANT_THREADS / 32;
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

template <int CAP>
cudaError_t launch_adamw(bool quant, bool packed, cocoDataType_t g_type, const ListTable<CAP> &table,
                         const AdamWArgs &args, size_t units, int device, int sm_count,
                         int max_ctas_per_sm, cudaStream_t stream) {
  LaunchShape sh;
  const bool wide = quant && units >= kWideUnits * (size_t)args.n && units >= kWideUnitsPerSm * (size_t)sm_count;
  const Kernel<CAP> k = pick<CAP>(quant, packed, wide, g_type, &sh);
  if (!k) return cudaErrorInvalidValue;
  if (sh.smem > 0) {  // more than the default: allowed once per kernel and device
    static std::atomic<unsigned long long> allowed[2][2][3];
    std::atomic<unsigned long long> &mask = allowed[quant][wide][g_type == cocoFloat32 ? 0 : g_type == cocoFloat16 ? 1 : 2];
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (!(mask.load(std::memory_order_acquire) & bit)) {
      const cudaError_t e = cudaFuncSetAttribute((const void *)k, cudaFuncAttributeMaxDynamicSharedMemorySize, sh.smem);
      if (e != cudaSuccess) return e;
      mask.fetch_or(bit, std::memory_order_release);
    }
  }
  const int per_sm = max_ctas_per_sm > 0 && max_ctas_per_sm < sh.ctas_per_sm ? max_ctas_per_sm : sh.ctas_per_sm;
  const size_t warps = (size_t)sh.threads / 32, need = (units + warps - 1) / warps, room = (size_t)per_sm * sm_count;
  void *params[] = {(void *)&table, (void *)&args};
  return cudaLaunchKernel((const void *)k, dim3((unsigned)(need < room ? need : room)), dim3(sh.threads), params,
                          sh.smem, stream);
}
template cudaError_t launch_adamw<kListCapSmall>(bool, bool, cocoDataType_t, const ListTable<kListCapSmall> &,
                                                 const AdamWArgs &, size_t, int, int, int, cudaStream_t);
template cudaError_t launch_adamw<kListCapLarge>(bool, bool, cocoDataType_t, const ListTable<kListCapLarge> &,
                                                 const AdamWArgs &, size_t, int, int, int, cudaStream_t);

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
int adamw_peer_threads() { return COCO_ADAMW_PEER_THREADS; }
cudaError_t adamw_peers_occupancy(bool quant, cocoDataType_t g_type, int world, int threads,
                                  int *ctas_per_sm) {
  const PeerKernel k = pick_peer(quant, g_type, world);
  if (!k) return cudaErrorInvalidValue;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(ctas_per_sm, (const void *)k, threads, 0);
}

}  // namespace coco
