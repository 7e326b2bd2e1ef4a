// AdamW over a list of tensors, with fp32 moments or with moments in 8 bits.
//
// Per element, t = step + 1, d1 = 1 - beta1^t, d2 = 1 - beta2^t (from the host):
//   g <- (sum over ranks of g) * grad_scale * clip
//   m <- beta1 m + (1 - beta1) g        v <- beta2 v + (1 - beta2) g^2
//   w <- w (1 - lr decay) - (lr / d1) m / (sqrt(v) / sqrt(d2) + eps)
// Every operation is rounded to fp32 by itself, so the results do not depend on
// the path an element takes and match a scalar evaluation bit for bit.
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
  unsigned short h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    h[e] = kind == kLpF16 ? Bits16<__half>::from_f32(x[e]) : Bits16<__nv_bfloat16>::from_f32(x[e]);
  const uint2 q = make_uint2(h[0] | ((unsigned)h[1] << 16), h[2] | ((unsigned)h[3] << 16));
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
__device__ __forceinline__ void moments(const AdamWArgs &a, float g, float &m, float &v) {
  m = __fadd_rn(__fmul_rn(m, a.beta1), __fmul_rn(g, a.omb1));
  v = __fadd_rn(__fmul_rn(v, a.beta2), __fmul_rn(__fmul_rn(g, g), a.omb2));
}
__device__ __forceinline__ float step_w(const AdamWArgs &a, float decay, float w, float m, float r) {
  const float den = __fadd_rn(__fmul_rn(r, a.rs2), a.eps);
  return __fsub_rn(__fmul_rn(w, decay), __fdiv_rn(__fmul_rn(m, a.c1), den));
}

// ---- 8-bit codes -----------------------------------------------------------------
// Multiply and xor-shift rounds; the multipliers are binary fractions of the
// golden ratio and of the roots of 2, 3 and 5.  Any well-mixed function would do.
__host__ __device__ __forceinline__ unsigned mix_bits(unsigned x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
__device__ __forceinline__ unsigned rounding_bits(unsigned long long place, unsigned key) {
  return mix_bits((unsigned)place * 0x9E3779B1u + (unsigned)(place >> 32) * 0x3C6EF373u + key);
}
// A code's 7 magnitude bits lead a float's exponent and mantissa, which is the
// same number times 2^-120, subnormals included.
__device__ __forceinline__ float decode(unsigned code, float scale) {
  const unsigned bits = ((code & 0x7fu) << 20) | ((code & 0x80u) << 24);
  return __fmul_rn(__fmul_rn(__uint_as_float(bits), 0x1p120f), scale);
}
__device__ __forceinline__ float scale_of(unsigned byte) {
  return byte == 0 ? 0x1p-127f : __uint_as_float(byte == 255 ? 0x7fc00000u : byte << 23);
}
// Scale byte of a block with this largest magnitude (as bits), and the scale's
// inverse: the block's largest code lies in [128, 256), which leaves room to
// round up below 448.  255 (not a number) for a block that holds inf or nan.
__device__ __forceinline__ unsigned block_scale(unsigned max_bits, float &inverse) {
  unsigned e = max_bits >> 23;
  e = e < 8u ? 8u : e > 254u ? 254u : e;
  inverse = __uint_as_float((261u - e) << 23);
  return max_bits >= 0x7f800000u ? 255u : e - 7u;
}
// 20 random bits: 16 of the hash, then a one that centres them, then zeros.
__device__ __forceinline__ unsigned encode(float x, float inverse, unsigned bits16) {
  const float y = __fmul_rn(__fmul_rn(fabsf(x), inverse), 0x1p-120f);
  return ((__float_as_uint(y) + ((bits16 << 4) | 8u)) >> 20) | ((__float_as_uint(x) >> 24) & 0x80u);
}

// ---- one unit: eight elements per lane ---------------------------------------------
// Vector form: elements i + 4 lane .. + 3 and i + 128 + 4 lane .. + 3, so that
// every 16-byte access of the warp is one run of memory.
template <int RB, typename GT>
__device__ __forceinline__ void unit_vec(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                         float decay, size_t i, float *m_, float *v_) {
  const int lane = threadIdx.x & 31;
  float g[2][4], w[2][4], m[2][4], v[2][4];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int o = 4 * lane + 128 * q;
    sum_grad4<RB, GT>(t.g, R, i + o, g[q]);
    const float4 w4 = *reinterpret_cast<const float4 *>(t.w + i + o);
    const float4 m4 = *reinterpret_cast<const float4 *>(m_ + o);
    const float4 v4 = *reinterpret_cast<const float4 *>(v_ + o);
    w[q][0] = w4.x, w[q][1] = w4.y, w[q][2] = w4.z, w[q][3] = w4.w;
    m[q][0] = m4.x, m[q][1] = m4.y, m[q][2] = m4.z, m[q][3] = m4.w;
    v[q][0] = v4.x, v[q][1] = v4.y, v[q][2] = v4.z, v[q][3] = v4.w;
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int o = 4 * lane + 128 * q;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      moments(a, __fmul_rn(g[q][e], s), m[q][e], v[q][e]);
      w[q][e] = step_w(a, decay, w[q][e], m[q][e], __fsqrt_rn(v[q][e]));
    }
    *reinterpret_cast<float4 *>(m_ + o) = make_float4(m[q][0], m[q][1], m[q][2], m[q][3]);
    *reinterpret_cast<float4 *>(v_ + o) = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
    put_w4<RB>(t, R, a.lp_kind, i + o, w[q]);
  }
}
// Scalar form: nv elements of this lane, `stride` apart.
template <int RB, typename GT>
__device__ __forceinline__ void unit_scalar(const View<RB> &t, const AdamWArgs &a, int R, float s,
                                            float decay, size_t i, int stride, int nv, float *m_,
                                            float *v_) {
  float g[8], w[8], m[8], v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < nv) {
      g[e] = sum_grad1<RB, GT>(t.g, R, i + e * stride);
      w[e] = t.w[i + e * stride];
      m[e] = m_[e * stride];
      v[e] = v_[e * stride];
    }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < nv) {
      moments(a, __fmul_rn(g[e], s), m[e], v[e]);
      w[e] = step_w(a, decay, w[e], m[e], __fsqrt_rn(v[e]));
      m_[e * stride] = m[e];
      v_[e * stride] = v[e];
      put_w1<RB>(t, R, a.lp_kind, i + e * stride, w[e]);
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
  float g[8], w[8], m[8], r[8];
  unsigned mc[2], rc[2];  // VEC: four codes each
  const unsigned sc = *reinterpret_cast<const unsigned short *>(scale);
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int o = 4 * lane + 128 * q;
      float g4[4];
      sum_grad4<RB, GT>(t.g, R, i + o, g4);
      const float4 w4 = *reinterpret_cast<const float4 *>(t.w + i + o);
      mc[q] = *reinterpret_cast<const unsigned *>(m_ + o);
      rc[q] = *reinterpret_cast<const unsigned *>(r_ + o);
#pragma unroll
      for (int e = 0; e < 4; ++e) g[4 * q + e] = g4[e];
      w[4 * q] = w4.x, w[4 * q + 1] = w4.y, w[4 * q + 2] = w4.z, w[4 * q + 3] = w4.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (at(e) < avail) {
        g[e] = sum_grad1<RB, GT>(t.g, R, i + at(e));
        w[e] = t.w[i + at(e)];
        m[e] = __uint_as_float(m_[at(e)]);
        r[e] = __uint_as_float(r_[at(e)]);
      }
  }
  const float m_scale = scale_of(sc & 0xffu), r_scale = scale_of(sc >> 8);
  unsigned m_max = 0, r_max = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (VEC || at(e) < avail) {
      const unsigned cm = VEC ? (mc[e >> 2] >> (8 * (e & 3))) & 0xffu : __float_as_uint(m[e]);
      const unsigned cr = VEC ? (rc[e >> 2] >> (8 * (e & 3))) & 0xffu : __float_as_uint(r[e]);
      m[e] = decode(cm, m_scale);
      const float r0 = decode(cr, r_scale);
      float v = __fmul_rn(r0, r0);
      moments(a, __fmul_rn(g[e], s), m[e], v);
      r[e] = __fsqrt_rn(v);
      w[e] = step_w(a, decay, w[e], m[e], r[e]);
      const unsigned mb = __float_as_uint(m[e]) & 0x7fffffffu, rb = __float_as_uint(r[e]) & 0x7fffffffu;
      m_max = mb > m_max ? mb : m_max;
      r_max = rb > r_max ? rb : r_max;
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
      if (at(e) < avail) put_w1<RB>(t, R, a.lp_kind, i + at(e), w[e]);
  }
  m_max = __reduce_max_sync(0xffffffffu, m_max);
  r_max = __reduce_max_sync(0xffffffffu, r_max);
  float m_inv, r_inv;
  const unsigned mb = block_scale(m_max, m_inv), rb = block_scale(r_max, r_inv);
  unsigned cm[8], cr[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (VEC || at(e) < avail) {
      const unsigned bits = rounding_bits(place + at(e), a.key);
      const unsigned x = encode(m[e], m_inv, bits & 0xffffu);
      unsigned y = encode(r[e], r_inv, bits >> 16);
      if (y == 0u && r[e] > 0.f) y = 1u;
      cm[e] = mb == 255u ? 0u : x;
      cr[e] = rb == 255u ? 0u : y;
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
      if (at(e) < avail) m_[at(e)] = (unsigned char)cm[e], r_[at(e)] = (unsigned char)cr[e];
  }
  if (lane == 0) *reinterpret_cast<unsigned short *>(scale) = (unsigned short)(mb | (rb << 8));
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
      unit_scalar<RB, GT>(t, a, R, s, decay, i + lane, 32, avail > lane ? (avail - lane + 31) / 32 : 0,
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
        unit_scalar<1, GT>(tl, a, 1, s, tab.decays[k] ? a.decay : 1.f,
                           (size_t)(el - s_off[k]) * kListGroup, 1, nv,
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
        unit_scalar<RB, GT>(t, a, R, s, pl.decays ? a.decay : 1.f, (size_t)pl.begin + done, 1,
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
  return mix_bits(mix_bits((unsigned)seed) + (unsigned)(seed >> 32) * 0x3C6EF373u +
                  (unsigned)step * 0x9E3779B1u);
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
