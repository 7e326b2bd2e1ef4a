// Device code shared by the kernels over lists of tensors: gradients of one or
// several ranks, the barriers between ranks, finding a piece of the list.
#pragma once

#include "device_util.cuh"
#include "list_step.cuh"

namespace coco {
namespace {

// ---- gradients ---------------------------------------------------------------
// RB bounds the world size at compile time: 1 (plain loads of the own
// gradient), 2 (exactly two ranks), 4, 8.  The sum runs in rank order in fp32.
template <typename GT> __device__ __forceinline__ void widen4(uint4 q, float (&x)[4]) {
  x[0] = __uint_as_float(q.x), x[1] = __uint_as_float(q.y);
  x[2] = __uint_as_float(q.z), x[3] = __uint_as_float(q.w);
}
template <typename GT> __device__ __forceinline__ void widen4(uint2 q, float (&x)[4]) {
  x[0] = Bits16<GT>::to_f32((unsigned short)(q.x & 0xffffu));
  x[1] = Bits16<GT>::to_f32((unsigned short)(q.x >> 16));
  x[2] = Bits16<GT>::to_f32((unsigned short)(q.y & 0xffffu));
  x[3] = Bits16<GT>::to_f32((unsigned short)(q.y >> 16));
}
template <typename GT> struct Raw {
  typedef uint2 Four;
  typedef unsigned short One;
  template <typename Index> static __device__ __forceinline__ Four peer4(const void *p, Index i) {
    return ld_sys_8((const unsigned short *)p + i);
  }
  template <typename Index> static __device__ __forceinline__ One peer1(const void *p, Index i) {
    return ld_sys_2((const unsigned short *)p + i);
  }
  template <typename Index> static __device__ __forceinline__ Four own4(const void *p, Index i) {
    return *reinterpret_cast<const uint2 *>((const unsigned short *)p + i);
  }
  template <typename Index> static __device__ __forceinline__ One own1(const void *p, Index i) {
    return ((const unsigned short *)p)[i];
  }
  static __device__ __forceinline__ float widen1(One b) { return Bits16<GT>::to_f32(b); }
};
template <> struct Raw<float> {
  typedef uint4 Four;
  typedef unsigned One;
  template <typename Index> static __device__ __forceinline__ Four peer4(const void *p, Index i) {
    return ld_sys_16((const float *)p + i);
  }
  template <typename Index> static __device__ __forceinline__ One peer1(const void *p, Index i) {
    return ld_sys_4((const float *)p + i);
  }
  template <typename Index> static __device__ __forceinline__ Four own4(const void *p, Index i) {
    return *reinterpret_cast<const uint4 *>((const float *)p + i);
  }
  template <typename Index> static __device__ __forceinline__ One own1(const void *p, Index i) {
    return ((const unsigned *)p)[i];
  }
  static __device__ __forceinline__ float widen1(One b) { return __uint_as_float(b); }
};

template <int RB, typename GT, typename Index>
__device__ __forceinline__ void sum_grad4(const void *const *g, int R, Index i, float (&x)[4]) {
  if constexpr (RB == 1) {
    widen4<GT>(Raw<GT>::own4(g[0], i), x);
  } else {
    typename Raw<GT>::Four raw[RB];
#pragma unroll
    for (int p = 0; p < RB; ++p)
      if (RB == 2 || p < R) raw[p] = Raw<GT>::peer4(g[p], i);
    widen4<GT>(raw[0], x);
#pragma unroll
    for (int p = 1; p < RB; ++p)
      if (RB == 2 || p < R) {
        float y[4];
        widen4<GT>(raw[p], y);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __fadd_rn(x[e], y[e]);
      }
  }
}
template <int RB, typename GT, typename Index>
__device__ __forceinline__ float sum_grad1(const void *const *g, int R, Index i) {
  if constexpr (RB == 1) {
    return Raw<GT>::widen1(Raw<GT>::own1(g[0], i));
  } else {
    float x = Raw<GT>::widen1(Raw<GT>::peer1(g[0], i));
    for (int p = 1; p < R; ++p) x = __fadd_rn(x, Raw<GT>::widen1(Raw<GT>::peer1(g[p], i)));
    return x;
  }
}

// ---- barriers between ranks --------------------------------------------------
// Every CTA waits until all ranks' kernels of this call have started.  Returns
// whether they did (the same in every thread); a late rank is in the status word.
__device__ __forceinline__ bool list_start_barrier(const PeerRank &pr, const PeerArgs &pa, int *s_ok) {
  FlagPage *me = pr.flags[pr.rank];
  if (threadIdx.x == 0) *s_ok = 1;
  __syncthreads();
  if (threadIdx.x < 32) {
    if (blockIdx.x == 0)
      warp_signal_peers(pr, pa.world, pr.rank, pa.seq, [](FlagPage *f) { return f->arrive; });
    const int late = warp_wait_peers(me->arrive, pa.world, pr.rank, pa.seq, pa.timeout_ns);
    if (late >= 0 && threadIdx.x == 0) {
      record_status(me, cocoTimeout, pr.rank, kPhaseStart, late, pa.seq);
      *s_ok = 0;
    }
  }
  __syncthreads();
  return *s_ok != 0;
}
// The rank's last CTA announces that its reads and writes are complete and
// waits for the others', so that the kernel ends only when nobody touches this
// rank's memory any more.  Where a CTA of the rank gave up at the start (ok), its
// part is missing: nothing is announced, and the other ranks' waits run out, so
// that their status words say so too.
__device__ __forceinline__ void list_end_barrier(const PeerRank &pr, const PeerArgs &pa, bool ok) {
  constexpr unsigned kGaveUp = 0x10000u;  // in the counter's upper half: CTAs that did
  static_assert(kMaxCtasPerRank < kGaveUp, "a rank's CTAs are counted in 16 bits");
  FlagPage *me = pr.flags[pr.rank];
  __threadfence_system();
  __syncthreads();
  if (threadIdx.x >= 32) return;
  unsigned ctas = 0;
  if (threadIdx.x == 0) {
    const unsigned mine = ok ? 1u : 1u + kGaveUp;
    __threadfence_system();
    ctas = atomicAdd(&me->done_count, mine) + mine;
    if (ctas % kGaveUp == gridDim.x) me->done_count = 0;
    __threadfence_system();
  }
  __syncwarp();
  ctas = __shfl_sync(0xffffffffu, ctas, 0);
  if (ctas != gridDim.x) return;  // not the last, or not complete
  __threadfence_system();
  warp_signal_peers(pr, pa.world, pr.rank, pa.seq, [](FlagPage *f) { return f->done; });
  const int late = warp_wait_peers(me->done, pa.world, pr.rank, pa.seq, pa.timeout_ns);
  if (late >= 0 && threadIdx.x == 0)
    record_status(me, cocoTimeout, pr.rank, kPhaseEnd, late, pa.seq);
}

// Makes the compiler forget that a pointer is to a kernel parameter: reads of the
// constant bank at 32 different places take turns, through a plain pointer they are
// one access per warp.
template <typename T> __device__ __forceinline__ void hide(const T *&p) { asm volatile("" : "+l"(p)); }
__device__ __forceinline__ void copy_offsets(unsigned *dst, const unsigned *off, int n) {
  for (int k = threadIdx.x; k <= n; k += blockDim.x) dst[k] = off[k];
}

// ---- finding a tensor ----------------------------------------------------------
// The last t in [0, n) with off[t] <= e, n <= 1024, off[0] <= e: two ballots.
// All 32 lanes call it with the same e.
__device__ __forceinline__ int find_tensor(const unsigned *off, int n, unsigned e) {
  const int lane = threadIdx.x & 31;
  const int coarse = lane * 32;
  const int hi = __popc(__ballot_sync(0xffffffffu, coarse < n && off[coarse < n ? coarse : 0] <= e)) - 1;
  const int fine = hi * 32 + lane;
  return hi * 32 + __popc(__ballot_sync(0xffffffffu, fine < n && off[fine < n ? fine : 0] <= e)) - 1;
}
// The same for one lane by bisection in [a, b].
template <typename OffOf>
__device__ __forceinline__ int bisect(int a, int b, unsigned e, OffOf off) {
  while (a < b) {
    const int mid = (a + b + 1) >> 1;
    if (off(mid) <= e) a = mid;
    else b = mid - 1;
  }
  return a;
}

__device__ __forceinline__ bool is_finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

}  // namespace
}  // namespace coco
