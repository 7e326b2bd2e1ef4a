// Device helpers shared by the kernels that read and write peers' memory:
// memory-model accesses, bounded waits and the status word, the exchange of
// flags between ranks, mbarriers and bulk copies, 16-bit element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "coconet_device.h"
#include "coconet_rt.h"

namespace coco {
namespace {

// ---------------------------------------------------------------------------
// memory-model helpers
// ---------------------------------------------------------------------------
__device__ __forceinline__ unsigned long long globaltimer_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ unsigned long long ld_acquire_sys(const unsigned long long *p) {
  unsigned long long v;
  asm volatile("ld.acquire.sys.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ void st_release_sys(unsigned long long *p, unsigned long long v) {
  asm volatile("st.release.sys.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

// Loads/stores of data that another GPU writes or reads: system-coherent
// (never served from a stale L1 line), 16 bytes wide where possible.
__device__ __forceinline__ uint4 ld_sys_16(const void *p) {
  uint4 v;
  asm volatile("ld.volatile.global.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_sys_8(const void *p) {
  uint2 v;
  asm volatile("ld.volatile.global.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ unsigned ld_sys_4(const void *p) {
  unsigned v;
  asm volatile("ld.volatile.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ unsigned short ld_sys_2(const void *p) {
  unsigned short v;
  asm volatile("ld.volatile.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ void st_sys_16(void *p, uint4 v) {
  asm volatile("st.volatile.global.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ void st_sys_8(void *p, uint2 v) {
  asm volatile("st.volatile.global.v2.u32 [%0], {%1,%2};" ::"l"(p), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void st_sys_4(void *p, unsigned v) {
  asm volatile("st.volatile.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
__device__ __forceinline__ void st_sys_2(void *p, unsigned short v) {
  asm volatile("st.volatile.global.u16 [%0], %1;" ::"l"(p), "h"(v) : "memory");
}
__device__ __forceinline__ double ld_volatile_f64(const double *p) {
  double v;
  asm volatile("ld.volatile.global.f64 %0, [%1];" : "=d"(v) : "l"(p));
  return v;
}

// ---------------------------------------------------------------------------
// bounded waits and the status word
// ---------------------------------------------------------------------------
constexpr unsigned kSpinHardCap = 1u << 28;  // backstop if the timer misbehaves

__device__ __noinline__ void record_status(FlagPage *me, int code, int rank, int phase, int peer,
                              unsigned long long seq) {
  if (atomicCAS(&me->status[0], 0, code) == 0) {
    me->status[1] = rank;
    me->status[2] = phase;
    me->status[3] = peer;
    me->status[4] = (int)(seq & 0xffffffffull);
    me->status[5] = (int)(seq >> 32);
  }
}

// Waits until flags[p] >= seq for every p in [0, world) except `skip`.
// Returns -1 on success, else the first peer that did not show up in time.
__device__ __noinline__ int wait_all(const unsigned long long *flags, int world, int skip,
                        unsigned long long seq, unsigned long long timeout_ns) {
  const unsigned long long t0 = globaltimer_ns();
  for (int p = 0; p < world; ++p) {
    if (p == skip) continue;
    unsigned spins = 0;
    while (ld_acquire_sys(flags + p) < seq) {
      ++spins;
      if ((spins & 63u) == 0u) {
        if (globaltimer_ns() - t0 > timeout_ns || spins > kSpinHardCap) return p;
        __nanosleep(64);
      }
    }
  }
  return -1;
}

// One flag.  Returns false if it did not reach seq in time.
__device__ __noinline__ bool wait_one(const unsigned long long *flag, unsigned long long seq,
                         unsigned long long timeout_ns) {
  if (ld_acquire_sys(flag) >= seq) return true;
  const unsigned long long t0 = globaltimer_ns();
  for (unsigned spins = 1; spins <= kSpinHardCap; ++spins) {
    if (ld_acquire_sys(flag) >= seq) return true;
    if ((spins & 63u) == 0u) {
      if (globaltimer_ns() - t0 > timeout_ns) return false;
      __nanosleep(32);
    }
  }
  return false;
}

// Flags are exchanged by the first warp of a CTA, lane p talking to rank p, so
// that the R-1 remote stores (each a release: fence + store) and the R-1 polls
// proceed in parallel instead of one after the other.
// signal: store seq into slot `rank` of flags_of(p) for every peer p.
// wait:   until own slot p >= seq for every peer p; returns the first late peer or -1.
// Must be called by all 32 lanes of warp 0.
// `args` is anything with the peers' flag pages in flags[].
template <typename Args, typename SlotOf>
__device__ __forceinline__ void warp_signal_peers(const Args &args, int R, int rank,
                                                  unsigned long long seq, SlotOf slot_of) {
  const int p = threadIdx.x & 31;
  if (p < R && p != rank) st_release_sys(slot_of(args.flags[p]) + rank, seq);
}
__device__ __forceinline__ int warp_wait_peers(const unsigned long long *slots, int R, int rank,
                                               unsigned long long seq,
                                               unsigned long long timeout_ns) {
  const int p = threadIdx.x & 31;
  bool late = false;
  if (p < R && p != rank) late = !wait_one(slots + p, seq, timeout_ns);
  const unsigned bad = __ballot_sync(0xffffffffu, late);
  return bad ? __ffs(bad) - 1 : -1;
}

// ---------------------------------------------------------------------------
// mbarriers and bulk copies
// ---------------------------------------------------------------------------
__device__ __forceinline__ unsigned smem_u32(const void *p) {
  return (unsigned)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_init(unsigned long long *bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long *bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(unsigned long long *bar, unsigned parity) {
  unsigned ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded: gives up after timeout_ns (checked every 256 probes) or 2^26 probes.
__device__ __noinline__ bool mbar_wait_slow(unsigned long long *bar, unsigned parity,
                                            unsigned long long timeout_ns) {
  const unsigned long long t0 = globaltimer_ns();
  for (unsigned spin = 1; spin < (1u << 26); ++spin) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((spin & 255u) == 0u && globaltimer_ns() - t0 > timeout_ns) return false;
  }
  return false;
}
__device__ __forceinline__ bool mbar_wait(unsigned long long *bar, unsigned parity,
                                          unsigned long long timeout_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, timeout_ns);
}
// global -> shared bulk copy; src, dst and bytes are multiples of 16.
__device__ __forceinline__ void bulk_load(void *dst, const void *src, unsigned bytes,
                                          unsigned long long *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// ---------------------------------------------------------------------------
// element types
// ---------------------------------------------------------------------------
struct NoLp {};  // "no low-precision copy": the fp32 weights are what is gathered

template <typename T> struct Bits16;
template <> struct Bits16<__half> {
  static __device__ __forceinline__ float to_f32(unsigned short b) {
    return __half2float(__ushort_as_half(b));
  }
  static __device__ __forceinline__ unsigned short from_f32(float f) {
    return __half_as_ushort(__float2half_rn(f));
  }
};
template <> struct Bits16<__nv_bfloat16> {
  static __device__ __forceinline__ float to_f32(unsigned short b) {
    return __uint_as_float(((unsigned)b) << 16);
  }
  static __device__ __forceinline__ unsigned short from_f32(float f) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  }
};

}  // namespace
}  // namespace coco
