// Global gradient norm over a list of tensors, and the clip factor from it:
//   n = |grad_scale| * sqrt(sum over the list of (sum over ranks of g)^2)
//   clip = max_norm / n where 0 < max_norm < n, else 1; 0 where n is not finite
// Both stay in device memory, where the AdamW calls read them.
//
// What bounds it: reading g once from HBM (2 or 4 bytes per element, a
// conversion and a multiply-add each): 336 M fp32 elements 193 us, 1.06 of the
// measured copy rate (reads alone are faster than a copy); a list of 12.6 M bf16
// elements 7.0 us, of which 2.5 us are an empty call's (from a captured graph).  Three
// CTAs of 512 threads with four 16-byte loads each: two CTAs with eight 255 us, four with
// four 216 us.  Squares are added in fp32 within 16
// bytes only and in fp64 from there on, in an order fixed by the launch shape:
// repeated calls give the same bits.  Where 16 bytes' sum leaves the range in
// which fp32 loses nothing that matters, it is redone in fp64.
#include "list_device.cuh"

#ifndef COCO_NORM_THREADS
#define COCO_NORM_THREADS 512
#endif
#ifndef COCO_NORM_CTAS
#define COCO_NORM_CTAS 3
#endif
#ifndef COCO_NORM_DEPTH
#define COCO_NORM_DEPTH 4
#endif

namespace coco {
namespace {

constexpr int kDepth = COCO_NORM_DEPTH;  // 16-byte groups a lane has in flight
constexpr int kUnit = 32 * kDepth;       // groups of a warp's pass

template <typename GT> struct Group {  // 16 bytes
  static constexpr int kN = 16 / (int)sizeof(GT);
  static __device__ __forceinline__ float get(const uint4 &q, int e) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
    return Bits16<GT>::to_f32((unsigned short)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu));
  }
};
template <> struct Group<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ float get(const uint4 &q, int e) {
    return __uint_as_float(e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w);
  }
};

template <typename GT> __device__ __noinline__ double squares_f64(uint4 q) {
  double s = 0.0;
  if ((q.x | q.y | q.z | q.w) == 0u) return s;
#pragma unroll
  for (int e = 0; e < Group<GT>::kN; ++e) {
    const double x = (double)Group<GT>::get(q, e);
    s += x * x;
  }
  return s;
}
// Below 2^-100 squares may have been lost to underflow, above 2^126 the sum
// overflows (or is not a number, which the comparison refuses too).
template <typename GT> __device__ __forceinline__ double squares(const uint4 &q) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < Group<GT>::kN; ++e) {
    const float x = Group<GT>::get(q, e);
    s = fmaf(x, x, s);
  }
  if (s >= 0x1p-100f && s <= 0x1p126f) return (double)s;
  return squares_f64<GT>(q);
}
// The first `head` and last `tail` elements of 16 bytes replaced by zeros.
template <typename GT> __device__ __forceinline__ uint4 masked(uint4 q, int head, int tail) {
  constexpr int kN = Group<GT>::kN, kBits = 128 / kN;
  unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int e = 0; e < kN; ++e)
    if (e < head || e >= kN - tail)
      w[e * kBits / 32] &= kBits == 32 ? 0u : e & 1 ? 0x0000ffffu : 0xffff0000u;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_down_sync(0xffffffffu, x, o);
  return x;
}

// The CTAs' sums (part, STRIDE apart), by the CTA that arrives last; true in that CTA
// only, with the total in thread 0.
template <int STRIDE>
__device__ __forceinline__ bool rank_sum(double x, unsigned *count, double *part, double &total) {
  __shared__ double s_part[32];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  x = warp_sum(x);
  if (lane == 0) s_part[wid] = x;
  __syncthreads();
  if (gridDim.x > 1) {
    if (wid == 0) {
      x = warp_sum(lane < nw ? s_part[lane] : 0.0);
      if (lane == 0) {
        part[(size_t)blockIdx.x * STRIDE] = x;
        __threadfence();
        s_last = atomicAdd(count, 1u) == gridDim.x - 1;
      }
    }
    __syncthreads();
    if (!s_last) return false;
    __threadfence();
    x = 0.0;
    for (unsigned c = threadIdx.x; c < gridDim.x; c += blockDim.x)
      x += ld_volatile_f64(&part[(size_t)c * STRIDE]);
    x = warp_sum(x);
    __syncthreads();
    if (lane == 0) s_part[wid] = x;
    __syncthreads();
    if (threadIdx.x == 0) *count = 0;
  }
  total = wid == 0 ? warp_sum(lane < nw ? s_part[lane] : 0.0) : 0.0;
  return true;
}

__device__ __forceinline__ void put_norm(const NormArgs &a, float *out, double total) {
  const double n = sqrt(total) * a.scale;
  const float nf = (float)n;
  out[0] = nf;
  out[1] = !is_finite(nf) ? 0.f : a.max_norm > 0.0 && n > a.max_norm ? (float)(a.max_norm / n) : 1.f;
}

// A tensor's first and last 16 bytes may hold elements of its neighbours: they are read
// with it (16 aligned bytes that hold one of its elements are memory of the same
// allocation) and masked.
template <typename GT, int CAP>
__global__ void __launch_bounds__(COCO_NORM_THREADS, COCO_NORM_CTAS)
    norm_kernel(const __grid_constant__ NormTable<CAP> tab, const __grid_constant__ NormArgs a,
                NormSlot *slot) {
  __shared__ unsigned s_off[CAP + 1];
  const NormTable<CAP> *tp = &tab;
  hide(tp);  // for lookups that differ from lane to lane
  copy_offsets(s_off, tp->off, a.n);
  __syncthreads();
  const int n = a.n, lane = threadIdx.x & 31;
  const unsigned total = s_off[n];
  const unsigned nw = blockDim.x >> 5;
  unsigned begin = 1, end = 0;  // the tensor at hand
  int head = 0, tail = 0;
  const uint4 *p = nullptr;
  double sum = 0.0;
  for (unsigned u = blockIdx.x * nw + (threadIdx.x >> 5); u < (total + kUnit - 1) / kUnit;
       u += gridDim.x * nw) {
    const unsigned e = u * kUnit;
    if (e < begin || e >= end) {
      const int k = find_tensor(s_off, n, e);
      begin = s_off[k], end = s_off[k + 1];
      p = (const uint4 *)tab.g[k];
      head = tab.head[k], tail = tab.tail[k];
    }
    uint4 q[kDepth];
    if (e + kUnit <= end) {
#pragma unroll
      for (int k = 0; k < kDepth; ++k) q[k] = p[e - begin + lane + 32 * k];
      if (head && e == begin && lane == 0) q[0] = masked<GT>(q[0], head, 0);
      if (tail && e + kUnit == end && lane == 31) q[kDepth - 1] = masked<GT>(q[kDepth - 1], 0, tail);
    } else {  // several tensors: every group looks up its own, between the warp's first and last
      int t_at[kDepth + 1];
#pragma unroll
      for (int k = 0; k <= kDepth; ++k) t_at[k] = find_tensor(s_off, n, min(e + 32 * k, total - 1));
#pragma unroll
      for (int k = 0; k < kDepth; ++k) {
        const unsigned x = e + lane + 32 * k;
        q[k] = make_uint4(0u, 0u, 0u, 0u);
        if (x < total) {
          const int t = bisect(t_at[k], t_at[k + 1], x, [&](int y) { return s_off[y]; });
          q[k] = ((const uint4 *)tp->g[t])[x - s_off[t]];
          const int h = x == s_off[t] ? tp->head[t] : 0, l = x == s_off[t + 1] - 1 ? tp->tail[t] : 0;
          if (h | l) q[k] = masked<GT>(q[k], h, l);
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int k = 0; k < kDepth; ++k) sum += squares<GT>(q[k]);
  }
  double all = 0.0;
  if (!rank_sum<1>(sum, &slot->count, reinterpret_cast<double *>(slot + 1), all) || threadIdx.x != 0) return;
  if (!a.first) all += ld_volatile_f64(&slot->so_far);
  if (a.last) put_norm(a, a.out, all);
  else slot->so_far = all;
}

template <typename GT, int RB>
__global__ void __launch_bounds__(COCO_NORM_THREADS)
    norm_peer_kernel(const __grid_constant__ PeerArgs pa, const __grid_constant__ NormArgs a) {
  __shared__ int s_ok;
  const PeerRank &pr = pa.ranks[blockIdx.y];
  FlagPage *me = pr.flags[pr.rank];
  const int R = pa.world, lane = threadIdx.x & 31;
  const bool started = list_start_barrier(pr, pa, &s_ok);
  const PeerPiece *pieces = pr.pieces;
  const unsigned units = started ? (pr.groups + kListUnitGroups - 1) / kListUnitGroups : 0;
  const unsigned nw = blockDim.x >> 5;
  // Every CTA waits for itself, and some may have given up where others, which came
  // later, did not: a sum without their part is no number, on every rank.
  double sum = started ? 0.0 : __longlong_as_double(0x7ff8000000000000ll);
  auto add = [&](float x) { sum += (double)x * (double)x; };
  for (unsigned u = blockIdx.x * nw + (threadIdx.x >> 5); u < units; u += gridDim.x * nw) {
    const unsigned e = u * kListUnitGroups;
    const int k = bisect(0, pr.n - 1, e, [&](int x) { return pieces[x].off; });
    const PeerPiece &pc = pieces[k];
    const size_t done = (size_t)(e - pc.off) * kListGroup, left = (size_t)pc.len - done;
    const size_t i = (size_t)pc.begin + done;
    if (left >= kListUnit && pc.aligned16) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float x[4];
        sum_grad4<RB, GT>(pc.g, R, i + 4 * lane + 128 * q, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) add(x[j]);
      }
    } else if (pc.end - e >= kListUnitGroups || pc.end == pr.groups) {
      for (int o = lane; o < kListUnit && o < left; o += 32) add(sum_grad1<RB, GT>(pc.g, R, i + o));
    } else if (e + lane < pr.groups) {
      const unsigned el = e + lane;
      const PeerPiece &pl = pieces[bisect(k, pr.n - 1, el, [&](int x) { return pieces[x].off; })];
      const size_t dl = (size_t)(el - pl.off) * kListGroup, ll = (size_t)pl.len - dl;
      for (int o = 0; o < kListGroup && o < ll; ++o)
        add(sum_grad1<RB, GT>(pl.g, R, (size_t)pl.begin + dl + o));
    }
    __syncwarp();
  }
  double all = 0.0;
  if (!rank_sum<2>(sum, &me->norm_count, &me->cta_part[0][0], all)) return;
  // The rank's last CTA: nothing of this rank reads gradients any more.  Its sum
  // goes to every rank, and the others' arrival says the same of them.
  if (threadIdx.x >= 32) return;
  all = __shfl_sync(0xffffffffu, all, 0);
  if (started && lane < R) {
    volatile double *dst = pr.flags[lane]->norm_part[pr.rank];
    dst[0] = all;
    __threadfence_system();
    st_release_sys(&pr.flags[lane]->norm_flag[pr.rank], pa.seq);
  }
  __syncwarp();
  const int late = started ? warp_wait_peers(me->norm_flag, R, pr.rank, pa.seq, pa.timeout_ns) : pr.rank;
  if (lane != 0) return;
  if (started && late < 0) {
    double total = 0.0;
    for (int p = 0; p < R; ++p) total += ld_volatile_f64(&me->norm_part[p][0]);
    put_norm(a, pr.norm_out, total);
  } else {
    if (started) record_status(me, cocoTimeout, pr.rank, kPhaseNorm, late, pa.seq);
    pr.norm_out[0] = __uint_as_float(0x7fc00000u);  // whoever reads it skips the step
    pr.norm_out[1] = 0.f;
  }
}

template <int CAP> using Kernel = void (*)(const NormTable<CAP>, const NormArgs, NormSlot *);
template <int CAP> Kernel<CAP> pick(cocoDataType_t g) {
  switch (g) {
    case cocoFloat32: return norm_kernel<float, CAP>;
    case cocoFloat16: return norm_kernel<__half, CAP>;
    case cocoBfloat16: return norm_kernel<__nv_bfloat16, CAP>;
  }
  return nullptr;
}
typedef void (*PeerKernel)(const PeerArgs, const NormArgs);
template <typename GT> PeerKernel pick_world(int world) {
  return world <= 2 ? norm_peer_kernel<GT, 2> : world <= 4 ? norm_peer_kernel<GT, 4> : norm_peer_kernel<GT, 8>;
}
PeerKernel pick_peer(cocoDataType_t g, int world) {
  switch (g) {
    case cocoFloat32: return pick_world<float>(world);
    case cocoFloat16: return pick_world<__half>(world);
    case cocoBfloat16: return pick_world<__nv_bfloat16>(world);
  }
  return nullptr;
}

}  // namespace

int grad_norm_threads() { return COCO_NORM_THREADS; }
int grad_norm_ctas_per_sm() { return COCO_NORM_CTAS; }
int grad_norm_groups_per_warp() { return kUnit; }

template <int CAP>
cudaError_t launch_grad_norm(cocoDataType_t g_type, const NormTable<CAP> &table,
                             const NormArgs &args, NormSlot *slot, int ctas, cudaStream_t stream) {
  const Kernel<CAP> k = pick<CAP>(g_type);
  if (!k) return cudaErrorInvalidValue;
  void *params[] = {(void *)&table, (void *)&args, (void *)&slot};
  return cudaLaunchKernel((const void *)k, dim3(ctas), dim3(COCO_NORM_THREADS), params, 0, stream);
}
template cudaError_t launch_grad_norm<kNormCapSmall>(cocoDataType_t, const NormTable<kNormCapSmall> &,
                                                     const NormArgs &, NormSlot *, int, cudaStream_t);
template cudaError_t launch_grad_norm<kNormCapLarge>(cocoDataType_t, const NormTable<kNormCapLarge> &,
                                                     const NormArgs &, NormSlot *, int, cudaStream_t);

cudaError_t launch_grad_norm_peers(cocoDataType_t g_type, const PeerArgs &peers, const NormArgs &args,
                                   const ListLaunch &cfg, cudaStream_t stream) {
  const PeerKernel k = pick_peer(g_type, peers.world);
  if (!k) return cudaErrorInvalidValue;
  void *params[] = {(void *)&peers, (void *)&args};
  const dim3 grid(cfg.ctas, cfg.nvirt);
  if (cfg.cooperative)
    return cudaLaunchCooperativeKernel((const void *)k, grid, dim3(cfg.threads), params, 0, stream);
  return cudaLaunchKernel((const void *)k, grid, dim3(cfg.threads), params, 0, stream);
}
cudaError_t grad_norm_peers_occupancy(cocoDataType_t g_type, int world, int threads, int *ctas_per_sm) {
  const PeerKernel k = pick_peer(g_type, world);
  if (!k) return cudaErrorInvalidValue;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(ctas_per_sm, (const void *)k, threads, 0);
}

}  // namespace coco
