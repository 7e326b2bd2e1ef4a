// Shared between the runtime (host) and the kernels over lists of tensors that
// are not part of the fused step's kernel: AdamW (adamw.cu) and the gradient
// norm (grad_norm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "coconet_device.h"
#include "coconet_rt.h"

namespace coco {

// A list lies in a virtual flat buffer, counted in groups of 8 elements.  A
// warp takes a unit of 32 groups at a time; with 8-bit moments a unit is also
// the block that shares a scale, and every tensor starts a new one.
constexpr int kListGroup = 8;
constexpr int kListUnitGroups = 32;
constexpr int kListUnit = kListGroup * kListUnitGroups;
static_assert(kListUnit == COCO_QUANT_BLOCK, "a warp's unit is a block of 8-bit state");

// World size 1: the list travels as a kernel parameter, so a call leaves
// nothing behind that another call, stream or captured graph could share.  The
// parameter space holds 32,764 bytes; longer lists take several launches.  The
// whole parameter is copied at every launch, hence the smaller form.
constexpr int kListCapSmall = 64, kListCapLarge = 1024;
template <int CAP> struct ListTable {
  const void *g[CAP];
  float *w[CAP];
  void *lp[CAP];
  unsigned off[CAP + 1];         // tensor's first group; [n]: one past the last
  unsigned char missing[CAP];    // elements of the tensor's groups that do not exist
  unsigned char flags[CAP];      // kListDecays, kListAligned
};

// weight decay applies; gradient, weights and copy start on 16 bytes and so does the state
enum : unsigned char { kListDecays = 1, kListAligned = 2 };
enum : int { kLpNone = 0, kLpF16 = 1, kLpBf16 = 2 };
enum : int { kListAdamW = 1, kListAdamWQuant = 2, kListGradNorm = 3 };  // operations on lists

struct AdamWArgs {
  void *m, *v;                   // state of this launch's first group on: fp32 m, v or codes of m, sqrt(v)
  unsigned char *scale;          // 8-bit state: two bytes per block
  const float *norm;             // {gradient norm, clip factor} or null
  unsigned long long flat0;      // place of that state in the flat state of the whole list
  FlagPage *page;                // world size 1: whose status word a copy that does not land is written to,
  unsigned long long timeout_ns; // after this time
  int n;                         // tensors in the table (world size 1)
  int lp_kind;
  int state_aligned;             // m and v start on 16 bytes
  unsigned key;                  // of the rounding bits
  float grad_scale, beta1, beta2, omb1, omb2;
  float neg_c1;                  // -lr / (1 - beta1^t)
  float rs2;                     // 1 / sqrt(1 - beta2^t)
  float neg_beta2, neg_omb2, neg_rs2;
  float eps, decay;              // decay: 1 - lr * weight_decay
};

// World sizes above 1: this rank's pieces of the list, in device memory.
struct PeerPiece {
  const void *g[kMaxRanks];      // the tensor's gradient on every rank, element 0
  void *out[kMaxRanks];          // its gathered weights (copy, or fp32) on every rank, element 0
  float *w;                      // own fp32 weights, element 0
  unsigned long long begin, len; // elements of the tensor inside the slice
  unsigned off, end;             // groups, counted from the slice's start; end: where the next piece starts
  int decays, aligned16;
};
struct PeerRank {
  FlagPage *flags[kMaxRanks];
  const PeerPiece *pieces;
  int n, rank;
  unsigned groups, pad_;         // groups up to the end of the last piece
  unsigned long long flat0;      // the slice's first element in the flat state
  void *m, *v;
  unsigned char *scale;
  const float *norm;
  float *norm_out;
  int state_aligned, pad2_;
};
struct PeerArgs {
  const PeerRank *ranks;         // [grid.y]
  int world, pad_;
  unsigned long long seq, timeout_ns;
};

// Gradient norm, world size 1: counted in groups of 16 bytes.  A tensor whose
// start is not 16-byte aligned is walked from the aligned address below it.
constexpr int kNormCapSmall = 64, kNormCapLarge = 1024;
template <int CAP> struct NormTable {
  const void *g[CAP];                  // rounded down to 16 bytes
  unsigned off[CAP + 1];               // first group; [n]: one past the last
  unsigned char head[CAP], tail[CAP];  // elements of the first / last group outside the tensor
};
// Partial sums of one call (device memory; the CTAs' sums lie behind it).  A call
// finds `count` at 0 and leaves it so.
struct NormSlot {
  unsigned count, pad_;  // CTAs that have posted their sums
  double so_far;         // sum of the list's earlier launches
};
struct NormArgs {
  int n;                         // tensors in the table (world size 1)
  int first, last;               // first / last launch of the list
  int pad_;
  float *out;                    // {norm, clip factor}
  double scale, max_norm;
};

struct ListLaunch {
  int ctas, threads, nvirt;
  bool cooperative;
};

// cudaErrorInvalidValue for a type that has no kernel.  packed: tensors of 256
// elements or more are not all aligned (aligned16), or the state is not.
template <int CAP>
cudaError_t launch_adamw(bool quant, bool packed, cocoDataType_t g_type, const ListTable<CAP> &table,
                         const AdamWArgs &args, size_t units, int device, int sm_count,
                         int max_ctas_per_sm, cudaStream_t stream);
unsigned adamw_rounding_key(uint64_t seed, int step);
cudaError_t launch_adamw_peers(bool quant, cocoDataType_t g_type, const PeerArgs &peers,
                               const AdamWArgs &args, const ListLaunch &cfg, cudaStream_t stream);
int adamw_peer_threads();
cudaError_t adamw_peers_occupancy(bool quant, cocoDataType_t g_type, int world, int threads,
                                  int *ctas_per_sm);

template <int CAP>
cudaError_t launch_grad_norm(cocoDataType_t g_type, const NormTable<CAP> &table,
                             const NormArgs &args, NormSlot *slot, int ctas, cudaStream_t stream);
int grad_norm_threads();
int grad_norm_ctas_per_sm();
int grad_norm_groups_per_warp();  // 16-byte groups a warp takes per pass
cudaError_t launch_grad_norm_peers(cocoDataType_t g_type, const PeerArgs &peers,
                                   const NormArgs &args, const ListLaunch &cfg,
                                   cudaStream_t stream);
cudaError_t grad_norm_peers_occupancy(cocoDataType_t g_type, int world, int threads,
                                      int *ctas_per_sm);

}  // namespace coco
