// One rank of two whose peer is late for some of its CTAs: the kernels over lists of
// tensors, launched with more CTAs than the GPU holds at once and a short time limit.
// The CTAs that run first wait for a flag that nobody sets, give up and say so in the
// status word; as soon as the host reads that there, it sets the peer's flag, and the
// CTAs that come after find it.  Every wait is bounded by the limit.
//   late_rank norm | adamw | adamw8  [in-time]
// prints one line of JSON.  in-time: the flag is set before the launch.
#include <chrono>
#include <cstdio>
#include <cstring>
#include <vector>

#include "list_step.cuh"

using namespace coco;

#define CHECK(x)                                                             \
  do {                                                                       \
    cudaError_t e_ = (x);                                                    \
    if (e_ != cudaSuccess) {                                                 \
      fprintf(stderr, "%s: %s\n", #x, cudaGetErrorString(e_));               \
      return 2;                                                              \
    }                                                                        \
  } while (0)

template <typename T> static cudaError_t to_device(T *dst, const T &x, cudaStream_t s) {
  return cudaMemcpyAsync(dst, &x, sizeof(T), cudaMemcpyHostToDevice, s);
}

int main(int argc, char **argv) {
  if (argc < 2) return 2;
  const bool norm = !strcmp(argv[1], "norm"), quant = !strcmp(argv[1], "adamw8");
  const bool in_time = argc > 2 && !strcmp(argv[2], "in-time");
  cudaDeviceProp prop;
  CHECK(cudaGetDeviceProperties(&prop, 0));
  const int threads = norm ? grad_norm_threads() : adamw_peer_threads();
  int occ = 0;
  CHECK(norm ? grad_norm_peers_occupancy(cocoFloat32, 2, threads, &occ)
             : adamw_peers_occupancy(quant, cocoFloat32, 2, threads, &occ));
  const int ctas = 3 * occ * prop.multiProcessorCount;  // three times what runs at once
  if (ctas > kMaxCtasPerRank) return 2;
  const size_t n = (size_t)ctas * (threads / 32) * kListUnit;  // one unit per warp

  cudaStream_t run, side;
  CHECK(cudaStreamCreateWithFlags(&run, cudaStreamNonBlocking));
  CHECK(cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking));
  FlagPage *page[2];
  float *g, *w[2], *out;
  char *m, *v;
  unsigned char *scale;
  PeerPiece *piece_dev;
  PeerRank *rank_dev;
  for (int r = 0; r < 2; ++r) {
    CHECK(cudaMalloc(&page[r], sizeof(FlagPage)));
    CHECK(cudaMemset(page[r], 0, sizeof(FlagPage)));
    CHECK(cudaMalloc(&w[r], n * 4));
    CHECK(cudaMemset(w[r], 0, n * 4));
  }
  CHECK(cudaMalloc(&g, n * 4));
  std::vector<float> ones(n, 1.0f);
  CHECK(cudaMemcpy(g, ones.data(), n * 4, cudaMemcpyHostToDevice));
  CHECK(cudaMalloc(&m, n * 4));
  CHECK(cudaMalloc(&v, n * 4));
  CHECK(cudaMalloc(&scale, n / kListUnit * 2));
  CHECK(cudaMemset(m, 0, n * 4));
  CHECK(cudaMemset(v, 0, n * 4));
  CHECK(cudaMemset(scale, 0, n / kListUnit * 2));
  CHECK(cudaMalloc(&out, 8));
  CHECK(cudaMemset(out, 0, 8));
  CHECK(cudaMalloc(&piece_dev, sizeof(PeerPiece)));
  CHECK(cudaMalloc(&rank_dev, sizeof(PeerRank)));

  const unsigned long long seq = 1;
  PeerPiece pc = {};
  pc.g[0] = pc.g[1] = g;
  pc.out[0] = w[0], pc.out[1] = w[1];
  pc.w = w[0];
  pc.len = n;
  pc.end = (unsigned)(n / kListGroup);
  pc.decays = pc.aligned16 = 1;
  PeerRank pr = {};
  pr.flags[0] = page[0], pr.flags[1] = page[1];
  pr.pieces = piece_dev;
  pr.n = 1, pr.rank = 0, pr.groups = pc.end;
  pr.m = m, pr.v = v, pr.scale = scale;
  pr.norm_out = out;
  pr.state_aligned = 1;
  CHECK(cudaMemcpy(piece_dev, &pc, sizeof(pc), cudaMemcpyHostToDevice));
  CHECK(cudaMemcpy(rank_dev, &pr, sizeof(pr), cudaMemcpyHostToDevice));
  // the peer's later flags are there already: only its start is late
  CHECK(to_device(&page[0]->norm_flag[1], seq, side));
  CHECK(to_device(&page[0]->done[1], seq, side));
  if (in_time) CHECK(to_device(&page[0]->arrive[1], seq, side));
  CHECK(cudaDeviceSynchronize());

  PeerArgs pa = {};
  pa.ranks = rank_dev;
  pa.world = 2, pa.seq = seq, pa.timeout_ns = 300ull * 1000 * 1000;
  ListLaunch cfg = {};
  cfg.ctas = ctas, cfg.threads = threads, cfg.nvirt = 1;
  NormArgs na = {};
  na.scale = 1.0, na.max_norm = 1.0;
  AdamWArgs aa = {};
  aa.grad_scale = 1.f, aa.beta1 = 0.9f, aa.beta2 = 0.999f, aa.omb1 = 0.1f, aa.omb2 = 0.001f;
  aa.neg_c1 = -1e-2f, aa.rs2 = 31.6f, aa.eps = 1e-8f, aa.decay = 1.f;
  aa.neg_beta2 = -aa.beta2, aa.neg_omb2 = -aa.omb2, aa.neg_rs2 = -aa.rs2;
  CHECK(norm ? launch_grad_norm_peers(cocoFloat32, pa, na, cfg, run)
             : launch_adamw_peers(quant, cocoFloat32, pa, aa, cfg, run));
  if (!in_time) {  // wait (10 s at most) until a CTA has given up, then let the peer arrive
    const auto t0 = std::chrono::steady_clock::now();
    int code = 0;
    while (code == 0 && std::chrono::steady_clock::now() - t0 < std::chrono::seconds(10)) {
      CHECK(cudaMemcpyAsync(&code, &page[0]->status[0], sizeof(int), cudaMemcpyDeviceToHost, side));
      CHECK(cudaStreamSynchronize(side));
    }
    CHECK(to_device(&page[0]->arrive[1], seq, side));
  }
  CHECK(cudaDeviceSynchronize());

  static FlagPage mine, peer;
  float res[2];
  std::vector<float> got(n);
  CHECK(cudaMemcpy(&mine, page[0], sizeof(mine), cudaMemcpyDeviceToHost));
  CHECK(cudaMemcpy(&peer, page[1], sizeof(peer), cudaMemcpyDeviceToHost));
  CHECK(cudaMemcpy(res, out, 8, cudaMemcpyDeviceToHost));
  CHECK(cudaMemcpy(got.data(), w[1], n * 4, cudaMemcpyDeviceToHost));
  size_t stepped = 0;
  for (float x : got) stepped += x != 0.f;
  printf("{\"n\": %zu, \"stepped\": %zu, \"norm\": \"%a\", \"clip\": \"%a\", \"status\": %d, \"phase\": %d, "
         "\"told_done\": %llu, \"told_norm\": %llu, \"told_part\": \"%a\", \"counters\": %u}\n",
         n, stepped, res[0], res[1], mine.status[0], mine.status[2], peer.done[0], peer.norm_flag[0],
         peer.norm_part[0][0], mine.done_count + mine.norm_count);
  return 0;
}
