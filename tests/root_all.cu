// The root of the 8-bit AdamW state, for every fp32 number from 0 to infinity, against the
// rounded root.  Prints how many differ: of neg_root, which takes 2^-100 and more, in its
// two places, and of neg_root_any.
#include <cstdio>

#include "pair_math.cuh"

namespace coco {
namespace {
__device__ unsigned long long g_differ[3];
__global__ void compare() {
  unsigned long long n[3] = {0, 0, 0};
  for (unsigned b = blockIdx.x * blockDim.x + threadIdx.x; b <= 0x7f800000u; b += gridDim.x * blockDim.x) {
    const float v = __uint_as_float(b);
    const unsigned root = __float_as_uint(__fsqrt_rn(v));
    if (v >= 0x1p-100f && b < 0x7f800000u) {
      float x, y;
      unpair(neg_root(pair(-v, -1.f)), x, y);
      n[0] += __float_as_uint(-x) != root || y != -1.f;
      unpair(neg_root(pair(-1.f, -v)), x, y);
      n[1] += __float_as_uint(-y) != root || x != -1.f;
    }
    n[2] += b == 0 ? neg_root_any(-v) != 0.f : __float_as_uint(-neg_root_any(-v)) != root;
  }
  for (int k = 0; k < 3; ++k) atomicAdd(&g_differ[k], n[k]);
}
}  // namespace
}  // namespace coco

int main() {
  unsigned long long n[3] = {1, 1, 1};
  coco::compare<<<148 * 4, 512>>>();
  const cudaError_t e = cudaMemcpyFromSymbol(n, coco::g_differ, sizeof(n));
  printf("%llu %llu %llu\n", n[0], n[1], n[2]);
  if (e != cudaSuccess) fprintf(stderr, "%s\n", cudaGetErrorString(e));
  return e != cudaSuccess;
}
