// What the routing and adapter kernels have in common.
#pragma once
#include <cstdint>

namespace ugc {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The sums of N (a power of two) values of each lane over `width` (N to 32) lanes: at every step a lane keeps half
// of its values and hands over the others, so that it takes N - 1 + log2(width / N) exchanges instead of N * log2(width).
// The order of the additions is the same wherever a value ends.  Returns the sum of value `which`.
template <int N>
__device__ __forceinline__ float sum_over_lanes(float (&v)[N], uint32_t width, uint32_t* which) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t at = 0;
  int n = N, d = (int)width / 2;
#pragma unroll
  for (int step = N; step > 1; step >>= 1, d >>= 1) {
    n = step / 2;
    const bool upper = lane & d;
#pragma unroll
    for (int i = 0; i < N / 2; i++)
      if (i < n) {
        const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
        v[i] = keep + __shfl_xor_sync(kFull, give, d);
      }
    if (upper) at += n;
  }
  for (; d; d >>= 1) v[0] += __shfl_xor_sync(kFull, v[0], d);
  *which = at;
  return v[0];
}

}  // namespace ugc
