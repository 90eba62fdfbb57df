// Launchers of the routing operators: tokens grouped by an id, their rows moved to the groups'
// order and back, low-rank adapters applied per group.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace ugc {

// All launchers enqueue on `stream` of the current device and return the launch status; none synchronises.

constexpr int kRouteMaxGroups = 1024;
constexpr int kAdapterMaxRank = 128;

enum Elem : int { kElemF32 = 0, kElemF16 = 1, kElemBf16 = 2 };

// Stable counting sort of n ids into n_groups groups; ids outside [0, n_groups) come last.
//   offsets[g]    where group g starts in `order` (n_groups + 1 entries)
//   order[p]      index of the id at place p, a permutation of 0 .. n-1
//   position[i]   place of id i, -1 for an id outside the groups
size_t route_plan_scratch_bytes(uint32_t n, int n_groups);
cudaError_t launch_route_plan(const void* ids, int id_bytes, uint32_t n, int n_groups, int32_t* offsets,
                              int32_t* order, int32_t* position, void* scratch, cudaStream_t stream);

// Rows of tokens ([n_tokens, dim]) and rows in groups' order ([n_rows, dim]); strides in bytes.
struct RouteRows {
  const void* token_in;    // spread: source; gather with dots: the other factor
  void* token_out;         // gather: destination
  const void* row_in;      // gather: source; spread with dots: the other factor
  void* row_out;           // spread: destination
  const float* weights;    // [n_tokens, k] or nullptr
  float* dots;             // [n_tokens, k] or nullptr
  const int32_t* position; // [n_tokens, k]
  const int32_t* n_routed; // spread: rows of row_out from *n_routed to n_rows are zeroed; nullptr: left alone
  long long token_in_stride, token_out_stride, row_in_stride, row_out_stride;
  uint32_t n_tokens, k, n_rows, dim;
};
// row_out[position[t,j]] = weights[t,j] * token_in[t];  dots[t,j] = <token_in[t], row_in[position[t,j]]>
cudaError_t launch_route_spread(const RouteRows& p, int elem, cudaStream_t stream);
// token_out[t] = sum_j weights[t,j] * row_in[position[t,j]];  dots as above
cudaError_t launch_route_gather(const RouteRows& p, int elem, cudaStream_t stream);

// out[t] = base[t] + scale[a] * (x[t] down[a]^T) up[a]^T, a = group of token t; strides in elements.
struct AdapterParams {
  const void *base, *x, *down, *up;
  void* out;
  const float* scale;  // per group, or nullptr
  const int32_t *offsets, *order;
  long long base_stride, x_stride, down_stride, up_stride, out_stride;
  uint32_t n_tokens, n_groups, rank, dim, out_dim;
};
// scratch: adapter_scratch_bytes, 16-byte aligned
size_t adapter_scratch_bytes(uint32_t n_tokens, uint32_t n_groups, uint32_t rank, uint32_t dim, uint32_t out_dim);
cudaError_t launch_adapter_add(const AdapterParams& p, int elem, void* scratch, cudaStream_t stream);
cudaError_t adapter_stalled(uint32_t* count);

}  // namespace ugc
