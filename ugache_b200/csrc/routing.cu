// Routing kernels: the plan (a stable counting sort of ids) and the rows' way to their groups' order
// and back, weighted, with the inner products that the weights' gradients are.
#include "routing.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace ugc {

namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ void wait_for_launch_ahead() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void release_launch_behind() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kern)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t s, bool pdl,
                   const Args&... args) {
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// ------------------------------------------------------------------------------------
// plan
// ------------------------------------------------------------------------------------
// A tile of ids is ranked inside one CTA: every warp takes a run of consecutive ids and counts them
// per group in shared memory (16-bit, a run is short), 32 at a time in order, equal ids of a step meeting
// by match; a scan over the warps and one over the groups give every id its place.  Several CTAs
// first count their parts (one more launch) and then add up the counts of the parts ahead.

constexpr int kPlanSteps = 8;                       // ids a lane holds
constexpr uint32_t kPlanBlock = 1024;
constexpr uint32_t kPlanTile = kPlanBlock * kPlanSteps;

template <typename IdT>
__device__ __forceinline__ uint32_t group_of(IdT id, uint32_t n_groups) {
  return (unsigned long long)(long long)id < n_groups ? (uint32_t)id : n_groups;  // one more group: no group
}

// Exclusive scan of v[0 .. n) in shared memory by the whole CTA; partial: one word per warp.
__device__ __forceinline__ void block_exclusive_scan(uint32_t* v, uint32_t n, uint32_t* partial) {
  const uint32_t per = (n + blockDim.x - 1) / blockDim.x, first = threadIdx.x * per;
  uint32_t sum = 0;
  for (uint32_t i = 0; i < per; i++)
    if (first + i < n) sum += v[first + i];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(kFull, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) partial[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const uint32_t n_warp = blockDim.x >> 5;
    const uint32_t mine = lane < n_warp ? partial[lane] : 0;
    uint32_t run = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(kFull, run, d);
      if (lane >= d) run += o;
    }
    partial[lane] = run - mine;
  }
  __syncthreads();
  uint32_t at = partial[warp] + inc - sum;
  for (uint32_t i = 0; i < per; i++)
    if (first + i < n) {
      const uint32_t c = v[first + i];
      v[first + i] = at;
      at += c;
    }
  __syncthreads();
}

// counts[c * (n_groups + 1) + g] = ids of group g in part c of the batch
template <typename IdT>
__global__ void __launch_bounds__(kPlanBlock) plan_count_kernel(const IdT* __restrict__ ids, uint32_t n, uint32_t n_groups,
                                                                uint32_t part, uint32_t* __restrict__ counts) {
  extern __shared__ uint32_t hist[];
  wait_for_launch_ahead();
  release_launch_behind();
  const uint32_t G1 = n_groups + 1;
  for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) hist[g] = 0;
  __syncthreads();
  const uint32_t begin = blockIdx.x * part, end = min(n, begin + part);
  for (uint32_t base = begin; base < end; base += blockDim.x) {
    const uint32_t i = base + threadIdx.x;
    const uint32_t g = i < end ? group_of(ids[i], n_groups) : 0xffffffffu;
    const unsigned same = __match_any_sync(kFull, g);
    if (i < end && (threadIdx.x & 31) == (uint32_t)__ffs(same) - 1) atomicAdd(&hist[g], __popc(same));
  }
  __syncthreads();
  for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) counts[(size_t)blockIdx.x * G1 + g] = hist[g];
}

// counts == nullptr: one CTA does the whole batch.
template <typename IdT>
__global__ void __launch_bounds__(kPlanBlock)
    plan_place_kernel(const IdT* __restrict__ ids, uint32_t n, uint32_t n_groups, uint32_t part, const uint32_t* counts,
                      int32_t* __restrict__ offsets, int32_t* __restrict__ order, int32_t* __restrict__ position) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t partial[32];
  const uint32_t G1 = n_groups + 1, n_warp = blockDim.x >> 5;
  uint32_t* start = smem;                                             // [G1] next place of each group
  uint32_t* ahead = smem + G1;                                        // [G1] counts of the parts ahead
  uint16_t* seen = reinterpret_cast<uint16_t*>(smem + 2 * G1);        // [n_warp][G1]
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint16_t* mine = seen + (size_t)warp * G1;
  const uint32_t begin = blockIdx.x * part, end = min(n, begin + part);

  bool first = true;
  if (!counts) wait_for_launch_ahead();  // with counts, the launch ahead started behind everything that wrote the ids
  for (uint32_t tile = begin; first || tile < end; tile += blockDim.x * kPlanSteps) {
    for (uint32_t i = threadIdx.x; i < n_warp * G1; i += blockDim.x) seen[i] = 0;
    __syncthreads();
    // ranks inside the warp's run
    const uint32_t steps = min((uint32_t)kPlanSteps, (min(end - min(tile, end), blockDim.x * kPlanSteps) + blockDim.x - 1) / blockDim.x);
    const uint32_t run = tile + warp * (32 * steps);
    uint32_t group[kPlanSteps], rank[kPlanSteps];
#pragma unroll
    for (int s = 0; s < kPlanSteps; s++) {
      const uint32_t i = run + s * 32 + lane;
      group[s] = (uint32_t)s < steps && i < end ? group_of(ids[i], n_groups) : 0xffffffffu;
    }
#pragma unroll
    for (int s = 0; s < kPlanSteps; s++) {
      if ((uint32_t)s >= steps) break;
      const bool live = group[s] != 0xffffffffu;
      const unsigned same = __match_any_sync(kFull, group[s]);
      const uint32_t before = live ? mine[group[s]] : 0;
      __syncwarp();
      if (live && lane == (uint32_t)__ffs(same) - 1) mine[group[s]] = (uint16_t)(before + __popc(same));
      __syncwarp();
      rank[s] = before + __popc(same & ((1u << lane) - 1));
    }
    __syncthreads();
    // the warps' counts become places inside the tile; the tile's counts go to `ahead` or `start`
    if (first) {
      if (counts) wait_for_launch_ahead();
      for (uint32_t g = threadIdx.x; g < 2 * G1; g += blockDim.x) smem[g] = 0;
      __syncthreads();
      if (counts) {
        const uint32_t slices = max(1u, blockDim.x / G1), slice = threadIdx.x / G1;
        for (uint32_t g = threadIdx.x % G1; slice < slices && g < G1; g += blockDim.x) {
          uint32_t total = 0, before = 0;
#pragma unroll 4
          for (uint32_t c = slice; c < gridDim.x; c += slices) {
            const uint32_t x = __ldcg(&counts[(size_t)c * G1 + g]);
            total += x;
            if (c < blockIdx.x) before += x;
          }
          atomicAdd(&start[g], total);
          atomicAdd(&ahead[g], before);
        }
      } else {
        for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) {
          uint32_t total = 0;
          for (uint32_t w = 0; w < n_warp; w++) total += seen[(size_t)w * G1 + g];
          start[g] = total;
        }
      }
      __syncthreads();
      block_exclusive_scan(start, G1, partial);
      if (blockIdx.x == 0)
        for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) offsets[g] = (int32_t)start[g];
      __syncthreads();
      for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) start[g] += ahead[g];
      __syncthreads();
      first = false;
    }
    // ahead[g] becomes the group's place at the tile's start, start[g] the one at the next tile's
    for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) {
      uint32_t at = 0;
      for (uint32_t w = 0; w < n_warp; w++) {
        const uint32_t c = seen[(size_t)w * G1 + g];
        seen[(size_t)w * G1 + g] = (uint16_t)at;
        at += c;
      }
      ahead[g] = start[g];
      start[g] += at;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kPlanSteps; s++) {
      const uint32_t g = group[s];
      if ((uint32_t)s >= steps || g == 0xffffffffu) break;  // a run's ids are a prefix of its lanes' steps
      const uint32_t i = run + s * 32 + lane, at = ahead[g] + mine[g] + rank[s];
      order[at] = (int32_t)i;
      position[i] = g < n_groups ? (int32_t)at : -1;
    }
    __syncthreads();
  }
}

// Parts (CTAs) of a batch and the ids of one, a multiple of a tile.
void plan_parts(uint32_t n, uint32_t* parts, uint32_t* part) {
  constexpr uint32_t kMost = 148;
  const uint32_t tiles = (n + kPlanTile - 1) / kPlanTile, each = (tiles + kMost - 1) / kMost;
  *part = std::max(1u, each) * kPlanTile;
  *parts = std::max(1u, (n + *part - 1) / *part);
}

// ------------------------------------------------------------------------------------
// rows
// ------------------------------------------------------------------------------------

template <int BYTES>
struct Piece;
template <>
struct __align__(16) Piece<16> {
  uint32_t v[4];
};
template <>
struct __align__(4) Piece<4> {
  uint32_t v[1];
};
template <>
struct __align__(2) Piece<2> {
  uint16_t v[1];
};

template <typename E>
__device__ __forceinline__ float widen(E x);
template <>
__device__ __forceinline__ float widen(float x) { return x; }
template <>
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename E>
__device__ __forceinline__ E narrow(float x);
template <>
__device__ __forceinline__ float narrow(float x) { return x; }
template <>
__device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }

template <typename E, int BYTES>
struct Floats {
  static constexpr int N = BYTES / (int)sizeof(E);
  float f[N];
  __device__ __forceinline__ void from(const Piece<BYTES>& p) {
    const E* e = reinterpret_cast<const E*>(&p);
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = widen<E>(e[i]);
  }
  __device__ __forceinline__ Piece<BYTES> rounded() const {
    Piece<BYTES> p;
    E* e = reinterpret_cast<E*>(&p);
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = narrow<E>(f[i]);
    return p;
  }
};

template <int BYTES>
__device__ __forceinline__ Piece<BYTES> ld_piece(const void* base, long long stride, uint32_t row, uint32_t piece) {
  return *reinterpret_cast<const Piece<BYTES>*>(static_cast<const char*>(base) + (long long)row * stride + (size_t)piece * BYTES);
}
template <int BYTES>
__device__ __forceinline__ void st_piece(void* base, long long stride, uint32_t row, uint32_t piece, const Piece<BYTES>& p) {
  *reinterpret_cast<Piece<BYTES>*>(static_cast<char*>(base) + (long long)row * stride + (size_t)piece * BYTES) = p;
}

// Rows of row_out that no choice took.
template <int BYTES>
__device__ __forceinline__ void zero_tail(const RouteRows& p, uint32_t pieces) {
  if (!p.n_routed) return;
  const uint32_t routed = min((uint32_t)max(*p.n_routed, 0), p.n_rows);
  const Piece<BYTES> zero = {};
  const unsigned long long n = (unsigned long long)(p.n_rows - routed) * pieces;
  for (unsigned long long u = (unsigned long long)blockIdx.x * blockDim.x + threadIdx.x; u < n;
       u += (unsigned long long)gridDim.x * blockDim.x)
    st_piece<BYTES>(p.row_out, p.row_out_stride, routed + (uint32_t)(u / pieces), (uint32_t)(u % pieces), zero);
}

constexpr int kRowsBlock = 256;

// A thread has one piece of one token's row and takes it to all the rows of the token's choices.
template <typename E, int BYTES, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsBlock) spread_kernel(RouteRows p, uint32_t pieces) {
  wait_for_launch_ahead();
  release_launch_behind();
  const unsigned long long u = (unsigned long long)blockIdx.x * kRowsBlock + threadIdx.x;
  const uint32_t t = (uint32_t)(u / pieces), c = (uint32_t)(u % pieces);
  if (t < p.n_tokens) {
    const Piece<BYTES> in = ld_piece<BYTES>(p.token_in, p.token_in_stride, t, c);
    Floats<E, BYTES> x;
    if (WEIGHTED) x.from(in);
    const size_t at = (size_t)t * p.k;
    for (uint32_t j = 0; j < p.k; j++) {
      const uint32_t row = (uint32_t)p.position[at + j];
      if (row >= p.n_rows) continue;
      if (WEIGHTED) {
        const float w = p.weights[at + j];
        Floats<E, BYTES> y;
#pragma unroll
        for (int i = 0; i < x.N; i++) y.f[i] = w * x.f[i];
        st_piece<BYTES>(p.row_out, p.row_out_stride, row, c, y.rounded());
      } else {
        st_piece<BYTES>(p.row_out, p.row_out_stride, row, c, in);
      }
    }
  }
  zero_tail<BYTES>(p, pieces);
}

// A thread sums one piece of one token's row over its choices, in their order, in fp32.
template <typename E, int BYTES, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsBlock) gather_kernel(RouteRows p, uint32_t pieces) {
  wait_for_launch_ahead();
  release_launch_behind();
  const unsigned long long u = (unsigned long long)blockIdx.x * kRowsBlock + threadIdx.x;
  const uint32_t t = (uint32_t)(u / pieces), c = (uint32_t)(u % pieces);
  if (t >= p.n_tokens) return;
  constexpr int kFlight = 4;
  const size_t at = (size_t)t * p.k;
  Floats<E, BYTES> sum = {};
  for (uint32_t j0 = 0; j0 < p.k; j0 += kFlight) {
    uint32_t row[kFlight];
    float w[kFlight];
    Piece<BYTES> in[kFlight];
#pragma unroll
    for (int j = 0; j < kFlight; j++) {
      row[j] = j0 + j < p.k ? (uint32_t)p.position[at + j0 + j] : kFull;
      if (row[j] < p.n_rows) {
        in[j] = ld_piece<BYTES>(p.row_in, p.row_in_stride, row[j], c);
        if (WEIGHTED) w[j] = p.weights[at + j0 + j];
      }
    }
#pragma unroll
    for (int j = 0; j < kFlight; j++) {
      if (row[j] >= p.n_rows) continue;
      Floats<E, BYTES> x;
      x.from(in[j]);
#pragma unroll
      for (int i = 0; i < x.N; i++) sum.f[i] = WEIGHTED ? fmaf(w[j], x.f[i], sum.f[i]) : sum.f[i] + x.f[i];
    }
  }
  st_piece<BYTES>(p.token_out, p.token_out_stride, t, c, sum.rounded());
}

// With inner products: `group` threads (a power of two) have one token; they walk its row together,
// a lane sums its share of each choice's product in fp32, the shares are added in a fixed order.
constexpr int kDots = 8;  // choices a pass

template <typename E, int BYTES, bool WEIGHTED, bool SPREAD>
__global__ void __launch_bounds__(kRowsBlock) dots_kernel(RouteRows p, uint32_t pieces, uint32_t group) {
  wait_for_launch_ahead();
  release_launch_behind();
  __shared__ float share[kRowsBlock / 32][kDots];
  const uint32_t in_group = threadIdx.x & (group - 1);
  const uint32_t t = blockIdx.x * (kRowsBlock / group) + threadIdx.x / group;
  const bool live = t < p.n_tokens;
  const size_t at = (size_t)t * p.k;
  for (uint32_t j0 = 0; j0 < p.k; j0 += kDots) {
    uint32_t row[kDots];
    float w[kDots], dot[kDots];
#pragma unroll
    for (int j = 0; j < kDots; j++) {
      dot[j] = 0.f;
      row[j] = live && j0 + j < p.k ? (uint32_t)p.position[at + j0 + j] : kFull;
      w[j] = WEIGHTED && row[j] < p.n_rows ? p.weights[at + j0 + j] : 1.f;
    }
    for (uint32_t c = in_group; live && c < pieces; c += group) {
      Floats<E, BYTES> x, y;
      x.from(ld_piece<BYTES>(p.token_in, p.token_in_stride, t, c));
      Floats<E, BYTES> sum = {};
#pragma unroll
      for (int j = 0; j < kDots; j++) {
        if (row[j] >= p.n_rows) continue;
        y.from(ld_piece<BYTES>(p.row_in, p.row_in_stride, row[j], c));
#pragma unroll
        for (int i = 0; i < x.N; i++) {
          dot[j] = fmaf(x.f[i], y.f[i], dot[j]);
          if (!SPREAD) sum.f[i] = WEIGHTED ? fmaf(w[j], y.f[i], sum.f[i]) : sum.f[i] + y.f[i];
        }
        if (SPREAD) {
#pragma unroll
          for (int i = 0; i < x.N; i++) y.f[i] = WEIGHTED ? w[j] * x.f[i] : x.f[i];
          st_piece<BYTES>(p.row_out, p.row_out_stride, row[j], c, y.rounded());
        }
      }
      if (!SPREAD && j0 == 0) {  // choices past the first pass join the sum here, their products come later
        for (uint32_t j = kDots; j < p.k; j++) {
          const uint32_t r = (uint32_t)p.position[at + j];
          if (r >= p.n_rows) continue;
          const float v = WEIGHTED ? p.weights[at + j] : 1.f;
          y.from(ld_piece<BYTES>(p.row_in, p.row_in_stride, r, c));
#pragma unroll
          for (int i = 0; i < x.N; i++) sum.f[i] = WEIGHTED ? fmaf(v, y.f[i], sum.f[i]) : sum.f[i] + y.f[i];
        }
        st_piece<BYTES>(p.token_out, p.token_out_stride, t, c, sum.rounded());
      }
    }
    const uint32_t width = min(group, 32u);
#pragma unroll
    for (int j = 0; j < kDots; j++)
      for (uint32_t d = width >> 1; d; d >>= 1) dot[j] += __shfl_xor_sync(kFull, dot[j], d);
    if (group > 32) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int j = 0; j < kDots; j++) share[threadIdx.x >> 5][j] = dot[j];
      }
      __syncthreads();
      if (in_group < kDots && live && j0 + in_group < p.k) {
        float sum = 0.f;
        for (uint32_t i = 0; i < group / 32; i++) sum += share[(threadIdx.x >> 5) + i][in_group];
        p.dots[at + j0 + in_group] = sum;
      }
    } else if (live && in_group == 0) {
#pragma unroll
      for (int j = 0; j < kDots; j++)
        if (j0 + j < p.k) p.dots[at + j0 + j] = dot[j];
    }
  }
  if (SPREAD) zero_tail<BYTES>(p, pieces);
}

// Widest piece of 16, 4 (or 2) bytes that divides the rows and every address and stride in use.
int piece_bytes(const RouteRows& p, int elem_bytes) {
  unsigned long long bits = (unsigned long long)p.dim * elem_bytes;
  auto add = [&](const void* q, long long stride) {
    if (q) bits |= reinterpret_cast<uintptr_t>(q) | (unsigned long long)stride;
  };
  add(p.token_in, p.token_in_stride);
  add(p.token_out, p.token_out_stride);
  add(p.row_in, p.row_in_stride);
  add(p.row_out, p.row_out_stride);
  return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
}

template <typename E, int BYTES>
cudaError_t rows_launch(const RouteRows& p, bool spread, cudaStream_t stream) {
  const uint32_t pieces = (uint32_t)((unsigned long long)p.dim * sizeof(E) / BYTES);
  const bool weighted = p.weights != nullptr;
  if (p.dots) {
    uint32_t group = 1;
    while (group < pieces && group < (uint32_t)kRowsBlock) group *= 2;
    const uint32_t per = kRowsBlock / group, grid = (p.n_tokens + per - 1) / per;
    auto kern = spread ? (weighted ? dots_kernel<E, BYTES, true, true> : dots_kernel<E, BYTES, false, true>)
                       : (weighted ? dots_kernel<E, BYTES, true, false> : dots_kernel<E, BYTES, false, false>);
    return launch(kern, grid, kRowsBlock, 0, stream, true, p, pieces, group);
  }
  const unsigned long long units = (unsigned long long)p.n_tokens * pieces;
  const unsigned long long grid = (units + kRowsBlock - 1) / kRowsBlock;
  if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
  auto kern = spread ? (weighted ? spread_kernel<E, BYTES, true> : spread_kernel<E, BYTES, false>)
                     : (weighted ? gather_kernel<E, BYTES, true> : gather_kernel<E, BYTES, false>);
  return launch(kern, (unsigned)grid, kRowsBlock, 0, stream, true, p, pieces);
}

cudaError_t rows_by_type(const RouteRows& p, int elem, bool spread, cudaStream_t stream) {
  if (p.n_tokens == 0) return cudaSuccess;
  const int bytes = piece_bytes(p, elem == kElemF32 ? 4 : 2);
  auto by_piece = [&](auto e) {
    using E = decltype(e);
    if (bytes == 16) return rows_launch<E, 16>(p, spread, stream);
    if constexpr (sizeof(E) == 2) {
      if (bytes == 2) return rows_launch<E, 2>(p, spread, stream);
    }
    return rows_launch<E, 4>(p, spread, stream);
  };
  if (elem == kElemF32) return by_piece(float{});
  if (elem == kElemF16) return by_piece(__half{});
  return by_piece(__nv_bfloat16{});
}

}  // namespace

size_t route_plan_scratch_bytes(uint32_t n, int n_groups) {
  uint32_t parts, part;
  plan_parts(n, &parts, &part);
  return parts > 1 ? (size_t)parts * (n_groups + 1) * sizeof(uint32_t) : 0;
}

cudaError_t launch_route_plan(const void* ids, int id_bytes, uint32_t n, int n_groups, int32_t* offsets,
                              int32_t* order, int32_t* position, void* scratch, cudaStream_t stream) {
  uint32_t parts, part;
  plan_parts(n, &parts, &part);
  const uint32_t G = (uint32_t)n_groups;
  uint32_t block = 128;
  while (block < n && block < kPlanBlock) block *= 2;
  const size_t smem = (size_t)(G + 1) * (2 * sizeof(uint32_t) + (block / 32) * sizeof(uint16_t));
  auto go = [&](auto id) {
    using IdT = decltype(id);
    const IdT* in = static_cast<const IdT*>(ids);
    uint32_t* counts = parts > 1 ? static_cast<uint32_t*>(scratch) : nullptr;
    if (counts) {
      cudaError_t e = launch(plan_count_kernel<IdT>, parts, kPlanBlock, (G + 1) * sizeof(uint32_t), stream, true, in, n, G,
                             part, counts);
      if (e != cudaSuccess) return e;
    }
    return launch(plan_place_kernel<IdT>, parts, block, smem, stream, true, in, n, G, part,
                  static_cast<const uint32_t*>(counts), offsets, order, position);
  };
  return id_bytes == 8 ? go((long long)0) : go((int32_t)0);
}

cudaError_t launch_route_spread(const RouteRows& p, int elem, cudaStream_t stream) { return rows_by_type(p, elem, true, stream); }
cudaError_t launch_route_gather(const RouteRows& p, int elem, cudaStream_t stream) { return rows_by_type(p, elem, false, stream); }

}  // namespace ugc
