// Routing kernels: the plan (a stable counting sort of ids) and the rows' way to their groups' order
// and back, weighted, with the inner products that the weights' gradients are.
#include "routing.cuh"

#include "lanes.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace ugc {

namespace {

__device__ __forceinline__ void wait_for_launch_ahead() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void release_launch_behind() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A word of shared memory as CTA `rank` of the cluster has it at the same place.
__device__ __forceinline__ uint32_t count_of(const uint32_t* mine, uint32_t rank) {
  uint32_t at, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// Shared memory of a CTA, at most: a plan's, two counts a group and the larger of 32 warps' counts and 8192 ids in order.
constexpr size_t kMostShared = (kRouteMaxGroups + 1) * 8 + 8192 * 8 + 1024;
static_assert((kRouteMaxGroups + 1) * 32 * 2 + 8 <= 8192 * 8 + 1024, "the counts are the smaller or fit as well");

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kern)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t s, bool pdl,
                   unsigned cluster, const Args&... args) {
  // with what is static (up to 9 KB) beyond the 48 KB that need no word; the same bound in every call, for another thread
  // may launch the kernel just now
  if (smem > 36 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  if (pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs++].val.clusterDim = {cluster, 1, 1};
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// ------------------------------------------------------------------------------------
// plan
// ------------------------------------------------------------------------------------
// A tile of ids is ranked inside one CTA: every warp takes a run of consecutive ids and counts them
// per group in shared memory (16-bit, a run is short), 32 at a time in order, equal ids of a step meeting
// by ballots; a scan over the warps and one over the groups give every id its place.  The CTAs of a cluster read
// one another's counts; more of them need a launch that counts first.  Latency bounds all of it.

constexpr int kPlanSteps = 8;                       // ids a lane holds
constexpr uint32_t kPlanBlock = 1024;
constexpr uint32_t kPlanTile = kPlanBlock * kPlanSteps;
constexpr uint32_t kNoId = 0xffffffffu;             // behind the last id

template <typename IdT>
__device__ __forceinline__ uint32_t group_of(IdT id, uint32_t n_groups) {
  return (unsigned long long)(long long)id < n_groups ? (uint32_t)id : n_groups;  // one more group: no group
}

// The lanes whose id is in the same group, bit by bit of the group (8192 ids in one CTA took 13.7 us with a match
// instruction, 12.1 with this).  Meant for lanes that are `live`.
__device__ __forceinline__ unsigned lanes_of_group(uint32_t group, bool live, uint32_t bits) {
  unsigned same = __ballot_sync(kFull, live);
#pragma unroll 4
  for (uint32_t b = 0; b < bits; b++) {
    const bool set = group >> b & 1;
    const unsigned with = __ballot_sync(kFull, set);
    same &= set ? with : ~with;
  }
  return same;
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

constexpr uint32_t kPlanCluster = 8;

// Eight parts a cluster: totals[c] = ids per group in the parts of cluster c, ahead[p] = those of the parts before
// part p in its cluster; rows of n_groups + 1.
template <typename IdT>
__global__ void __launch_bounds__(kPlanBlock) plan_count_kernel(const IdT* __restrict__ ids, uint32_t n, uint32_t n_groups,
                                                                uint32_t part, uint32_t* __restrict__ totals,
                                                                uint32_t* __restrict__ ahead) {
  extern __shared__ uint32_t hist[];
  wait_for_launch_ahead();
  release_launch_behind();
  const uint32_t G1 = n_groups + 1;
  for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) hist[g] = 0;
  __syncthreads();
  const uint32_t begin = min(n, blockIdx.x * part), end = min(n, begin + part);
  for (uint32_t base = begin; base < end; base += kPlanTile) {
    uint32_t group[kPlanSteps];
#pragma unroll
    for (int k = 0; k < kPlanSteps; k++) {
      const uint32_t i = base + k * kPlanBlock + threadIdx.x;
      group[k] = i < end ? group_of(ids[i], n_groups) : kNoId;
    }
#pragma unroll
    for (int k = 0; k < kPlanSteps; k++)  // at worst, all in one group, a lane at a time: as long as the ballots would take
      if (group[k] != kNoId) atomicAdd(&hist[group[k]], 1u);
  }
  cluster_arrive();
  cluster_wait();
  const uint32_t rank = blockIdx.x % kPlanCluster;
  for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) {
    uint32_t x[kPlanCluster], total = 0, before = 0;
#pragma unroll
    for (uint32_t c = 0; c < kPlanCluster; c++) x[c] = count_of(hist + g, c);
#pragma unroll
    for (uint32_t c = 0; c < kPlanCluster; c++) {
      total += x[c];
      before += c < rank ? x[c] : 0;
    }
    ahead[(size_t)blockIdx.x * G1 + g] = before;
    if (rank == 0) totals[(size_t)(blockIdx.x / kPlanCluster) * G1 + g] = total;
  }
  cluster_arrive();
  cluster_wait();  // nobody leaves while its counts are being read
}

// Who shares the batch: one CTA has it all; the CTAs of one cluster, which read one another's counts through
// distributed shared memory; or parts that plan_count_kernel has counted.
enum class Shared { kNot, kCluster, kParts };

template <typename IdT, Shared SHARED>
__global__ void __launch_bounds__(kPlanBlock)
    plan_place_kernel(const IdT* __restrict__ ids, uint32_t n, uint32_t n_groups, uint32_t part, uint32_t bits, const uint32_t* totals,
                      const uint32_t* ahead_in_cluster,
                      int32_t* __restrict__ offsets, int32_t* __restrict__ order, int32_t* __restrict__ position) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t partial[32], ahead[SHARED == Shared::kNot ? 1 : kRouteMaxGroups + 1], local[SHARED == Shared::kNot ? 1 : kRouteMaxGroups + 1];
  const uint32_t G1 = n_groups + 1, n_warp = blockDim.x >> 5;
  uint32_t* start = smem;                                       // [G1] the tile's first place of each group
  uint32_t* count = smem + G1;                                  // [G1] ids of the tile
  uint16_t* seen = reinterpret_cast<uint16_t*>(smem + 2 * G1);  // [n_warp][G1], 8-byte aligned
  uint2* sorted = reinterpret_cast<uint2*>(smem + 2 * G1);      // later: the tile's ids in order, each with its place
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint16_t* mine = seen + (size_t)warp * G1;
  const uint32_t begin = min(n, blockIdx.x * part), end = min(n, begin + part);

  // the parts are launched behind their count, which started behind everything that wrote the ids
  if (SHARED != Shared::kParts) wait_for_launch_ahead();
  bool first = true;
  for (uint32_t tile = begin; first || tile < end; tile += blockDim.x * kPlanSteps) {
    const uint32_t steps = min((uint32_t)kPlanSteps, (end - min(tile, end) + blockDim.x - 1) / blockDim.x);
    const uint32_t run = tile + warp * (32 * steps);  // the warp's ids
    uint32_t group[kPlanSteps], rank[kPlanSteps];
#pragma unroll
    for (int s = 0; s < kPlanSteps; s++) {
      const uint32_t i = run + s * 32 + lane;
      group[s] = (uint32_t)s < steps && i < end ? group_of(ids[i], n_groups) : kNoId;
    }
    for (uint32_t i = threadIdx.x; i < (n_warp * G1 + 3) / 4; i += blockDim.x) reinterpret_cast<uint2*>(seen)[i] = make_uint2(0, 0);
    __syncthreads();
    // ranks inside the warp's run
#pragma unroll
    for (int s = 0; s < kPlanSteps; s++) {
      if ((uint32_t)s >= steps) break;
      const bool live = group[s] != kNoId;
      const unsigned same = lanes_of_group(group[s], live, bits);
      const uint32_t before = live ? mine[group[s]] : 0;
      __syncwarp();
      if (live && lane == (uint32_t)__ffs(same) - 1) mine[group[s]] = (uint16_t)(before + __popc(same));
      __syncwarp();
      rank[s] = before + __popc(same & ((1u << lane) - 1));
    }
    __syncthreads();
    // the warps' counts become places inside the tile
    for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) {
      uint32_t at = 0;
#pragma unroll 8
      for (uint32_t w = 0; w < n_warp; w++) {
        const uint32_t c = seen[(size_t)w * G1 + g];
        seen[(size_t)w * G1 + g] = (uint16_t)at;
        at += c;
      }
      count[g] = at;
    }
    if (first) {
      // where the groups start in the batch, then where this part's share of them does
      if (SHARED == Shared::kNot) {
        for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) start[g] = count[g];
      } else if (SHARED == Shared::kCluster) {
        cluster_arrive();
        cluster_wait();
        for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) {
          uint32_t x[kPlanCluster], total = 0, before = 0;
#pragma unroll
          for (uint32_t c = 0; c < kPlanCluster; c++) x[c] = count_of(count + g, c);
#pragma unroll
          for (uint32_t c = 0; c < kPlanCluster; c++) {
            total += x[c];
            before += c < blockIdx.x ? x[c] : 0;
          }
          start[g] = total;
          ahead[g] = before;
        }
        cluster_arrive();  // waited for at the end: nobody leaves while its counts are being read
      } else {
        wait_for_launch_ahead();
        for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) {
          uint32_t total = 0, before = __ldcg(&ahead_in_cluster[(size_t)blockIdx.x * G1 + g]);
#pragma unroll 8
          for (uint32_t c = 0; c < (gridDim.x + kPlanCluster - 1) / kPlanCluster; c++) {
            const uint32_t x = __ldcg(&totals[(size_t)c * G1 + g]);
            total += x;
            before += c < blockIdx.x / kPlanCluster ? x : 0;
          }
          start[g] = total;
          ahead[g] = before;
        }
      }
      __syncthreads();
      block_exclusive_scan(start, G1, partial);
      for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) {
        if (blockIdx.x == 0) offsets[g] = (int32_t)start[g];
        if (SHARED != Shared::kNot) start[g] += ahead[g];
      }
      first = false;
    }
    __syncthreads();
    if (SHARED != Shared::kNot) {
      for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) local[g] = count[g];
      __syncthreads();
      block_exclusive_scan(local, G1, partial);
    }
    // in order through shared memory, so that a group's ids leave together
    uint32_t place[kPlanSteps];
#pragma unroll
    for (int s = 0; s < kPlanSteps; s++) {
      const uint32_t g = group[s];
      if ((uint32_t)s >= steps || g == kNoId) break;  // a run's ids are a prefix of its lanes' steps
      rank[s] += mine[g];
      place[s] = start[g] + rank[s];
      if (SHARED != Shared::kNot) rank[s] += local[g];
      else rank[s] = place[s];
      position[run + s * 32 + lane] = g < n_groups ? (int32_t)place[s] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kPlanSteps; s++) {
      if ((uint32_t)s >= steps || group[s] == kNoId) break;
      sorted[rank[s]] = make_uint2(run + s * 32 + lane, place[s]);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < min(end - min(tile, end), blockDim.x * steps); i += blockDim.x) {
      const uint2 id = sorted[i];
      order[id.y] = (int32_t)id.x;
    }
    __syncthreads();
    if (SHARED == Shared::kParts)
      for (uint32_t g = threadIdx.x; g < G1; g += blockDim.x) start[g] += count[g];
  }
  if (SHARED == Shared::kCluster) cluster_wait();
}

// How a batch is shared, the CTAs that share it and the ids of one.
struct PlanShape {
  Shared shared;
  uint32_t parts, part, block;
};
// On the GPU: 256 ids 2.5 us and 1024 4.1 in one CTA; 8192 took 12 there and take 6.3 in a cluster of eight, 65,536 ids
// 11; 524,288 12.8 in parts, a million 18.6.
PlanShape plan_shape(uint32_t n) {
  auto up_to = [](uint32_t v, uint32_t a) { return (v + a - 1) / a * a; };
  PlanShape s{Shared::kNot, 1, n, 128};
  if (n > kPlanCluster * kPlanTile) {
    s.shared = Shared::kParts;
    s.part = up_to((n + 147) / 148, kPlanBlock);
    s.parts = up_to((n + s.part - 1) / s.part, kPlanCluster);
  } else if (n > kPlanBlock) {
    s.shared = Shared::kCluster;
    s.parts = kPlanCluster;
    s.part = up_to((n + kPlanCluster - 1) / kPlanCluster, 32);
  }
  while (s.block < s.part && s.block < kPlanBlock) s.block *= 2;
  return s;
}

// ------------------------------------------------------------------------------------
// rows
// ------------------------------------------------------------------------------------

// Rows move in pieces of 16 bytes.
struct __align__(16) Piece {
  uint32_t v[4];
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

template <typename E>
struct Floats {
  static constexpr int N = 16 / (int)sizeof(E);
  float f[N];
  __device__ __forceinline__ void from(const Piece& p) {
    const E* e = reinterpret_cast<const E*>(&p);
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = widen<E>(e[i]);
  }
  // The sums were fp32; this is their one rounding.
  __device__ __forceinline__ Piece rounded() const {
    Piece p;
    E* e = reinterpret_cast<E*>(&p);
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = narrow<E>(f[i]);
    return p;
  }
  __device__ __forceinline__ void add(const Floats& x) {
#pragma unroll
    for (int i = 0; i < N; i++) f[i] += x.f[i];
  }
  __device__ __forceinline__ void add(const Floats& x, float w) {
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = fmaf(w, x.f[i], f[i]);
  }
  __device__ __forceinline__ Floats times(float w) const {
    Floats y;
#pragma unroll
    for (int i = 0; i < N; i++) y.f[i] = w * f[i];
    return y;
  }
  __device__ __forceinline__ float dot(const Floats& x, float sum) const {
#pragma unroll
    for (int i = 0; i < N; i++) sum = fmaf(f[i], x.f[i], sum);
    return sum;
  }
};

__device__ __forceinline__ const char* row_at(const void* base, long long stride, uint32_t row) {
  return static_cast<const char*>(base) + (long long)row * stride;
}
__device__ __forceinline__ char* row_at(void* base, long long stride, uint32_t row) {
  return static_cast<char*>(base) + (long long)row * stride;
}
__device__ __forceinline__ Piece ld_piece(const char* row, uint32_t piece) {
  return *reinterpret_cast<const Piece*>(row + (size_t)piece * 16);
}
__device__ __forceinline__ void st_piece(char* row, uint32_t piece, const Piece& p) {
  *reinterpret_cast<Piece*>(row + (size_t)piece * 16) = p;
}

// Place of a choice among the rows; kNowhere where it has none.
constexpr uint32_t kNowhere = 0xffffffffu;
__device__ __forceinline__ uint32_t place_of(const RouteRows& p, size_t choice) {
  const uint32_t row = (uint32_t)p.position[choice];
  return row < p.n_rows ? row : kNowhere;
}
// First row of row_out that no choice took, n_rows if they are not to be zeroed.
__device__ __forceinline__ uint32_t first_untaken(const RouteRows& p) {
  return p.n_routed ? min((uint32_t)max(*p.n_routed, 0), p.n_rows) : p.n_rows;
}

// n / d of a thread's number in the launch; 64-bit division is several times the instructions
__device__ __forceinline__ void divide(unsigned long long n, uint32_t d, uint32_t* q, uint32_t* r) {
  if (n >> 32 == 0) {
    *q = (uint32_t)n / d;
    *r = (uint32_t)n - *q * d;
  } else {
    *q = (uint32_t)(n / d);
    *r = (uint32_t)(n - (unsigned long long)*q * d);
  }
}

constexpr int kRowsBlock = 256;

__device__ __forceinline__ void zero_untaken(const RouteRows& p, uint32_t pieces) {
  const uint32_t first = first_untaken(p);
  const unsigned long long n = (unsigned long long)(p.n_rows - first) * pieces;
  for (unsigned long long u = (unsigned long long)blockIdx.x * kRowsBlock + threadIdx.x; u < n;
       u += (unsigned long long)gridDim.x * kRowsBlock) {
    uint32_t row, c;
    divide(u, pieces, &row, &c);
    st_piece(row_at(p.row_out, p.row_out_stride, first + row), c, Piece{});
  }
}

// A thread has one piece of one token's row and takes it to the rows of the token's choices.  Bound by the
// writes: 16,384 tokens of 4 KiB to 8 rows each 96 us, 6.3 TB/s.
template <typename E, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsBlock) spread_kernel(RouteRows p, uint32_t pieces) {
  wait_for_launch_ahead();
  release_launch_behind();
  uint32_t t, c;
  divide((unsigned long long)blockIdx.x * kRowsBlock + threadIdx.x, pieces, &t, &c);
  if (t < p.n_tokens) {
    const Piece in = ld_piece(row_at(p.token_in, p.token_in_stride, t), c);
    Floats<E> x;
    if (WEIGHTED) x.from(in);
    const size_t at = (size_t)t * p.k;
    for (uint32_t j = 0; j < p.k; j++) {
      const uint32_t row = place_of(p, at + j);
      if (row == kNowhere) continue;
      st_piece(row_at(p.row_out, p.row_out_stride, row), c, WEIGHTED ? x.times(p.weights[at + j]).rounded() : in);
    }
  }
  zero_untaken(p, pieces);
}

// A thread sums PIECES pieces of one token's row over its choices, in their order, in fp32: FLIGHT choices and
// all pieces are on their way at once.  Bound by the bytes in flight: 32,768 tokens of 4 rows of 8 KiB 220 us (6.1 TB/s) with
// 4 x 2, 249 with 4 x 1, 292 with 4 x 4 (registers); two rows of 32 KiB 120 us with 2 x 4, 167 with 4 x 1.
template <typename E, bool WEIGHTED, int FLIGHT, int PIECES>
__global__ void __launch_bounds__(kRowsBlock) gather_kernel(RouteRows p, uint32_t pieces) {
  wait_for_launch_ahead();
  release_launch_behind();
  const uint32_t stride = pieces / PIECES;  // between a thread's pieces
  uint32_t t, c;
  divide((unsigned long long)blockIdx.x * kRowsBlock + threadIdx.x, stride, &t, &c);
  if (t >= p.n_tokens) return;
  const size_t at = (size_t)t * p.k;
  Floats<E> sum[PIECES] = {};
  for (uint32_t j0 = 0; j0 < p.k; j0 += FLIGHT) {
    uint32_t row[FLIGHT];
    float w[FLIGHT];
    Piece in[FLIGHT][PIECES];
#pragma unroll
    for (int j = 0; j < FLIGHT; j++) {
      row[j] = j0 + j < p.k ? place_of(p, at + j0 + j) : kNowhere;
      w[j] = WEIGHTED && row[j] != kNowhere ? p.weights[at + j0 + j] : 1.f;
    }
#pragma unroll
    for (int j = 0; j < FLIGHT; j++)
      if (row[j] != kNowhere) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) in[j][i] = ld_piece(row_at(p.row_in, p.row_in_stride, row[j]), c + i * stride);
      }
#pragma unroll
    for (int j = 0; j < FLIGHT; j++)
      if (row[j] != kNowhere) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
          Floats<E> x;
          x.from(in[j][i]);
          if (WEIGHTED) sum[i].add(x, w[j]);
          else sum[i].add(x);
        }
      }
  }
#pragma unroll
  for (int i = 0; i < PIECES; i++) st_piece(row_at(p.token_out, p.token_out_stride, t), c + i * stride, sum[i].rounded());
}

// The lanes' sums of N choices' products into the dots: by the whole CTA.
template <int N>
__device__ __forceinline__ void share_sums(float (&dot)[N], float (*share)[N], const RouteRows& p, size_t at, uint32_t j0,
                                           bool live, uint32_t lane, uint32_t lanes) {
  if (lanes < N) {
#pragma unroll
    for (int j = 0; j < N; j++) {
      for (uint32_t d = lanes >> 1; d; d >>= 1) dot[j] += __shfl_xor_sync(kFull, dot[j], d);
      if (live && lane == 0 && j0 + j < p.k) p.dots[at + j0 + j] = dot[j];
    }
    return;
  }
  uint32_t which;
  const uint32_t width = min(lanes, 32u);
  const float sum = sum_over_lanes(dot, width, &which);
  const bool has = (lane & (width / N - 1)) == 0;  // one lane of those that end with the value
  if (lanes <= 32) {
    if (has && live && j0 + which < p.k) p.dots[at + j0 + which] = sum;
    return;
  }
  __syncthreads();
  if (has) share[threadIdx.x >> 5][which] = sum;
  __syncthreads();
  if (lane < N && live && j0 + lane < p.k) {
    float all = 0.f;
    for (uint32_t i = 0; i < lanes / 32; i++) all += share[(threadIdx.x >> 5) + i][lane];
    p.dots[at + j0 + lane] = all;
  }
}

// Inner products of a token's row with the rows of its choices, and the spread or the gather on the way: `lanes`
// threads (a power of two, fixed by the row's length, so that results do not depend on the batch) walk the row
// together.  All rows' pieces are loaded before anything is stored.  16,384 tokens of 6 rows of 4 KiB 145 us (216 with
// loads and stores in turn), of 8 gathered 117 us; bound by HBM, reads and writes mixed.
template <typename E, bool WEIGHTED, bool SPREAD, int CHOICES>
__global__ void __launch_bounds__(kRowsBlock, 2) dots_kernel(RouteRows p, uint32_t pieces, uint32_t lanes) {
  wait_for_launch_ahead();
  release_launch_behind();
  __shared__ float share[kRowsBlock / 32][CHOICES];
  const uint32_t lane = threadIdx.x & (lanes - 1);
  const uint32_t t = blockIdx.x * (kRowsBlock / lanes) + threadIdx.x / lanes;
  const bool live = t < p.n_tokens;
  const size_t at = (size_t)t * p.k;
  for (uint32_t j0 = 0; j0 < p.k; j0 += CHOICES) {
    uint32_t row[CHOICES];
    float w[CHOICES], dot[CHOICES];
#pragma unroll
    for (int j = 0; j < CHOICES; j++) {
      dot[j] = 0.f;
      row[j] = live && j0 + j < p.k ? place_of(p, at + j0 + j) : kNowhere;
      w[j] = WEIGHTED && row[j] != kNowhere ? p.weights[at + j0 + j] : 1.f;
    }
    for (uint32_t c = lane; live && c < pieces; c += lanes) {
      Piece in[CHOICES];
      const Piece mine = ld_piece(row_at(p.token_in, p.token_in_stride, t), c);
#pragma unroll
      for (int j = 0; j < CHOICES; j++)
        if (row[j] != kNowhere) in[j] = ld_piece(row_at(p.row_in, p.row_in_stride, row[j]), c);
      Floats<E> x, y, sum = {};
      x.from(mine);
#pragma unroll
      for (int j = 0; j < CHOICES; j++)
        if (row[j] != kNowhere) {
          y.from(in[j]);
          dot[j] = x.dot(y, dot[j]);
          if (SPREAD) {
            st_piece(row_at(p.row_out, p.row_out_stride, row[j]), c, WEIGHTED ? x.times(w[j]).rounded() : mine);
          } else if (WEIGHTED) {
            sum.add(y, w[j]);
          } else {
            sum.add(y);
          }
        }
      if (!SPREAD && j0 == 0) {  // choices past the first pass join the sum here, their products come later
        for (uint32_t j = CHOICES; j < p.k; j++) {
          const uint32_t r = place_of(p, at + j);
          if (r == kNowhere) continue;
          y.from(ld_piece(row_at(p.row_in, p.row_in_stride, r), c));
          if (WEIGHTED) sum.add(y, p.weights[at + j]);
          else sum.add(y);
        }
        st_piece(row_at(p.token_out, p.token_out_stride, t), c, sum.rounded());
      }
    }
    share_sums<CHOICES>(dot, share, p, at, j0, live, lane, lanes);
  }
  if (SPREAD) zero_untaken(p, pieces);
}

// ---- rows off the 16-byte boundaries ---------------------------------------------------------
// Rows of odd lengths start anywhere.  A row that is written is cut at its own 16-byte boundaries and stored in whole
// pieces; what goes there is read from the other row as the two pieces that hold it, shifted into place.
// 4097 x 3 rows of 1001 fp16 are summed in 10.8 us (element by element 19.8); instructions and the threads an SM holds bound
// it: with the loads of four choices ahead of their use, in more registers, it is 13.8.

// The 16 bytes at q (aligned), zeros outside [begin, end).
__device__ __forceinline__ Piece piece_within(const char* q, const char* begin, const char* end) {
  Piece p = {};
  if (q >= begin && q + 16 <= end) {
    p = *reinterpret_cast<const Piece*>(q);
  } else if (q + 16 > begin && q < end) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const char* h = q + 2 * i;
      const uint32_t x = h >= begin && h < end ? *reinterpret_cast<const uint16_t*>(h) : 0u;
      p.v[i / 2] |= x << (i & 1 ? 16 : 0);
    }
  }
  return p;
}
// The 16 bytes from byte `low` (below 16, even) of a and b on.
__device__ __forceinline__ Piece shifted(const Piece& a, const Piece& b, uint32_t low) {
  uint32_t w[8] = {a.v[0], a.v[1], a.v[2], a.v[3], b.v[0], b.v[1], b.v[2], b.v[3]};
  if (low & 8) {
#pragma unroll
    for (int i = 0; i < 6; i++) w[i] = w[i + 2];
  }
  if (low & 4) {
#pragma unroll
    for (int i = 0; i < 5; i++) w[i] = w[i + 1];
  }
  Piece p;
#pragma unroll
  for (int i = 0; i < 4; i++) p.v[i] = __funnelshift_r(w[i], w[i + 1], (uint32_t)low * 8);  // by low % 4 bytes
  return p;
}
// The 16 bytes from `at` (an even address) on, zeros outside the row.
// `amid`: the row has 16 bytes more on both sides.
__device__ __forceinline__ Piece piece_anywhere(const char* at, const char* begin, const char* end, bool amid) {
  const uint32_t low = (uint32_t)reinterpret_cast<uintptr_t>(at) & 15;
  const char* q = at - low;
  Piece a, b;
  if (amid) {
    a = *reinterpret_cast<const Piece*>(q);
    b = *reinterpret_cast<const Piece*>(q + 16);
  } else {
    a = piece_within(q, begin, end);
    b = piece_within(q + 16, begin, end);
  }
  return shifted(a, b, low);
}
template <typename E>
__device__ __forceinline__ void store_within(char* q, const Piece& p, char* begin, char* end) {
  if (q >= begin && q + 16 <= end) {
    *reinterpret_cast<Piece*>(q) = p;
    return;
  }
  const E* e = reinterpret_cast<const E*>(&p);
#pragma unroll
  for (int i = 0; i < Floats<E>::N; i++) {
    char* h = q + i * sizeof(E);
    if (h >= begin && h < end) *reinterpret_cast<E*>(h) = e[i];
  }
}

// Piece `c` of a row that is written: its address, and how far it lies from the row's begin.
struct Cut {
  char *begin, *end, *at;
  long long off;
  __device__ __forceinline__ Cut(char* row, uint32_t bytes, uint32_t c) : begin(row), end(row + bytes) {
    at = row - (reinterpret_cast<uintptr_t>(row) & 15) + (size_t)c * 16;
    off = at - row;
  }
  __device__ __forceinline__ bool inside() const { return at < end; }
};
__device__ __forceinline__ Piece piece_of(const Cut& cut, const char* row, uint32_t bytes) {
  return piece_anywhere(row + cut.off, row, row + bytes, cut.off >= 16 && cut.at + 32 <= cut.end);
}
template <typename E>
__device__ __forceinline__ Floats<E> read_at(const Cut& cut, const char* row, uint32_t bytes) {
  Floats<E> x;
  x.from(piece_of(cut, row, bytes));
  return x;
}

// lanes threads a token, as in dots_kernel; `cuts` of a row, at most.
template <typename E, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsBlock) gather_any_kernel(RouteRows p, uint32_t cuts, uint32_t lanes) {
  wait_for_launch_ahead();
  release_launch_behind();
  constexpr int kChoices = 4;
  const uint32_t lane = threadIdx.x & (lanes - 1), bytes = p.dim * (uint32_t)sizeof(E);
  const uint32_t t = blockIdx.x * (kRowsBlock / lanes) + threadIdx.x / lanes;
  if (t >= p.n_tokens) return;
  const size_t at = (size_t)t * p.k;
  for (uint32_t u = lane; u < cuts; u += lanes) {
    const uint32_t c = u + 1 < cuts ? u + 1 : 0;  // the row's begin beside its end: one warp has both
    const Cut cut(row_at(p.token_out, p.token_out_stride, t), bytes, c);
    if (!cut.inside()) continue;
    Floats<E> sum = {};
#pragma unroll
    for (int j = 0; j < kChoices; j++) {
      const uint32_t row = (uint32_t)j < p.k ? place_of(p, at + j) : kNowhere;
      if (row == kNowhere) continue;
      const Floats<E> y = read_at<E>(cut, row_at(p.row_in, p.row_in_stride, row), bytes);
      if (WEIGHTED) sum.add(y, p.weights[at + j]);
      else sum.add(y);
    }
    for (uint32_t j = kChoices; j < p.k; j++) {
      const uint32_t row = place_of(p, at + j);
      if (row == kNowhere) continue;
      const Floats<E> y = read_at<E>(cut, row_at(p.row_in, p.row_in_stride, row), bytes);
      if (WEIGHTED) sum.add(y, p.weights[at + j]);
      else sum.add(y);
    }
    store_within<E>(cut.at, sum.rounded(), cut.begin, cut.end);
  }
}

__device__ __forceinline__ void zero_untaken_any(const RouteRows& p, uint32_t bytes, uint32_t cuts) {
  const uint32_t first = first_untaken(p);
  const unsigned long long n = (unsigned long long)(p.n_rows - first) * cuts;
  for (unsigned long long u = (unsigned long long)blockIdx.x * kRowsBlock + threadIdx.x; u < n;
       u += (unsigned long long)gridDim.x * kRowsBlock) {
    uint32_t row, c;
    divide(u, cuts, &row, &c);
    const Cut cut(row_at(p.row_out, p.row_out_stride, first + row), bytes, c);
    if (cut.inside()) store_within<uint16_t>(cut.at, Piece{}, cut.begin, cut.end);
  }
}

// lanes threads a choice: the rows written are cut differently.
template <typename E, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsBlock) spread_any_kernel(RouteRows p, uint32_t cuts, uint32_t lanes) {
  wait_for_launch_ahead();
  release_launch_behind();
  const uint32_t lane = threadIdx.x & (lanes - 1), bytes = p.dim * (uint32_t)sizeof(E);
  const uint32_t choice = blockIdx.x * (kRowsBlock / lanes) + threadIdx.x / lanes, t = choice / p.k;
  const uint32_t row = choice < p.n_rows ? place_of(p, choice) : kNowhere;
  const float w = WEIGHTED && row != kNowhere ? p.weights[choice] : 1.f;
  for (uint32_t u = lane; row != kNowhere && u < cuts; u += lanes) {
    const uint32_t c = u + 1 < cuts ? u + 1 : 0;
    const Cut cut(row_at(p.row_out, p.row_out_stride, row), bytes, c);
    if (!cut.inside()) continue;
    const Piece in = piece_of(cut, row_at(p.token_in, p.token_in_stride, t), bytes);
    Floats<E> x;
    x.from(in);
    store_within<E>(cut.at, WEIGHTED ? x.times(w).rounded() : in, cut.begin, cut.end);
  }
  zero_untaken_any(p, bytes, cuts);
}

// Bytes 16 u to 16 u + 15 of a row that starts anywhere, zeros behind it.
__device__ __forceinline__ Piece piece_of_row(const char* row, uint32_t bytes, uint32_t u) {
  return piece_anywhere(row + (size_t)u * 16, row, row + bytes, u > 0 && (u + 2) * 16 <= bytes);
}

// Inner products of rows that start anywhere.  Pieces are counted from the rows' begins, wherever those lie: results do not
// depend on the addresses, which change with a choice's place.  lanes threads a token (gather) or a choice (spread).
// 16,384 x 8 rows of 1001 bf16: spread 256 us, the token's row read once more for the cuts (about 330 with pieces exchanged
// between lanes as in the gather); gathered 198 us (290 with 116 registers a thread).
struct Share {  // a lane's pieces: its warp has neighbouring ones, `width` of them at a time
  uint32_t width, seat, begin, end;
  __device__ __forceinline__ Share(uint32_t lane, uint32_t lanes, uint32_t pieces) {
    width = min(lanes, 32u);
    seat = lane & (width - 1);
    const uint32_t per = (pieces + lanes - 1) / lanes * width;
    begin = min(lane / width * per, pieces);
    end = min(begin + per, pieces);
  }
};

template <typename E, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsBlock, sizeof(E) == 4 ? 5 : 4) gather_any_dots_kernel(RouteRows p, uint32_t cuts, uint32_t lanes) {
  wait_for_launch_ahead();
  release_launch_behind();
  constexpr int kChoices = 4;
  __shared__ float share[kRowsBlock / 32][kChoices];
  const uint32_t lane = threadIdx.x & (lanes - 1), bytes = p.dim * (uint32_t)sizeof(E), pieces = cuts - 1;
  const uint32_t t = blockIdx.x * (kRowsBlock / lanes) + threadIdx.x / lanes;
  const bool live = t < p.n_tokens;
  const size_t at = (size_t)t * p.k;
  const Share mine(lane, lanes, pieces);
  for (uint32_t j0 = 0; j0 < p.k; j0 += kChoices) {
    float dot[kChoices] = {};
    Piece ahead = {};
    for (uint32_t u0 = mine.begin; u0 < mine.end; u0 += mine.width) {
      const uint32_t u = u0 + mine.seat;
      const bool on = live && u < mine.end;
      Floats<E> x, sum = {};
      if (on) x.from(piece_of_row(row_at(p.token_in, p.token_in_stride, t), bytes, u));
#pragma unroll
      for (int j = 0; j < kChoices; j++) {
        const uint32_t row = on && j0 + j < p.k ? place_of(p, at + j0 + j) : kNowhere;
        if (row == kNowhere) continue;
        Floats<E> y;
        y.from(piece_of_row(row_at(p.row_in, p.row_in_stride, row), bytes, u));
        if (WEIGHTED) sum.add(y, p.weights[at + j0 + j]);
        else sum.add(y);
        dot[j] = x.dot(y, dot[j]);
      }
      if (j0) continue;
      for (uint32_t j = kChoices; on && j < p.k; j++) {  // choices past the first pass join the sum here, their products come later
        const uint32_t row = place_of(p, at + j);
        if (row == kNowhere) continue;
        Floats<E> y;
        y.from(piece_of_row(row_at(p.row_in, p.row_in_stride, row), bytes, u));
        if (WEIGHTED) sum.add(y, p.weights[at + j]);
        else sum.add(y);
      }
      // What lies between two 16-byte boundaries is the left neighbour's end and the own begin; the first and the last
      // piece of the warp's run are stored in part.
      __syncwarp();
      const Piece out = sum.rounded();
      const uint32_t neighbour = (threadIdx.x & 31 & ~(mine.width - 1)) | ((mine.seat - 1) & (mine.width - 1));
      Piece left;
#pragma unroll
      for (int i = 0; i < 4; i++) left.v[i] = __shfl_sync(kFull, mine.seat + 1 == mine.width ? ahead.v[i] : out.v[i], neighbour);
      ahead = out;
      if (!on) continue;
      char *row = row_at(p.token_out, p.token_out_stride, t), *q = row + (size_t)u * 16, *end = row + bytes;
      const uint32_t low = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15;
      if (low == 0) {
        store_within<E>(q, out, row, end);
        continue;
      }
      store_within<E>(q - low, shifted(left, out, 16 - low), u == mine.begin ? q : row, end);
      if (u + 1 == mine.end) store_within<E>(q - low + 16, shifted(out, out, 16 - low), row, q + 16 < end ? q + 16 : end);
    }
    share_sums<kChoices>(dot, share, p, at, j0, live, lane, lanes);
  }
}

template <typename E, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsBlock, 6) spread_any_dots_kernel(RouteRows p, uint32_t cuts, uint32_t lanes) {
  wait_for_launch_ahead();
  release_launch_behind();
  __shared__ float share[kRowsBlock / 32][1];
  const uint32_t lane = threadIdx.x & (lanes - 1), bytes = p.dim * (uint32_t)sizeof(E);
  const uint32_t choice = blockIdx.x * (kRowsBlock / lanes) + threadIdx.x / lanes, t = choice / p.k;
  const uint32_t row = choice < p.n_rows ? place_of(p, choice) : kNowhere;
  const float w = WEIGHTED && row != kNowhere ? p.weights[choice] : 1.f;
  const char *from = row_at(p.token_in, p.token_in_stride, t), *other = row_at(p.row_in, p.row_in_stride, row);
  float dot[1] = {};
  const Share mine(lane, lanes, cuts - 1);
  const uint32_t end = mine.begin < mine.end && mine.end + 1 == cuts ? cuts : mine.end;  // one cut more than pieces
  for (uint32_t u = mine.begin + mine.seat; row != kNowhere && u < end; u += mine.width) {
    Floats<E> x, y;
    if (u + 1 < cuts) {
      x.from(piece_of_row(from, bytes, u));
      y.from(piece_of_row(other, bytes, u));
      dot[0] = x.dot(y, dot[0]);
    }
    const Cut cut(row_at(p.row_out, p.row_out_stride, row), bytes, u + 1 < cuts ? u + 1 : 0);
    if (!cut.inside()) continue;
    const Piece in = piece_of(cut, from, bytes);  // again, from the L1
    x.from(in);
    store_within<E>(cut.at, WEIGHTED ? x.times(w).rounded() : in, cut.begin, cut.end);
  }
  share_sums<1>(dot, share, p, choice, 0, choice < p.n_rows, lane, lanes);
  zero_untaken_any(p, bytes, cuts);
}

// Whether every row in use starts on a 16-byte boundary and is whole pieces long.
bool rows_aligned(const RouteRows& p, int elem_bytes) {
  unsigned long long bits = (unsigned long long)p.dim * elem_bytes;
  auto add = [&](const void* q, long long stride) {
    if (q) bits |= reinterpret_cast<uintptr_t>(q) | (unsigned long long)stride;
  };
  add(p.token_in, p.token_in_stride);
  add(p.token_out, p.token_out_stride);
  add(p.row_in, p.row_in_stride);
  add(p.row_out, p.row_out_stride);
  return bits % 16 == 0;
}

// Threads that walk a row together: `each` pieces a thread, but 8 threads (a line) where the row has that many.
// With products, 8 pieces: 16,384 x 8 rows of 4 KiB gathered in 117 us, with 4 in 129, with 2 in 146; what a token
// costs besides its loads then counts little.
uint32_t row_lanes(uint32_t pieces, uint32_t each) {
  uint32_t lanes = 1;
  while (lanes < 8 ? lanes < pieces : lanes * each < pieces && lanes < (uint32_t)kRowsBlock) lanes *= 2;
  return lanes;
}

template <typename E, bool WEIGHTED>
cudaError_t rows_launch(const RouteRows& p, bool spread, cudaStream_t stream) {
  const unsigned long long bytes = (unsigned long long)p.dim * sizeof(E);
  auto per_row = [&](auto kern, uint32_t rows, uint32_t pieces, uint32_t each) {
    const uint32_t lanes = row_lanes(pieces, each), per = kRowsBlock / lanes;
    return launch(kern, (rows + per - 1) / per, kRowsBlock, 0, stream, true, 1, p, pieces, lanes);
  };
  auto per_token = [&](auto kern, uint32_t pieces, uint32_t each) { return per_row(kern, p.n_tokens, pieces, each); };
  if (!rows_aligned(p, sizeof(E))) {
    const uint32_t cuts = (uint32_t)((bytes + 15) / 16 + 1);
    if (p.dots && spread) return per_row(spread_any_dots_kernel<E, WEIGHTED>, p.n_rows, cuts, 4);
    if (p.dots) return per_token(gather_any_dots_kernel<E, WEIGHTED>, cuts, 4);
    if (spread) return per_row(spread_any_kernel<E, WEIGHTED>, p.n_rows, cuts, 4);
    return per_token(gather_any_kernel<E, WEIGHTED>, cuts, 1);
  }
  const uint32_t pieces = (uint32_t)(bytes / 16);
  if (p.dots) {
    if (spread)
      return per_token(p.k <= 2 ? dots_kernel<E, WEIGHTED, true, 2> : p.k <= 4 ? dots_kernel<E, WEIGHTED, true, 4> : dots_kernel<E, WEIGHTED, true, 8>, pieces, 8);
    return per_token(p.k <= 2 ? dots_kernel<E, WEIGHTED, false, 2> : p.k <= 4 ? dots_kernel<E, WEIGHTED, false, 4> : dots_kernel<E, WEIGHTED, false, 8>, pieces, 8);
  }
  const unsigned long long units = (unsigned long long)p.n_tokens * pieces;
  auto per_piece = [&](auto kern, uint32_t each) {
    const unsigned long long grid = (units / each + kRowsBlock - 1) / kRowsBlock;
    return grid > 0x7fffffffull ? cudaErrorInvalidValue : launch(kern, (unsigned)grid, kRowsBlock, 0, stream, true, 1, p, pieces);
  };
  if (spread) return per_piece(spread_kernel<E, WEIGHTED>, 1);
  // eight loads in flight a thread, once there are threads enough to fill the GPU
  const bool many = units >= 148ull * 2048 * 4;
  if (p.k <= 2 && many && pieces % 4 == 0) return per_piece(gather_kernel<E, WEIGHTED, 2, 4>, 4);
  if (many && pieces % 2 == 0) return per_piece(gather_kernel<E, WEIGHTED, 4, 2>, 2);
  return per_piece(gather_kernel<E, WEIGHTED, 4, 1>, 1);
}

cudaError_t rows_by_type(const RouteRows& p, int elem, bool spread, cudaStream_t stream) {
  if (p.n_tokens == 0) return cudaSuccess;
  auto by_weight = [&](auto e) {
    using E = decltype(e);
    return p.weights ? rows_launch<E, true>(p, spread, stream) : rows_launch<E, false>(p, spread, stream);
  };
  if (elem == kElemF32) return by_weight(float{});
  if (elem == kElemF16) return by_weight(__half{});
  return by_weight(__nv_bfloat16{});
}

}  // namespace

size_t route_plan_scratch_bytes(uint32_t n, int n_groups) {
  const PlanShape s = plan_shape(n);
  return s.shared == Shared::kParts ? (size_t)(s.parts + s.parts / kPlanCluster) * (n_groups + 1) * sizeof(uint32_t) : 0;
}

cudaError_t launch_route_plan(const void* ids, int id_bytes, uint32_t n, int n_groups, int32_t* offsets,
                              int32_t* order, int32_t* position, void* scratch, cudaStream_t stream) {
  const PlanShape s = plan_shape(n);
  const uint32_t G = (uint32_t)n_groups;
  uint32_t bits = 0;
  while (G >> bits) bits++;  // groups 0 .. G: G is that of the ids without one
  const size_t tile = std::min(s.part, s.block * kPlanSteps);
  const size_t smem = (size_t)(G + 1) * 2 * sizeof(uint32_t) + std::max((G + 1) * (s.block / 32) * sizeof(uint16_t) + 8, tile * sizeof(uint2));
  auto go = [&](auto id) {
    using IdT = decltype(id);
    const IdT* in = static_cast<const IdT*>(ids);
    uint32_t *ahead = static_cast<uint32_t*>(scratch), *totals = ahead + (size_t)s.parts * (G + 1);
    auto place = [&](auto kern, uint32_t cluster) {
      return launch(kern, s.parts, s.block, smem, stream, true, cluster, in, n, G, s.part, bits,
                    static_cast<const uint32_t*>(totals), static_cast<const uint32_t*>(ahead), offsets, order, position);
    };
    if (s.shared == Shared::kNot) return place(plan_place_kernel<IdT, Shared::kNot>, 1);
    if (s.shared == Shared::kCluster) return place(plan_place_kernel<IdT, Shared::kCluster>, kPlanCluster);
    cudaError_t e = launch(plan_count_kernel<IdT>, s.parts, kPlanBlock, (G + 1) * sizeof(uint32_t), stream, true, kPlanCluster, in, n, G,
                           s.part, totals, ahead);
    return e == cudaSuccess ? place(plan_place_kernel<IdT, Shared::kParts>, 1) : e;
  };
  return id_bytes == 8 ? go((long long)0) : go((int32_t)0);
}

cudaError_t launch_route_spread(const RouteRows& p, int elem, cudaStream_t stream) { return rows_by_type(p, elem, true, stream); }
cudaError_t launch_route_gather(const RouteRows& p, int elem, cudaStream_t stream) { return rows_by_type(p, elem, false, stream); }

}  // namespace ugc
