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
// all pieces are on their way at once.
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
// together.  All rows' pieces are loaded before anything is stored.
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
// (Elements one by one: 4097 x 3 rows of 1001 fp16 summed in 19.8 us.)

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
// The 16 bytes from `at` (an even address) on, zeros outside the row.
__device__ __forceinline__ Piece piece_anywhere(const char* at, const char* begin, const char* end) {
  const uintptr_t low = reinterpret_cast<uintptr_t>(at) & 15;
  const char* q = at - low;
  const Piece a = piece_within(q, begin, end);
  if (low == 0) return a;
  const Piece b = piece_within(q + 16, begin, end);
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
  for (int i = 0; i < 4; i++) p.v[i] = low & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
  return p;
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
template <typename E>
__device__ __forceinline__ Floats<E> read_at(const Cut& cut, const char* row, uint32_t bytes) {
  Floats<E> x;
  x.from(piece_anywhere(row + cut.off, row, row + bytes));
  return x;
}

// lanes threads a token, as in dots_kernel; `pieces`: cuts of a row, at most.
template <typename E, bool WEIGHTED, bool DOTS>
__global__ void __launch_bounds__(kRowsBlock) gather_any_kernel(RouteRows p, uint32_t pieces, uint32_t lanes) {
  wait_for_launch_ahead();
  release_launch_behind();
  constexpr int kChoices = 4;
  __shared__ float share[kRowsBlock / 32][kChoices];
  const uint32_t lane = threadIdx.x & (lanes - 1), bytes = p.dim * (uint32_t)sizeof(E);
  const uint32_t t = blockIdx.x * (kRowsBlock / lanes) + threadIdx.x / lanes;
  const bool live = t < p.n_tokens;
  const size_t at = (size_t)t * p.k;
  for (uint32_t j0 = 0; j0 < (DOTS ? p.k : 1); j0 += kChoices) {
    float dot[kChoices] = {};
    for (uint32_t c = lane; live && c < pieces; c += lanes) {
      const Cut cut(row_at(p.token_out, p.token_out_stride, t), bytes, c);
      if (!cut.inside()) continue;
      Floats<E> x, sum = {};
      if (DOTS) x = read_at<E>(cut, row_at(p.token_in, p.token_in_stride, t), bytes);
#pragma unroll
      for (int j = 0; j < kChoices; j++) {
        const uint32_t row = j0 + j < p.k ? place_of(p, at + j0 + j) : kNowhere;
        if (row == kNowhere) continue;
        const Floats<E> y = read_at<E>(cut, row_at(p.row_in, p.row_in_stride, row), bytes);
        if (WEIGHTED) sum.add(y, p.weights[at + j0 + j]);
        else sum.add(y);
        if (DOTS) dot[j] = x.dot(y, dot[j]);
      }
      if (j0) continue;
      for (uint32_t j = kChoices; j < p.k; j++) {  // choices past the first pass join the sum here, their products come later
        const uint32_t row = place_of(p, at + j);
        if (row == kNowhere) continue;
        const Floats<E> y = read_at<E>(cut, row_at(p.row_in, p.row_in_stride, row), bytes);
        if (WEIGHTED) sum.add(y, p.weights[at + j]);
        else sum.add(y);
      }
      store_within<E>(cut.at, sum.rounded(), cut.begin, cut.end);
    }
    if (DOTS) share_sums<kChoices>(dot, share, p, at, j0, live, lane, lanes);
  }
}

template <typename E, bool WEIGHTED, bool DOTS>
__global__ void __launch_bounds__(kRowsBlock) spread_any_kernel(RouteRows p, uint32_t pieces, uint32_t lanes) {
  wait_for_launch_ahead();
  release_launch_behind();
  constexpr int kChoices = 4;
  __shared__ float share[kRowsBlock / 32][kChoices];
  const uint32_t lane = threadIdx.x & (lanes - 1), bytes = p.dim * (uint32_t)sizeof(E);
  const uint32_t t = blockIdx.x * (kRowsBlock / lanes) + threadIdx.x / lanes;
  const bool live = t < p.n_tokens;
  const size_t at = (size_t)t * p.k;
  for (uint32_t j0 = 0; j0 < p.k; j0 += kChoices) {
    float dot[kChoices] = {};
    for (uint32_t c = lane; live && c < pieces; c += lanes) {
#pragma unroll
      for (int j = 0; j < kChoices; j++) {
        const uint32_t row = j0 + j < p.k ? place_of(p, at + j0 + j) : kNowhere;
        if (row == kNowhere) continue;
        const Cut cut(row_at(p.row_out, p.row_out_stride, row), bytes, c);
        if (!cut.inside()) continue;
        const Floats<E> x = read_at<E>(cut, row_at(p.token_in, p.token_in_stride, t), bytes);
        if (DOTS) dot[j] = x.dot(read_at<E>(cut, row_at(p.row_in, p.row_in_stride, row), bytes), dot[j]);
        store_within<E>(cut.at, WEIGHTED ? x.times(p.weights[at + j0 + j]).rounded() : x.rounded(), cut.begin, cut.end);
      }
    }
    if (DOTS) share_sums<kChoices>(dot, share, p, at, j0, live, lane, lanes);
  }
  const uint32_t first = first_untaken(p);
  const unsigned long long n = (unsigned long long)(p.n_rows - first) * pieces;
  for (unsigned long long u = (unsigned long long)blockIdx.x * kRowsBlock + threadIdx.x; u < n;
       u += (unsigned long long)gridDim.x * kRowsBlock) {
    uint32_t row, c;
    divide(u, pieces, &row, &c);
    const Cut cut(row_at(p.row_out, p.row_out_stride, first + row), bytes, c);
    if (cut.inside()) store_within<E>(cut.at, Piece{}, cut.begin, cut.end);
  }
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
  auto per_token = [&](auto kern, uint32_t pieces, uint32_t each) {
    const uint32_t lanes = row_lanes(pieces, each), per = kRowsBlock / lanes;
    return launch(kern, (p.n_tokens + per - 1) / per, kRowsBlock, 0, stream, true, p, pieces, lanes);
  };
  if (!rows_aligned(p, sizeof(E))) {
    const uint32_t cuts = (uint32_t)((bytes + 15) / 16 + 1);
    if (spread) return per_token(p.dots ? spread_any_kernel<E, WEIGHTED, true> : spread_any_kernel<E, WEIGHTED, false>, cuts, p.dots ? 2 : 1);
    return per_token(p.dots ? gather_any_kernel<E, WEIGHTED, true> : gather_any_kernel<E, WEIGHTED, false>, cuts, p.dots ? 2 : 1);
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
    return grid > 0x7fffffffull ? cudaErrorInvalidValue : launch(kern, (unsigned)grid, kRowsBlock, 0, stream, true, p, pieces);
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
