// Low-rank adapters of many requests at once: out[t] = base[t] + scale[a] * (x[t] down[a]^T) up[a]^T.
#include "routing.cuh"

#include "lanes.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace cg = cooperative_groups;

namespace ugc {

namespace {

constexpr int kWarps = 8;
constexpr int kBlock = kWarps * 32;
constexpr int kTile = 16;     // tokens of a tile: the rows of one matrix instruction

template <typename E>
struct Half;
template <>
struct Half<__half> {
  static __device__ __forceinline__ float2 widen(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static __device__ __forceinline__ uint32_t narrow(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // Terms: a token's largest rank product is scaled to [2^14, 2^15), so that what a term leaves of smaller ones is
  // above the type's last step (2^-24) too: 24 bits of values down to 2^-16 of the largest, 2^-39 of the largest below.
  static constexpr bool kScaled = true;
  static __device__ __forceinline__ uint32_t first_bits(float a, float b) { return narrow(a, b); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ float2 widen(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
  static __device__ __forceinline__ uint32_t narrow(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // Terms: the range is that of fp32, so nothing is scaled; cut off, not rounded, so that none becomes infinite.
  static constexpr bool kScaled = false;
  static __device__ __forceinline__ uint32_t first_bits(float a, float b) {
    uint32_t h;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(b), "f"(a));
    return h;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// W words of 16-bit elements from p, zeros from element `valid` on.
template <int W, bool VECTOR>
__device__ __forceinline__ void load_words(uint32_t (&w)[W], const uint16_t* p, int valid) {
  if (VECTOR && valid >= 2 * W) {
    if (W == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2 % W] = v.z, w[3 % W] = v.w;
    } else if (W == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1 % W] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < W; i++) {
    const uint32_t lo = 2 * i < valid ? p[2 * i] : 0, hi = 2 * i + 1 < valid ? p[2 * i + 1] : 0;
    w[i] = lo | hi << 16;
  }
}

// The rank products enter the second product as three 16-bit terms: each takes what the ones before it left, so that
// together they hold the 24 bits of the fp32 sum (8 + 8 + 8, or 11 + 11 and the rest).
constexpr int kTerms = 3;
template <typename E>
__device__ __forceinline__ void split(float a, float b, uint32_t (&term)[kTerms]) {
#pragma unroll
  for (int t = 0; t < kTerms; t++) {
    term[t] = Half<E>::first_bits(a, b);
    const float2 h = Half<E>::widen(term[t]);
    a = t == 0 && isinf(h.x) ? 0.f : a - h.x;  // exact; nothing is left of an infinite value
    b = t == 0 && isinf(h.y) ? 0.f : b - h.y;
  }
}

// The part of a rank product that counts for its token's scale.
__device__ __forceinline__ float size_of(float v) { return isinf(v) ? 0.f : fabsf(v); }
// A power of two s, 1 / s one too, with max * s in [2^14, 2^15), or below where max is tiny.
__device__ __forceinline__ float scale_for(float max) {
  const int e = (int)(__float_as_uint(max) >> 23 & 255) - 127;
  return __uint_as_float((uint32_t)(127 + min(14 - e, 126)) << 23);
}

// Tile `index` of the batch: tiles of ROWS tokens, group by group, those without a group last.  By the whole CTA.
struct Tile {
  uint32_t group, first, count;  // first: place in `order`
};
template <int ROWS, int THREADS>
__device__ Tile find_tile(const int32_t* offsets, uint32_t n_groups, uint32_t n_tokens, uint32_t index) {
  __shared__ uint32_t partial[THREADS / 32];
  __shared__ Tile found;
  const uint32_t n = n_groups + 1, per = (n + THREADS - 1) / THREADS, g0 = threadIdx.x * per;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto begin_of = [&](uint32_t g) { return min((uint32_t)max(offsets[g], 0), n_tokens); };
  auto tiles_of = [&](uint32_t g) {
    const uint32_t a = begin_of(g), b = g < n_groups ? begin_of(g + 1) : n_tokens;
    return b > a ? (b - a + ROWS - 1) / ROWS : 0;
  };
  uint32_t sum = 0;
  for (uint32_t i = 0; i < per; i++)
    if (g0 + i < n) sum += tiles_of(g0 + i);
  uint32_t inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(kFull, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) partial[warp] = inc;
  if (threadIdx.x == 0) found = Tile{0, 0, 0};
  __syncthreads();
  uint32_t at = inc - sum;
  for (uint32_t w = 0; w < warp; w++) at += partial[w];
  if (index >= at && index < at + sum) {
    for (uint32_t i = 0; i < per && g0 + i < n; i++) {
      const uint32_t m = tiles_of(g0 + i);
      if (index < at + m) {
        const uint32_t a = begin_of(g0 + i), b = g0 + i < n_groups ? begin_of(g0 + i + 1) : n_tokens;
        const uint32_t first = a + (index - at) * ROWS;
        found = Tile{g0 + i, first, min(b - first, (uint32_t)ROWS)};
        break;
      }
      at += m;
    }
  }
  __syncthreads();
  return found;
}

__device__ unsigned int g_stalled;  // waits that ran out

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// False after about two seconds: nothing here takes that long, so something is broken and the kernel ends.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
  long long began = 0;
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    const long long now = clock64();
    if (!began) began = now;
    if (now - began > 4000000000ll) {
      atomicAdd(&g_stalled, 1u);
      return false;
    }
  }
}
// By a whole warp, which stays together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(kFull, barrier_wait(bar, parity)); }

// ------------------------------------------------------------------------------------
// single tokens: a cluster of CTAs has a tile of 16 tokens
// ------------------------------------------------------------------------------------
// Bound by the adapters' matrices and, with few tokens, by the chain plan - tile - x, down - up.  Every CTA of
// the cluster has a slice of dim and, later, of out_dim; the CTAs hand one another their partial rank products
// through distributed shared memory.  `up` does not wait for those: a bulk copy brings the slice
// (what fits) into shared memory meanwhile.  The matrix instructions take the columns of a product in any
// order as long as both operands agree, so every lane loads 16 consecutive bytes of a row.  4096 x 4096, bf16: one token
// of rank 16 6.5 us (about 2.1 until its tile is known, 1.0 for the first product, 1.6 for the cluster's sums, 1.4 for
// the second), 48 tokens of 64 adapters 8.5 us (8.1 MB of matrices), of rank 64 17 us, of rank 128 33 us (66 MB, 2.0 TB/s).

constexpr int kMostCluster = 8;

// Columns [begin, end) of the rows of a tile's tokens from one matrix to another; by THREADS threads, four pieces each in
// flight.  token(m): the m-th token of the tile, negative for none.
template <int THREADS, bool VECTOR, typename Token>
__device__ __forceinline__ void copy_rows(const AdapterParams& p, Token token, uint32_t count, uint32_t begin, uint32_t end,
                                          uint32_t thread) {
  constexpr uint32_t kPiece = VECTOR ? 8 : 1;
  const uint16_t* from = static_cast<const uint16_t*>(p.base);
  uint16_t* to = static_cast<uint16_t*>(p.out);
  const uint32_t pieces = (end - begin + kPiece - 1) / kPiece, all = count * pieces;
  for (uint32_t i0 = thread; i0 < all; i0 += 4 * THREADS) {
    uint4 v[4];
    int t[4];
#pragma unroll
    for (int f = 0; f < 4; f++) t[f] = i0 + f * THREADS < all ? token((i0 + f * THREADS) / pieces) : -1;
#pragma unroll
    for (int f = 0; f < 4; f++) {
      if (t[f] < 0) continue;
      const uint16_t* at = from + (long long)t[f] * p.base_stride + begin + (i0 + f * THREADS) % pieces * kPiece;
      if (VECTOR) v[f] = *reinterpret_cast<const uint4*>(at);
      else v[f].x = *at;
    }
#pragma unroll
    for (int f = 0; f < 4; f++) {
      if (t[f] < 0) continue;
      uint16_t* at = to + (long long)t[f] * p.out_stride + begin + (i0 + f * THREADS) % pieces * kPiece;
      if (VECTOR) *reinterpret_cast<uint4*>(at) = v[f];
      else *at = (uint16_t)v[f].x;
    }
  }
}

// RP: rank rounded up to 8, 16, 32, 64 or 128.
template <int RP>
struct SmallShape {
  static constexpr int kWarpRanks = RP < 32 ? RP : 32;          // ranks a warp has in the first product
  static constexpr int kRankGroups = RP / kWarpRanks;
  static constexpr int kDepthGroups = kWarps / kRankGroups;     // warps that share a slice of dim
  // the second product's depth; at 8 ranks the first two terms lie side by side in it
  static constexpr int kDepth = RP < 16 ? 16 : RP;
  static constexpr int kSlabs = RP < 16 ? 2 : kTerms;
  static constexpr int kPart = kDepthGroups * kTile * RP * 4;
  static constexpr int kInner = kSlabs * kTile * (kDepth + 8) * 2;
  static constexpr int kShared = kPart + kInner;                // and what is held of `up`
};

template <typename E, int RP, bool VECTOR>
__global__ void __launch_bounds__(kBlock, RP <= 16 ? 4 : RP <= 32 ? 3 : 2) adapter_kernel(AdapterParams p, uint32_t up_room) {
  using S = SmallShape<RP>;
  constexpr int KR = S::kDepth;
  extern __shared__ __align__(128) unsigned char smem[];
  using Inner = uint16_t[kTile][KR + 8];
  float* part = reinterpret_cast<float*>(smem);                              // [depth group][token][rank]
  Inner* inner = reinterpret_cast<Inner*>(smem + S::kPart);                  // [slab]
  uint16_t* up_here = reinterpret_cast<uint16_t*>(smem + S::kPart + S::kInner);
  __shared__ float back[kTile];
  __shared__ int32_t token[kTile];
  __shared__ __align__(8) uint64_t up_landed;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t member = cluster.block_rank(), members = cluster.num_blocks();
  if (threadIdx.x == 0) {
    barrier_init(shared_address(&up_landed), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const Tile tile = find_tile<kTile, kBlock>(p.offsets, p.n_groups, p.n_tokens, blockIdx.x / members);
  if (tile.count == 0) return;  // of the whole cluster
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const uint32_t n_slice = (p.out_dim + members * 32 - 1) / (members * 32) * 32;
  const uint32_t n_begin = min(p.out_dim, member * n_slice);
  uint32_t n_end = min(p.out_dim, n_begin + n_slice);
  const uint16_t* up = static_cast<const uint16_t*>(p.up) + (long long)tile.group * p.up_stride;
  const bool bare = tile.group == p.n_groups;
  const uint32_t held = VECTOR && !bare ? min(n_end - n_begin, up_room / 2 / p.rank) : 0;  // rows of `up` to bring here
  if (threadIdx.x == 0 && held) {
    const uint32_t bytes = held * p.rank * 2;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(&up_landed)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(shared_address(up_here)),
                 "l"(up + (size_t)n_begin * p.rank), "r"(bytes), "r"(shared_address(&up_landed))
                 : "memory");
    if (held < n_end - n_begin)  // the rest on its way from HBM
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(up + (size_t)(n_begin + held) * p.rank),
                   "r"((n_end - n_begin - held) * p.rank * 2)
                   : "memory");
  }
  if (threadIdx.x < kTile) {
    const uint32_t t = threadIdx.x < tile.count ? (uint32_t)p.order[tile.first + threadIdx.x] : kFull;
    token[threadIdx.x] = t < p.n_tokens ? (int32_t)t : -1;
  }
  __syncthreads();
  const uint16_t* base = static_cast<const uint16_t*>(p.base);
  uint16_t* out = static_cast<uint16_t*>(p.out);

  if (bare) {  // no adapter
    if (out == base) return;
    copy_rows<kBlock, VECTOR>(p, [&](uint32_t m) { return token[m]; }, tile.count, n_begin, n_end, threadIdx.x);
    return;
  }
  // first product: every CTA a slice of dim, 32 of it a warp at a time, several such loads in flight
  {
    const uint16_t* down = static_cast<const uint16_t*>(p.down) + (long long)tile.group * p.down_stride;
    const uint16_t* x = static_cast<const uint16_t*>(p.x);
    const uint32_t k_slice = (p.dim + members * 32 - 1) / (members * 32) * 32;
    const uint32_t k_end = min(p.dim, (member + 1) * k_slice);
    const uint32_t depth_group = warp % S::kDepthGroups, rank0 = warp / S::kDepthGroups * S::kWarpRanks;
    const int t0 = token[g], t1 = token[g + 8];
    constexpr int RT = S::kWarpRanks / 8, kFlight = 2;
    constexpr uint32_t kPace = S::kDepthGroups * 32;
    float acc[RT][4] = {};
    for (uint32_t k0 = member * k_slice + depth_group * 32; k0 < k_end; k0 += kFlight * kPace) {
      uint32_t r0[kFlight][4], r1[kFlight][4], b[kFlight][RT][4];
#pragma unroll
      for (int f = 0; f < kFlight; f++) {
        const uint32_t k = k0 + f * kPace;
        const int at = (int)k + (int)c * 8, valid = k < k_end ? (int)p.dim - at : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) r0[f][i] = r1[f][i] = 0;
        if (t0 >= 0 && valid > 0) load_words<4, VECTOR>(r0[f], x + (long long)t0 * p.x_stride + at, valid);
        if (t1 >= 0 && valid > 0) load_words<4, VECTOR>(r1[f], x + (long long)t1 * p.x_stride + at, valid);
#pragma unroll
        for (int r = 0; r < RT; r++) {
          const uint32_t rank = rank0 + r * 8 + g;
#pragma unroll
          for (int i = 0; i < 4; i++) b[f][r][i] = 0;
          if (rank < p.rank && valid > 0) load_words<4, VECTOR>(b[f][r], down + (size_t)rank * p.dim + at, valid);
        }
      }
#pragma unroll
      for (int r = 0; r < RT; r++) {
        // The matrix unit cuts its sums off, always towards zero, which adds up: where few warps share a row, four
        // instructions are a sum of their own (16,384 columns of one sign, rank 128: 2e-7 off instead of 6e-6).  Up to rank 32
        // a warp has at most 1/32 of the row, and no register to spare.
        float own[4] = {};
        float (&sum)[4] = RP >= 64 ? own : acc[r];
#pragma unroll
        for (int f = 0; f < kFlight; f++) {
          const uint32_t a0[4] = {r0[f][0], r1[f][0], r0[f][1], r1[f][1]}, a1[4] = {r0[f][2], r1[f][2], r0[f][3], r1[f][3]};
          Half<E>::mma(sum, a0, b[f][r][0], b[f][r][1]);
          Half<E>::mma(sum, a1, b[f][r][2], b[f][r][3]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (RP >= 64) acc[r][i] += own[i];
      }
    }
    float* mine = part + (size_t)depth_group * kTile * RP + rank0;
#pragma unroll
    for (int r = 0; r < RT; r++) {
      *reinterpret_cast<float2*>(mine + g * RP + r * 8 + c * 2) = make_float2(acc[r][0], acc[r][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * RP + r * 8 + c * 2) = make_float2(acc[r][2], acc[r][3]);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x * 4; i < tile.count * RP; i += kBlock * 4) {
      float4 sum = *reinterpret_cast<const float4*>(part + i);
#pragma unroll
      for (int w = 1; w < S::kDepthGroups; w++) {
        const float4 v = *reinterpret_cast<const float4*>(part + w * kTile * RP + i);
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      *reinterpret_cast<float4*>(part + i) = sum;
    }
  }
  cluster_arrive();
  uint32_t in[2][2][4] = {};  // base of the warp's next two runs of columns
  auto load_base = [&](uint32_t (&to)[2][4], uint32_t n0) {
#pragma unroll
    for (int o = 0; o < 2; o++) {
      const int t = token[g + 8 * o], at = (int)(n0 + c * 8), valid = (int)n_end - at;
      if (t >= 0 && valid > 0) load_words<4, VECTOR>(to[o], base + (long long)t * p.base_stride + at, valid);
    }
  };
  load_base(in[0], n_begin + warp * 32);
  load_base(in[1], n_begin + warp * 32 + kWarps * 32);
  cluster_wait();
  // the CTAs' sums, in their order, and their terms
  {
    const float scale = p.scale ? p.scale[tile.group] : 1.f;
    constexpr int kRounds = (RP + 63) / 64;
    for (uint32_t m = warp; m < tile.count; m += kWarps) {  // rows behind stay as they are: their products are not stored
      float2 u[kRounds];
      float top = 0.f;
#pragma unroll
      for (int o = 0; o < kRounds; o++) {
        const uint32_t r = o * 64 + lane * 2;
        u[o] = make_float2(0.f, 0.f);
        if (r < RP) {
          float2 v[kMostCluster];
#pragma unroll
          for (int w = 0; w < kMostCluster; w++)
            if (w < members) v[w] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(part, w) + m * RP + r);
#pragma unroll
          for (int w = 0; w < kMostCluster; w++)
            if (w < members) u[o].x += v[w].x, u[o].y += v[w].y;
          // beyond the rank are no products: an infinite x would leave NaN there
          u[o] = make_float2(r < p.rank ? u[o].x * scale : 0.f, r + 1 < p.rank ? u[o].y * scale : 0.f);
        }
        top = fmaxf(top, fmaxf(size_of(u[o].x), size_of(u[o].y)));
      }
      float s = 1.f;
      if (Half<E>::kScaled) {
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
        s = scale_for(top);
      }
      if (lane == 0) back[m] = 1.f / s;
#pragma unroll
      for (int o = 0; o < kRounds; o++) {
        const uint32_t r = o * 64 + lane * 2;
        if (r >= RP) continue;
        uint32_t term[kTerms];
        split<E>(u[o].x * s, u[o].y * s, term);
#pragma unroll
        for (int t = 0; t < kTerms; t++)
          *reinterpret_cast<uint32_t*>(&inner[t * RP / KR][m][t * RP % KR + r]) = term[t];
        if (RP < KR) *reinterpret_cast<uint32_t*>(&inner[1][m][RP + r]) = 0;
      }
    }
  }
  __syncthreads();
  cluster_arrive();  // waited for at the end: nobody leaves while its sums are being read
  if (held && !warp_wait(shared_address(&up_landed), 0)) {
    warp_wait(shared_address(&up_landed), 0);  // once more: the copy's target is the CTA's own memory
    n_end = n_begin;                           // nothing is stored
  }
  __syncwarp();

  // second product: every CTA a slice of out_dim, 32 of it a warp at a time.  Column 2c + b of the
  // q-th of four matrix tiles is output 8c + 2q + b, so that a lane ends with 8 consecutive outputs.
  {
    constexpr int KS = KR >= 32 ? KR / 32 : 1;   // steps of 32 (16) ranks
    constexpr int W = KR >= 32 ? 4 : 2;          // words a lane has of one
    constexpr bool kKeep = KS <= 2;              // 96 registers of terms are too many: rank 128 reads them again
    uint32_t u[kKeep ? KS : 1][S::kSlabs][2][W]; // slab, half of the tile
    auto load_terms = [&](uint32_t (&to)[S::kSlabs][2][W], int s) {
#pragma unroll
      for (int h = 0; h < S::kSlabs; h++)
#pragma unroll
        for (int o = 0; o < 2; o++) load_words<W, true>(to[h][o], &inner[h][g + 8 * o][(s * 4 + c) * 2 * W], 2 * W);
    };
#pragma unroll
    for (int s = 0; s < KS; s++)
      if (kKeep) load_terms(u[kKeep ? s : 0], s);
    for (uint32_t n0 = n_begin + warp * 32; n0 < n_end; n0 += kWarps * 32) {
      const int at = (int)(n0 + c * 8), valid = (int)n_end - at;
      uint32_t y[2][4];
#pragma unroll
      for (int o = 0; o < 2; o++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          y[o][i] = in[0][o][i];
          in[0][o][i] = in[1][o][i];
        }
      load_base(in[1], n0 + 2 * kWarps * 32);
      const bool here = n0 - n_begin + 32 <= held;  // all of the run's rows of `up` are in shared memory
      float acc[4][4] = {};
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const int r = (s * 4 + (int)c) * 2 * W % RP, left = (int)p.rank - r;
        if (!kKeep) load_terms(u[0], s);
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const uint32_t n = n0 + (g >> 1) * 8 + q * 2 + (g & 1);
          uint32_t b[W] = {};
          if (here) {
            if (left > 0) load_words<W, VECTOR>(b, up_here + (n - n_begin) * p.rank + r, left);
          } else if (n < n_end && left > 0) {
            load_words<W, VECTOR>(b, up + (size_t)n * p.rank + r, left);
          }
#pragma unroll
          for (int h = S::kSlabs - 1; h >= 0; h--)  // the small terms first
#pragma unroll
            for (int w = 0; w < W; w += 2) {
              const auto& x = u[kKeep ? s : 0][h];
              const uint32_t a[4] = {x[0][w], x[1][w], x[0][w + 1], x[1][w + 1]};
              Half<E>::mma(acc[q], a, b[w], b[w + 1]);
            }
        }
      }
#pragma unroll
      for (int o = 0; o < 2; o++) {
        const int t = token[g + 8 * o];
        if (t < 0 || valid <= 0) continue;
        const float s = back[g + 8 * o];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const float2 v = Half<E>::widen(y[o][q]);
          y[o][q] = Half<E>::narrow(fmaf(acc[q][2 * o], s, v.x), fmaf(acc[q][2 * o + 1], s, v.y));
        }
        uint16_t* to = out + (long long)t * p.out_stride + at;
        if (VECTOR && valid >= 8) {
          *reinterpret_cast<uint4*>(to) = make_uint4(y[o][0], y[o][1], y[o][2], y[o][3]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (i < valid) to[i] = (uint16_t)(y[o][i / 2] >> (i & 1 ? 16 : 0));
        }
      }
    }
  }
  cluster_wait();
}

// ------------------------------------------------------------------------------------
// fp32 adapters
// ------------------------------------------------------------------------------------
// The matrix units have no fp32 products, so these are fused multiply-adds, 16 tokens a cluster as above: x goes
// through shared memory 256 columns at a time, a warp has a rank and all tokens; then a thread has an output and all
// tokens.  Bound by its instructions: 48 tokens of 64 adapters of rank 16 (4096 x 4096) take 27 us, 16,384 of 24 of
// rank 64 1.55 ms (17 GFLOP; 3.2 ms with every sum shuffled alone and `up` read an element at a time).

constexpr int kF32Columns = 256;

__global__ void __launch_bounds__(kBlock) adapter_f32_kernel(AdapterParams p) {
  extern __shared__ __align__(16) float fsmem[];
  float* part = fsmem;                                             // [token][rank]
  float* inner = part + kTile * kAdapterMaxRank;                   // [rank][token]
  float (*columns)[kF32Columns] = reinterpret_cast<float (*)[kF32Columns]>(inner + kTile * kAdapterMaxRank);  // [token]
  __shared__ int32_t token[kTile];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t member = cluster.block_rank(), members = cluster.num_blocks();
  const Tile tile = find_tile<kTile, kBlock>(p.offsets, p.n_groups, p.n_tokens, blockIdx.x / members);
  if (tile.count == 0) return;  // of the whole cluster
  if (threadIdx.x < kTile) {
    const uint32_t t = threadIdx.x < tile.count ? (uint32_t)p.order[tile.first + threadIdx.x] : kFull;
    token[threadIdx.x] = t < p.n_tokens ? (int32_t)t : -1;
  }
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = p.rank;
  const float* base = static_cast<const float*>(p.base);
  float* out = static_cast<float*>(p.out);
  const bool bare = tile.group == p.n_groups;
  if (bare && out == base) return;
  __syncthreads();

  if (!bare) {
    const float* down = static_cast<const float*>(p.down) + (long long)tile.group * p.down_stride;
    const float* x = static_cast<const float*>(p.x);
    const uint32_t k_slice = (p.dim + members - 1) / members;
    const uint32_t k_end = min(p.dim, (member + 1) * k_slice);
    for (uint32_t i = threadIdx.x; i < kTile * rank; i += kBlock) part[i] = 0.f;
    for (uint32_t k0 = member * k_slice; k0 < k_end; k0 += kF32Columns) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < kTile * kF32Columns; i += kBlock) {
        const uint32_t m = i / kF32Columns, k = k0 + i % kF32Columns;
        columns[m][i % kF32Columns] = token[m] >= 0 && k < k_end ? x[(long long)token[m] * p.x_stride + k] : 0.f;
      }
      __syncthreads();
      for (uint32_t r = warp; r < rank; r += kWarps) {
        float acc[kTile] = {};
#pragma unroll
        for (int c = 0; c < kF32Columns / 32; c++) {
          const uint32_t k = k0 + c * 32 + lane;
          const float d = k < k_end ? down[(size_t)r * p.dim + k] : 0.f;
#pragma unroll
          for (int m = 0; m < kTile; m++) acc[m] = fmaf(columns[m][c * 32 + lane], d, acc[m]);
        }
        uint32_t m;
        const float sum = sum_over_lanes(acc, 32, &m);
        if ((lane & (32 / kTile - 1)) == 0) part[m * rank + r] += sum;
      }
    }
    cluster_arrive();
    cluster_wait();
    const float scale = p.scale ? p.scale[tile.group] : 1.f;
    for (uint32_t i = threadIdx.x; i < kTile * rank; i += kBlock) {  // the CTAs' sums, in their order
      float sum = 0.f;
      for (uint32_t w = 0; w < members; w++) sum += cluster.map_shared_rank(part, w)[i];
      inner[i % rank * kTile + i / rank] = sum * scale;
    }
    __syncthreads();
    cluster_arrive();  // waited for at the end: nobody leaves while its sums are being read
  }
  const uint32_t n_slice = (p.out_dim + members - 1) / members, n_end = min(p.out_dim, (member + 1) * n_slice);
  if (bare) {  // bit for bit: a sum with 0 would turn -0 into 0
    for (uint32_t n = member * n_slice + threadIdx.x; n < n_end; n += kBlock)
#pragma unroll
      for (int m = 0; m < kTile; m++)
        if (token[m] >= 0) out[(long long)token[m] * p.out_stride + n] = base[(long long)token[m] * p.base_stride + n];
    return;
  }
  const float* up = static_cast<const float*>(p.up) + (long long)tile.group * p.up_stride;
  const bool vector = rank % 4 == 0 && reinterpret_cast<uintptr_t>(up) % 16 == 0;
  for (uint32_t n = member * n_slice + threadIdx.x; n < n_end; n += kBlock) {
    float acc[kTile] = {};
    for (uint32_t r = 0; r < rank; r += 4) {
      float u[4] = {};
      if (vector) {
        const float4 v = *reinterpret_cast<const float4*>(up + (size_t)n * rank + r);
        u[0] = v.x, u[1] = v.y, u[2] = v.z, u[3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (r + i < rank) u[i] = up[(size_t)n * rank + r + i];
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (r + i >= rank) break;  // what lies behind the last rank in shared memory is no product
#pragma unroll
        for (int m = 0; m < kTile; m += 4) {
          const float4 x = *reinterpret_cast<const float4*>(inner + (r + i) * kTile + m);
          acc[m] = fmaf(x.x, u[i], acc[m]), acc[m + 1] = fmaf(x.y, u[i], acc[m + 1]);
          acc[m + 2] = fmaf(x.z, u[i], acc[m + 2]), acc[m + 3] = fmaf(x.w, u[i], acc[m + 3]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < kTile; m++)
      if (token[m] >= 0) out[(long long)token[m] * p.out_stride + n] = base[(long long)token[m] * p.base_stride + n] + acc[m];
  }
  cluster_wait();
}

// ------------------------------------------------------------------------------------
// prompts: tiles of 128 tokens on the 5th-generation tensor cores
// ------------------------------------------------------------------------------------
// Two launches.  The first multiplies the tiles' rows of x with their adapters' `down` and leaves fp32
// partial sums in the workspace; the second adds those up, splits them into three 16-bit terms and multiplies
// them with `up`, adding `base` on the way out.  In both a tile is so many steps of 128 columns, the tiles of the
// batch stand one behind the other, and every CTA of a full GPU takes the same number of consecutive
// steps, so that no number of tiles leaves part of the GPU idle; where a CTA's run starts or ends inside a tile
// of the first product, the tile has one more partial sum.
// Steps go through a ring of stages in shared memory: four warps copy (token rows lie anywhere, so 16
// bytes a thread), one thread issues the matrix instructions, the other warps take the products out of
// tensor memory.  HBM bounds it, through the bytes that the ring keeps in flight, and from rank 64 on the shared memory
// that the products read: 4096 x 4096, bf16, 16,384 tokens of 24 adapters of rank 16 / 64 / 128 take 82 / 91 / 122 us (62 /
// 65 / 69 at the rate of a plain copy), 65,536 of rank 64 318 to 328 (250); with two stages less 90 at rank 16.
//
// Operands lie in shared memory in rows of 128 bytes whose 16-byte pieces are exchanged by row (piece c
// of row r at c ^ (r % 8)), as the matrix unit reads them: a line of global memory is a line there, and
// one token a thread reads `base` without bank conflicts.  (Blocks of 8 rows x 16 bytes, the other layout
// the unit takes, split every line over eight and cost 2.5 times the time.)

constexpr int kBigTile = 128;
constexpr int kStep = 128;                                  // columns a step
constexpr int kBlock64 = kBigTile * 128;                    // 64 columns of a tile's rows
constexpr int kRowsBytes = kBigTile * kStep * 2;            // x or base of a step
constexpr int kProducers = 128;
constexpr int kDownThreads = kProducers + 128 + 32;         // copy, take out, multiply
constexpr int kUpThreads = kProducers + 256 + 32;
constexpr int kMostTiles = 36;                              // a CTA's run touches

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// What the thread has written or been told of becomes visible to the matrix instructions issued behind it.
// For copied operands the issuing thread does this, behind the barrier: a copying thread's fence would wait
// for its copies of later steps too.
__device__ __forceinline__ void order_for_tensor_cores() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Operand in shared memory: rows of 128 bytes with exchanged pieces, 1024 bytes from 8 rows to the next.
__device__ __forceinline__ uint64_t operand(uint32_t address) {
  return (uint64_t)(address >> 4 & 0x3fff) | 1ull << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// 16-byte piece c of row r
__device__ __forceinline__ uint32_t piece_at(uint32_t r, uint32_t c) { return r * 128 + ((c ^ (r & 7)) << 4); }
// 128 x n products of 16-bit values, both operands with their depth contiguous, fp32 sums.
template <typename E>
__host__ __device__ constexpr uint32_t instruction(int n) {
  const uint32_t type = std::is_same<E, __half>::value ? 0 : 1;
  return 1u << 4 | type << 7 | type << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(kBigTile >> 4) << 24;
}
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(what), "r"(add ? 1u : 0u)
      : "memory");
}
// The barrier gets an arrival when the matrix instructions issued so far are done.
__device__ __forceinline__ void arrive_behind_products(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <int COLUMNS>
__device__ __forceinline__ void tensor_memory(uint32_t* slot) {  // by one warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(slot)), "n"(COLUMNS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLUMNS>
__device__ __forceinline__ void free_tensor_memory(uint32_t at) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "n"(COLUMNS));
}
// 16 columns of the warp's 32 lanes, one lane a thread.
__device__ __forceinline__ void from_tensor_memory(float (&v)[16], uint32_t at) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
// The loads into v have landed (v passes through, so that nothing reads it ahead of this).
template <int N>
__device__ __forceinline__ void loads_done(float (&v)[N][16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int c = 0; c < N; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) asm volatile("" : "+f"(v[c][i]));
}
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ int token_at(const AdapterParams& p, const Tile& tile, uint32_t place) {
  const uint32_t t = place < tile.count ? (uint32_t)p.order[tile.first + place] : kFull;
  return t < p.n_tokens ? (int)t : -1;
}

// The barrier gets the thread's arrival when the copies that it has issued so far have landed.
__device__ __forceinline__ void arrive_behind_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// A thread's share of a step's token rows, one of four warps: piece lane % 8 of rows 4 * (warp + 4 * i) + lane / 8.
struct RowCopies {
  const uint16_t* row[8];  // nullptr: no token there
  __device__ __forceinline__ void set(const void* rows, long long stride, const AdapterParams& p, const Tile& tile) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int t = token_at(p, tile, place(i));
      row[i] = t < 0 ? nullptr : static_cast<const uint16_t*>(rows) + (long long)t * stride + (threadIdx.x & 7) * 8;
    }
  }
  static __device__ __forceinline__ uint32_t place(int i) { return 4 * ((threadIdx.x >> 5) + 4 * i) + (threadIdx.x >> 3 & 3); }
  __device__ __forceinline__ void issue(uint32_t to, uint32_t column, uint32_t end) const {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (!row[i]) continue;
#pragma unroll
      for (int b = 0; b < kStep / 64; b++) {
        const bool live = column + b * 64 + (threadIdx.x & 7) * 8 < end;
        copy16(to + b * kBlock64 + piece_at(place(i), threadIdx.x & 7), live ? row[i] + column + b * 64 : row[i], live);
      }
    }
  }
};

// N_ROWS x (8 * N_PIECES) elements of a matrix; beyond 64 elements a row goes on in another block of all rows.
// Rows from live_rows on and columns from live_end on are zeros.
template <int N_ROWS, int N_PIECES>
__device__ __forceinline__ void copy_matrix(uint32_t to, const uint16_t* from, size_t stride, uint32_t row, uint32_t live_rows,
                                            uint32_t column, uint32_t live_end) {
  static_assert(N_ROWS * N_PIECES % kProducers == 0, "every thread copies the same number");
#pragma unroll
  for (int i = 0; i < N_ROWS * N_PIECES / kProducers; i++) {
    const uint32_t item = threadIdx.x + i * kProducers, c = item % N_PIECES, r = item / N_PIECES, at = column + c * 8;
    const bool live = row + r < live_rows && at < live_end;
    copy16(to + c / 8 * (N_ROWS * 128) + piece_at(r, c % 8), live ? from + (row + r) * stride + at : from, live);
  }
}

template <int RP>
struct BigShape {
  static constexpr int kDownStage = kRowsBytes + RP * kStep * 2;                // x, down
  static constexpr int kUpStage = kRowsBytes + (RP + 63) / 64 * kStep * 128;    // base, up
  static constexpr int kTermBytes = (kTerms * RP + 63) / 64 * kBigTile * 128;   // the rank products: first terms, then second, then third
  // one CTA an SM, as many stages as fit
  static constexpr int kDownStages = RP <= 32 ? 5 : RP <= 64 ? 4 : 3;
  static constexpr int kUpStages = RP <= 32 ? 4 : RP <= 64 ? 3 : 2;
  static constexpr int kDownShared = kDownStages * kDownStage + 1024;
  static constexpr int kUpShared = kUpStages * kUpStage + kTermBytes + 1024;
};

__device__ __forceinline__ uint32_t aligned_shared(unsigned char* smem) { return (shared_address(smem) + 1023) / 1024 * 1024; }

// How many steps a CTA of a launch takes.
struct BigShare {
  uint32_t tile_steps;  // steps of a tile
  uint32_t least;       // steps of a run, at least
  uint32_t grid;
  __device__ __forceinline__ uint32_t run(uint32_t tiles) const {
    return max((uint32_t)(((unsigned long long)tiles * tile_steps + grid - 1) / grid), least);
  }
};

// A CTA's run: its tiles and the steps of each.
struct Run {
  uint32_t tiles;          // tiles with an adapter in the batch
  uint32_t first, count;   // tiles of the run
  unsigned long long begin, end;
  uint32_t tile_steps;
  __device__ __forceinline__ uint32_t from(uint32_t i) const {
    const unsigned long long at = (unsigned long long)(first + i) * tile_steps;
    return begin > at ? (uint32_t)(begin - at) : 0;
  }
  __device__ __forceinline__ uint32_t to(uint32_t i) const {
    const unsigned long long at = (unsigned long long)(first + i) * tile_steps;
    return (uint32_t)min(end - at, (unsigned long long)tile_steps);
  }
};

// By the whole CTA; `bare`: tiles of tokens without an adapter count as well.
template <int THREADS>
__device__ Run find_run(const AdapterParams& p, const BigShare& share, bool bare, Tile* found) {
  __shared__ uint32_t partial[THREADS / 32], total[2];
  const uint32_t n = p.n_groups + 1, per = (n + THREADS - 1) / THREADS, g0 = threadIdx.x * per;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto begin_of = [&](uint32_t g) { return min((uint32_t)max(p.offsets[g], 0), p.n_tokens); };
  auto tile_of = [&](uint32_t g) {  // the group as one tile
    const uint32_t a = begin_of(g), b = g < p.n_groups ? begin_of(g + 1) : p.n_tokens;
    return Tile{g, a, b > a ? b - a : 0};
  };
  uint32_t sum = 0;
  for (uint32_t i = 0; i < per; i++)
    if (g0 + i < n) sum += (tile_of(g0 + i).count + kBigTile - 1) / kBigTile;
  uint32_t inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(kFull, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) partial[warp] = inc;
  __syncthreads();
  uint32_t at = inc - sum;
  for (uint32_t w = 0; w < warp; w++) at += partial[w];
  for (uint32_t i = 0, t = at; i < per && g0 + i < n; i++) {
    if (g0 + i == p.n_groups) total[0] = t;
    t += (tile_of(g0 + i).count + kBigTile - 1) / kBigTile;
    if (g0 + i == p.n_groups) total[1] = t;
  }
  __syncthreads();
  Run r;
  r.tiles = total[0];
  r.tile_steps = share.tile_steps;
  const uint32_t all = bare ? total[1] : total[0];
  const unsigned long long steps = share.run(all);
  r.begin = min(blockIdx.x * steps, (unsigned long long)all * share.tile_steps);
  r.end = min(r.begin + steps, (unsigned long long)all * share.tile_steps);
  r.first = (uint32_t)(r.begin / share.tile_steps);
  r.count = r.end > r.begin ? min((uint32_t)((r.end - 1) / share.tile_steps) - r.first + 1, (uint32_t)kMostTiles) : 0;
  if (at < r.first + r.count && at + sum > r.first) {
    for (uint32_t i = 0; i < per && g0 + i < n; i++) {
      const Tile g = tile_of(g0 + i);
      for (uint32_t o = 0; o < g.count; o += kBigTile, at++)
        if (at >= r.first && at < r.first + r.count) found[at - r.first] = Tile{g.group, g.first + o, min(g.count - o, (uint32_t)kBigTile)};
    }
  }
  __syncthreads();
  return r;
}

// inner[part] = x rows of the tile times a run of columns of `down`; a tile's RP products a token lie as
// [RP / 4][tokens][4], so that one token a thread writes and reads whole lines.
template <typename E, int RP>
__global__ void __launch_bounds__(kDownThreads, 1) adapter_down_kernel(AdapterParams p, float* __restrict__ inner, BigShare share) {
  using S = BigShape<RP>;
  constexpr int kStages = S::kDownStages, kColumns = 2 * RP, kLoads = RP < 64 ? RP / 16 : 4;
  extern __shared__ unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], ready[2], taken[2];
  __shared__ uint32_t tmem_slot;
  __shared__ Tile tiles[kMostTiles];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Run run = find_run<kDownThreads>(p, share, false, tiles);
  if (run.count == 0) return;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; i++) {
      barrier_init(shared_address(&full[i]), kProducers);
      barrier_init(shared_address(&empty[i]), 1);
    }
    for (int i = 0; i < 2; i++) {
      barrier_init(shared_address(&ready[i]), 1);
      barrier_init(shared_address(&taken[i]), 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) tensor_memory<kColumns>(&tmem_slot);
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = tmem_slot, ring = aligned_shared(smem);

  if (warp < 4) {
    uint32_t i = 0;
    bool ok = true;
    for (uint32_t n = 0; ok && n < run.count; n++) {
      const Tile tile = tiles[n];
      RowCopies x;
      x.set(p.x, p.x_stride, p, tile);
      const uint16_t* down = static_cast<const uint16_t*>(p.down) + (long long)tile.group * p.down_stride;
      for (uint32_t k = run.from(n), end = run.to(n); k < end; k++, i++) {
        const uint32_t s = i % kStages;
        if (i >= kStages && !(ok = barrier_wait(shared_address(&empty[s]), (i / kStages - 1) & 1))) break;
        const uint32_t to = ring + s * S::kDownStage, column = k * kStep;
        x.issue(to, column, p.dim);
        copy_matrix<RP, kStep / 8>(to + kRowsBytes, down, p.dim, 0, p.rank, column, p.dim);
        arrive_behind_copies(shared_address(&full[s]));
      }
    }
    copies_done();
  } else if (warp < 8) {
    // The matrix unit cuts its sums off at 24 bits, always towards zero: over the 256 instructions of 4096 columns of one
    // sign that made 7e-6 of the sum.  So a step's products (8 instructions) are a sum of their own, added up here.
    const uint32_t row = threadIdx.x - kProducers;
    uint32_t i = 0;
    bool ok = true;
    for (uint32_t n = 0; ok && n < run.count; n++) {
      const Tile tile = tiles[n];
      float sum[RP / 16][16];
#pragma unroll
      for (int c = 0; c < RP; c++) sum[c / 16][c % 16] = 0.f;
      for (uint32_t k = run.from(n), end = run.to(n); k < end; k++, i++) {
        if (!(ok = warp_wait(shared_address(&ready[i & 1]), i / 2 & 1))) break;
        after_sync();
#pragma unroll
        for (int c0 = 0; c0 < RP / 16; c0 += kLoads) {
          float v[kLoads][16];
#pragma unroll
          for (int c = 0; c < kLoads; c++) from_tensor_memory(v[c], tmem + ((warp - 4) * 32 << 16) + (i & 1) * RP + (c0 + c) * 16);
          loads_done(v);
#pragma unroll
          for (int c = 0; c < kLoads * 16; c++) sum[c0 + c / 16][c % 16] += v[c / 16][c % 16];
        }
        before_sync();
        __syncwarp();
        if (lane == 0) barrier_arrive(shared_address(&taken[i & 1]));
      }
      if (!ok) break;
      const uint32_t part = blockIdx.x - (uint32_t)((unsigned long long)(run.first + n) * run.tile_steps / share.run(run.tiles));
      float* to = inner + ((size_t)part * p.n_tokens + tile.first) * RP + row * 4;
      if (row < tile.count) {
#pragma unroll
        for (int c = 0; c < RP; c += 4) {
          const float* s = &sum[c / 16][c % 16];
          *reinterpret_cast<float4*>(to + (size_t)c * tile.count) = make_float4(s[0], s[1], s[2], s[3]);
        }
      }
    }
  } else if (lane == 0) {
    uint32_t i = 0;
    bool ok = true;
    for (uint32_t n = 0; ok && n < run.count; n++)
      for (uint32_t k = run.from(n), end = run.to(n); k < end; k++, i++) {
        const uint32_t s = i % kStages, at = ring + s * S::kDownStage;
        ok = barrier_wait(shared_address(&full[s]), i / kStages & 1) &&
             (i < 2 || barrier_wait(shared_address(&taken[i & 1]), (i / 2 - 1) & 1));
        if (!ok) break;
        order_for_tensor_cores();
        after_sync();
#pragma unroll
        for (int q = 0; q < kStep / 16; q++)
          multiply(tmem + (i & 1) * RP, operand(at + q / 4 * kBlock64 + q % 4 * 32),
                   operand(at + kRowsBytes + q / 4 * (RP * 128) + q % 4 * 32), instruction<E>(RP), q > 0);
        arrive_behind_products(shared_address(&empty[s]));
        arrive_behind_products(shared_address(&ready[i & 1]));
      }
  }
  before_sync();
  __syncthreads();
  after_sync();
  __syncwarp();
  if (warp == 8) free_tensor_memory<kColumns>(tmem);
}

template <typename E, int RP>
__global__ void __launch_bounds__(kUpThreads, 1)
    adapter_up_kernel(AdapterParams p, const float* __restrict__ inner, BigShare down_share, BigShare share) {
  using S = BigShape<RP>;
  constexpr int kStages = S::kUpStages, kColumns = 2 * kStep;
  constexpr int kWide = 4;  // pieces a thread takes out at once; with eight rank 128 is no faster and rank 64 slower (92 us)
  extern __shared__ unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kStages], drained[kStages], product[2], taken[2], terms, tops;
  __shared__ uint32_t tmem_slot;
  __shared__ float top_of[2][kBigTile];
  __shared__ Tile tiles[kMostTiles];
  // the launch ahead (the first product) started behind everything that wrote base, up and the plan
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Run run = find_run<kUpThreads>(p, share, p.out != p.base, tiles);
  if (run.count == 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; i++) {
      barrier_init(shared_address(&full[i]), kProducers);
      barrier_init(shared_address(&drained[i]), 8);
    }
    for (int i = 0; i < 2; i++) {
      barrier_init(shared_address(&product[i]), 1);
      barrier_init(shared_address(&taken[i]), 8);
    }
    barrier_init(shared_address(&terms), 256);
    barrier_init(shared_address(&tops), 256);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) tensor_memory<kColumns>(&tmem_slot);
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = tmem_slot, ring = aligned_shared(smem), term = ring + kStages * S::kUpStage;
  uint16_t* out = static_cast<uint16_t*>(p.out);

  if (warp < 4) {
    uint32_t i = 0;
    bool ok = true;
    for (uint32_t n = 0; ok && n < run.count; n++) {
      const Tile tile = tiles[n];
      const bool bare = tile.group == p.n_groups;  // no adapter: these tiles come last, their rows just pass through
      RowCopies base;
      base.set(p.base, p.base_stride, p, tile);
      const uint16_t* up = static_cast<const uint16_t*>(p.up) + (long long)tile.group * p.up_stride;
      for (uint32_t k = run.from(n), end = run.to(n); k < end; k++, i++) {
        const uint32_t s = i % kStages;
        if (i >= kStages && !(ok = barrier_wait(shared_address(&drained[s]), (i / kStages - 1) & 1))) break;
        const uint32_t to = ring + s * S::kUpStage, column = k * kStep;
        base.issue(to, column, p.out_dim);
        if (!bare) copy_matrix<kStep, RP / 8>(to + kRowsBytes, up, p.rank, column, p.out_dim, 0, p.rank);
        arrive_behind_copies(shared_address(&full[s]));
      }
    }
    copies_done();
  } else if (warp < 12) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t quarter = warp & 3, half = (warp - 4) >> 2, row = quarter * 32 + lane;
    static_assert(kStep == 128, "a half of the step's columns is one block of 64");
    const uint32_t block = half * kBlock64, out_piece = lane & 7, out_row = quarter * 32 + (lane >> 3);
    uint32_t i = 0;
    bool ok = true;
    for (uint32_t n = 0; ok && n < run.count; n++) {
      const Tile tile = tiles[n];
      const bool bare = tile.group == p.n_groups;
      float back = 1.f;
      if (!bare) {  // half of the token's rank products a thread: added up, scaled, in three terms
        constexpr int R = RP / 2;
        const float scale = p.scale ? p.scale[tile.group] : 1.f;
        const uint32_t per = down_share.run(run.tiles);
        const unsigned long long at = (unsigned long long)(run.first + n) * down_share.tile_steps;
        const uint32_t parts = (uint32_t)((at + down_share.tile_steps - 1) / per - at / per) + 1;
        const float* from = inner + (size_t)tile.first * RP + (size_t)half * R * tile.count + min(row, tile.count - 1) * 4;
        float u[R], top = 0.f;
#pragma unroll
        for (int c = 0; c < R; c++) u[c] = 0.f;
        for (uint32_t m = 0; m < parts; m++, from += (size_t)p.n_tokens * RP) {
#pragma unroll
          for (int c = 0; c < R; c += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(from + (size_t)c * tile.count));
            u[c] += v.x, u[c + 1] += v.y, u[c + 2] += v.z, u[c + 3] += v.w;
          }
        }
#pragma unroll
        for (int c = 0; c < R; c++) {
          u[c] = half * R + c < p.rank ? u[c] * scale : 0.f;  // an infinite x leaves NaN beyond the rank
          top = fmaxf(top, size_of(u[c]));
        }
        float s = 1.f;
        if (Half<E>::kScaled) {
          top_of[half][row] = top;
          barrier_arrive(shared_address(&tops));
          if (!(ok = warp_wait(shared_address(&tops), n & 1))) break;
          s = scale_for(fmaxf(top, top_of[half ^ 1][row]));
          back = 1.f / s;
        }
#pragma unroll
        for (int c = 0; c < R; c += 8) {
          uint32_t term_of[4][kTerms];
#pragma unroll
          for (int j = 0; j < 4; j++) split<E>(u[c + 2 * j] * s, u[c + 2 * j + 1] * s, term_of[j]);
#pragma unroll
          for (int t = 0; t < kTerms; t++) {
            const uint32_t q = t * (RP / 8) + (half * R + c) / 8, to = term + q / 8 * kBlock64 + piece_at(row, q % 8);
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(term_of[0][t]), "r"(term_of[1][t]),
                         "r"(term_of[2][t]), "r"(term_of[3][t])
                         : "memory");
          }
        }
      }
      if (!bare) {
        order_for_tensor_cores();
        barrier_arrive(shared_address(&terms));
      }
      uint16_t* to[8];  // on the way out the thread has one piece of eight rows
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int t = token_at(p, tile, out_row + 4 * j);
        to[j] = t < 0 ? nullptr : out + (long long)t * p.out_stride + half * 64 + out_piece * 8;
      }
      for (uint32_t k = run.from(n), end = run.to(n); k < end; k++, i++) {
        const uint32_t s = i % kStages, at = ring + s * S::kUpStage, column = k * kStep;
        ok = warp_wait(shared_address(&full[s]), i / kStages & 1) && (bare || warp_wait(shared_address(&product[i & 1]), i / 2 & 1));
        if (!ok) break;
        after_sync();
#pragma unroll
        for (int c0 = 0; c0 < 8 && !bare; c0 += kWide) {
          float v[kWide / 2][16];
#pragma unroll
          for (int c = 0; c < kWide / 2; c++)
            from_tensor_memory(v[c], tmem + (quarter * 32 << 16) + (i & 1) * kStep + half * 64 + c0 * 8 + c * 16);
          uint32_t w[kWide][4];
#pragma unroll
          for (int c = 0; c < kWide; c++)
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[c][0]), "=r"(w[c][1]), "=r"(w[c][2]), "=r"(w[c][3])
                         : "r"(at + block + piece_at(row, c0 + c))
                         : "memory");
          loads_done(v);
#pragma unroll
          for (int c = 0; c < kWide; c++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float2 b = Half<E>::widen(w[c][j]);
              const float* d = &v[c / 2][c % 2 * 8 + 2 * j];
              w[c][j] = Half<E>::narrow(fmaf(d[0], back, b.x), fmaf(d[1], back, b.y));
            }
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + block + piece_at(row, c0 + c)), "r"(w[c][0]),
                         "r"(w[c][1]), "r"(w[c][2]), "r"(w[c][3])
                         : "memory");
          }
        }
        before_sync();
        __syncwarp();
        if (lane == 0 && !bare) barrier_arrive(shared_address(&taken[i & 1]));
#pragma unroll
        for (int j = 0; j < 8; j++) {
          uint32_t w[4];
          asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(at + block + piece_at(out_row + 4 * j, out_piece))
                       : "memory");
          if (to[j] && column + half * 64 + out_piece * 8 < p.out_dim) *reinterpret_cast<uint4*>(to[j] + column) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        if (lane == 0) barrier_arrive(shared_address(&drained[s]));
      }
    }
  } else if (lane == 0) {
    uint32_t i = 0;
    bool ok = true;
    for (uint32_t n = 0; ok && n < run.count; n++) {
      if (tiles[n].group == p.n_groups) break;
      if (!(ok = barrier_wait(shared_address(&terms), n & 1))) break;
      for (uint32_t k = run.from(n), end = run.to(n); k < end; k++, i++) {
        const uint32_t s = i % kStages, at = ring + s * S::kUpStage + kRowsBytes;
        ok = barrier_wait(shared_address(&full[s]), i / kStages & 1) &&
             (i < 2 || barrier_wait(shared_address(&taken[i & 1]), (i / 2 - 1) & 1));
        if (!ok) break;
        order_for_tensor_cores();
        after_sync();
#pragma unroll
        for (int q = kTerms * (RP / 16) - 1; q >= 0; q--) {  // sixteen ranks of a term; the small terms first, while little is cut off
          const int r = q % (RP / 16);
          multiply(tmem + (i & 1) * kStep, operand(term + q / 4 * kBlock64 + q % 4 * 32),
                   operand(at + r / 4 * (kStep * 128) + r % 4 * 32), instruction<E>(kStep), q < kTerms * (RP / 16) - 1);
        }
        arrive_behind_products(shared_address(&product[i & 1]));
      }
    }
  }
  before_sync();
  __syncthreads();
  after_sync();
  __syncwarp();
  if (warp == 12) free_tensor_memory<kColumns>(tmem);
}

// Tiles of 16 tokens, at most: every group may end in one of its own.
uint32_t small_tiles(const AdapterParams& p) { return p.n_tokens / kTile + std::min(p.n_groups + 1, p.n_tokens); }

constexpr uint32_t kMostShared = 200 * 1024;  // of a CTA of the kernels below, at most

// A cluster of CTAs a tile.
template <typename... KArgs, typename... Args>
cudaError_t cluster_launch(void (*kern)(KArgs...), uint32_t tiles, uint32_t cluster, size_t smem, cudaStream_t stream,
                           const Args&... args) {
  if (smem > 47 * 1024) {  // beside what is static; the same bound in every call, for another thread may launch the kernel just now
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * cluster);
  cfg.blockDim = dim3(kBlock);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {cluster, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <typename E, int RP>
cudaError_t adapter_launch(const AdapterParams& p, bool vector, cudaStream_t stream) {
  using S = SmallShape<RP>;
  auto kern = vector ? adapter_kernel<E, RP, true> : adapter_kernel<E, RP, false>;
  constexpr uint32_t kSms = 148;
  const uint32_t tiles = small_tiles(p);
  // Clusters of 8 are the shorter chain, of 4 the less work a tile: 64 tokens of 63 adapters of rank 16 (4096 x 4096) 9.9
  // against 11.0 us, 128 of 127 18.5 against 14.4.
  const bool few = tiles * kMostCluster <= kSms * 9 / 2;
  const uint32_t cluster = few ? kMostCluster : kMostCluster / 2;
  // CTAs an SM, by shared memory: as few as hold the batch, so that they spread over all SMs (packed onto few
  // of them 30 tiles took 9.9 us instead of 8.5), and of small clusters at most three (1111 tokens of 200 adapters 30.2 us
  // with four, 28.9 with three).  What is left of it holds `up`.
  constexpr uint32_t kMost = RP <= 32 ? 3 : 2;
  const uint32_t per_sm = std::min((tiles * cluster + kSms - 1) / kSms, few && RP <= 16 ? 4 : kMost);
  const uint32_t budget = std::min(216u * 1024 / per_sm, kMostShared);
  const uint32_t slice = (p.out_dim + cluster * 32 - 1) / (cluster * 32) * 32;
  const uint32_t room = vector ? (uint32_t)std::min<size_t>(budget - S::kShared, (size_t)slice * p.rank * 2) / 16 * 16 : 0;
  return cluster_launch(kern, tiles, cluster, budget, stream, p, room);
}

int padded_rank(uint32_t rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// Runs of both products.  At most: every group may end in a tile of its own.
struct BigSplit {
  BigShare down, up;
  uint32_t parts;  // partial sums a tile has, at most
};
BigSplit big_split(uint32_t n_tokens, uint32_t n_groups, uint32_t rank, uint32_t dim, uint32_t out_dim) {
  constexpr uint32_t kSlots = 148, kLeastUp = 2;
  // what a run of the second product reads first is 512 bytes x ranks x parts
  const uint32_t most_parts = std::max(3, std::min(8, 256 / padded_rank(rank)));
  const uint32_t most_tiles = n_tokens / kBigTile + std::min(n_groups + 1, n_tokens), tiles = (n_tokens + kBigTile - 1) / kBigTile;
  const uint32_t grid = std::max(kSlots, (most_tiles + kMostTiles - 4) / (kMostTiles - 3));
  auto over = [](unsigned long long a, unsigned long long b) { return (uint32_t)((a + b - 1) / b); };
  BigSplit b;
  b.down.tile_steps = over(dim, kStep);
  b.up.tile_steps = over(out_dim, kStep);
  b.down.grid = b.up.grid = grid;
  b.down.least = std::max(over((unsigned long long)tiles * b.down.tile_steps, grid), over(b.down.tile_steps, most_parts - 1));
  b.up.least = std::min(kLeastUp, b.up.tile_steps);
  b.parts = over(b.down.tile_steps, b.down.least) + 1;
  return b;
}

// Tiles of 128 or of 16 tokens.  Against a tile of 16, one of 128 reads an adapter's matrices an eighth as often
// but has a longer chain and two launches; what the former costs grows with tokens x rank.  Measured, 4096 x 4096,
// inputs beyond the L2, 16 | 128 a tile, us: rank 16: 4096 tokens of 8 adapters 50 | 28, of 128 55 | 62, of 256 65 | 111; rank 64:
// 256 of 8 15 | 21, 640 of 8 28 | 21, 1024 of 32 48 | 33, of 64 52 | 42; rank 128: 256 of 8 29 | 28, 320 of 8 29 | 28, 512 of 8 48 | 28.
// Near the borders the two are close, or lie a little to either side (rank 16: 2048 of 8 32 | 23; 26 | 22 from the L2).
bool big_batch(uint32_t n_tokens, uint32_t n_groups, uint32_t rank) {
  const unsigned long long work = (unsigned long long)n_tokens * padded_rank(rank);
  return work >= 40960 && work >= 512ull * n_groups;
}

template <typename E, int RP>
cudaError_t big_launch(const AdapterParams& p, float* inner, cudaStream_t stream) {
  using S = BigShape<RP>;
  auto down = adapter_down_kernel<E, RP>;
  auto up = adapter_up_kernel<E, RP>;
  cudaError_t e = cudaFuncSetAttribute(down, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kDownShared);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(up, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kUpShared);
  if (e != cudaSuccess) return e;
  const BigSplit b = big_split(p.n_tokens, p.n_groups, p.rank, p.dim, p.out_dim);
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(b.down.grid);
  cfg.blockDim = dim3(kDownThreads);
  cfg.dynamicSmemBytes = S::kDownShared;
  e = cudaLaunchKernelEx(&cfg, down, p, inner, b.down);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(b.up.grid);
  cfg.blockDim = dim3(kUpThreads);
  cfg.dynamicSmemBytes = S::kUpShared;
  return cudaLaunchKernelEx(&cfg, up, p, static_cast<const float*>(inner), b.down, b.up);
}

}  // namespace

size_t adapter_scratch_bytes(uint32_t n_tokens, uint32_t n_groups, uint32_t rank, uint32_t dim, uint32_t out_dim) {
  if (!big_batch(n_tokens, n_groups, rank)) return 0;
  return (size_t)big_split(n_tokens, n_groups, rank, dim, out_dim).parts * n_tokens * padded_rank(rank) * sizeof(float);
}

cudaError_t adapter_stalled(uint32_t* count) { return cudaMemcpyFromSymbol(count, g_stalled, sizeof(*count)); }

cudaError_t launch_adapter_add(const AdapterParams& p, int elem, void* scratch, cudaStream_t stream) {
  if (p.n_tokens == 0) return cudaSuccess;
  if (elem == kElemF32) {
    const size_t smem = (2 * kTile * kAdapterMaxRank + kTile * kF32Columns) * sizeof(float);
    return cluster_launch(adapter_f32_kernel, small_tiles(p), kMostCluster, smem, stream, p);
  }
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(p.base) | reinterpret_cast<uintptr_t>(p.x) |
                              reinterpret_cast<uintptr_t>(p.down) | reinterpret_cast<uintptr_t>(p.up) |
                              reinterpret_cast<uintptr_t>(p.out);
  const unsigned long long strides = (unsigned long long)p.base_stride | p.x_stride | p.down_stride | p.up_stride | p.out_stride;
  const bool vector = addresses % 16 == 0 && strides % 8 == 0 && p.dim % 8 == 0 && p.out_dim % 8 == 0 && p.rank % 8 == 0;
  auto by_rank = [&](auto e) {
    using E = decltype(e);
    if (vector && big_batch(p.n_tokens, p.n_groups, p.rank)) {
      float* inner = static_cast<float*>(scratch);
      switch (padded_rank(p.rank)) {
        case 16: return big_launch<E, 16>(p, inner, stream);
        case 32: return big_launch<E, 32>(p, inner, stream);
        case 64: return big_launch<E, 64>(p, inner, stream);
        default: return big_launch<E, 128>(p, inner, stream);
      }
    }
    if (p.rank <= 8) return adapter_launch<E, 8>(p, vector, stream);
    if (p.rank <= 16) return adapter_launch<E, 16>(p, vector, stream);
    if (p.rank <= 32) return adapter_launch<E, 32>(p, vector, stream);
    if (p.rank <= 64) return adapter_launch<E, 64>(p, vector, stream);
    return adapter_launch<E, 128>(p, vector, stream);
  };
  return elem == kElemF16 ? by_rank(__half{}) : by_rank(__nv_bfloat16{});
}

}  // namespace ugc
