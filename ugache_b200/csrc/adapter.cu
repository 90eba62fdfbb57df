// Low-rank adapters of many requests at once: out[t] = base[t] + scale[a] * (x[t] down[a]^T) up[a]^T.
#include "routing.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace ugc {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 8;
constexpr int kBlock = kWarps * 32;
constexpr int kCluster = 8;   // CTAs that share a tile of tokens
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

// A power of two s with max * s in [1, 2); 1 where there is none.
__device__ __forceinline__ float unit_scale(float max) {
  const int e = (int)(__float_as_uint(max) >> 23 & 255) - 127;
  return max > 0.f && e > -120 && e < 126 ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.f;
}

// The tile of this cluster: tiles of 16 tokens, group by group, those without a group last.
struct Tile {
  uint32_t group, first, count;  // first: place in `order`
};
__device__ Tile find_tile(const int32_t* offsets, uint32_t n_groups, uint32_t n_tokens, uint32_t index) {
  __shared__ uint32_t partial[kWarps];
  __shared__ Tile found;
  const uint32_t n = n_groups + 1, per = (n + kBlock - 1) / kBlock, g0 = threadIdx.x * per;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto begin_of = [&](uint32_t g) { return min((uint32_t)max(offsets[g], 0), n_tokens); };
  auto tiles_of = [&](uint32_t g) {
    const uint32_t a = begin_of(g), b = g < n_groups ? begin_of(g + 1) : n_tokens;
    return b > a ? (b - a + kTile - 1) / kTile : 0;
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
        const uint32_t first = a + (index - at) * kTile;
        found = Tile{g0 + i, first, min(b - first, (uint32_t)kTile)};
        break;
      }
      at += m;
    }
  }
  __syncthreads();
  return found;
}

// RP: rank rounded up to 8, 16, 32, 64 or 128.
template <typename E, int RP, bool VECTOR>
__global__ void __launch_bounds__(kBlock) adapter_kernel(AdapterParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int RT = RP / 8;                 // tiles of 8 ranks
  constexpr int KR = RP < 16 ? 16 : RP;      // ranks as the second product's depth
  extern __shared__ __align__(16) unsigned char smem[];
  using Part = float[kTile][RP];
  using Inner = uint16_t[kTile][KR + 8];
  Part* part = reinterpret_cast<Part*>(smem);                            // [kWarps] of each warp, then [0]: of the CTA
  Inner* inner = reinterpret_cast<Inner*>(smem + kWarps * sizeof(Part)); // [2] the two terms
  __shared__ float back[kTile];
  __shared__ int32_t token[kTile];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t member = cluster.block_rank();
  const Tile tile = find_tile(p.offsets, p.n_groups, p.n_tokens, blockIdx.x / kCluster);
  if (tile.count == 0) return;  // of the whole cluster
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  if (threadIdx.x < kTile) {
    const uint32_t t = threadIdx.x < tile.count ? (uint32_t)p.order[tile.first + threadIdx.x] : kFull;
    token[threadIdx.x] = t < p.n_tokens ? (int32_t)t : -1;
  }
  __syncthreads();
  const uint16_t* base = static_cast<const uint16_t*>(p.base);
  uint16_t* out = static_cast<uint16_t*>(p.out);
  const uint32_t n_slice = (p.out_dim + kCluster * 32 - 1) / (kCluster * 32) * 32;
  const uint32_t n_begin = member * n_slice, n_end = min(p.out_dim, n_begin + n_slice);

  if (tile.group == p.n_groups) {  // no adapter
    if (out == base) return;
    for (uint32_t m = warp; m < tile.count; m += kWarps) {
      if (token[m] < 0) continue;
      const uint16_t* from = base + (long long)token[m] * p.base_stride;
      uint16_t* to = out + (long long)token[m] * p.out_stride;
      for (uint32_t n = n_begin + lane * 8; n < n_end; n += 256) {
        if (VECTOR && n + 8 <= n_end) {
          *reinterpret_cast<uint4*>(to + n) = *reinterpret_cast<const uint4*>(from + n);
        } else {
          for (uint32_t i = n; i < min(n + 8, n_end); i++) to[i] = from[i];
        }
      }
    }
    return;
  }

  // first product: every CTA a slice of dim, its warps 32 of it at a time
  {
    const uint16_t* down = static_cast<const uint16_t*>(p.down) + (long long)tile.group * p.down_stride;
    const uint16_t* x = static_cast<const uint16_t*>(p.x);
    const uint32_t k_slice = (p.dim + kCluster * 32 - 1) / (kCluster * 32) * 32;
    const uint32_t k_end = min(p.dim, (member + 1) * k_slice);
    const int t0 = token[g], t1 = token[g + 8];
    float acc[RT][4] = {};
    for (uint32_t k = member * k_slice + warp * 32; k < k_end; k += kWarps * 32) {
      const int at = (int)k + (int)c * 8, valid = (int)p.dim - at;
      uint32_t r0[4] = {}, r1[4] = {};
      if (t0 >= 0 && valid > 0) load_words<4, VECTOR>(r0, x + (long long)t0 * p.x_stride + at, valid);
      if (t1 >= 0 && valid > 0) load_words<4, VECTOR>(r1, x + (long long)t1 * p.x_stride + at, valid);
      const uint32_t a0[4] = {r0[0], r1[0], r0[1], r1[1]}, a1[4] = {r0[2], r1[2], r0[3], r1[3]};
#pragma unroll
      for (int r = 0; r < RT; r++) {
        uint32_t b[4] = {};
        const uint32_t rank = r * 8 + g;
        if (rank < p.rank && valid > 0) load_words<4, VECTOR>(b, down + (size_t)rank * p.dim + at, valid);
        Half<E>::mma(acc[r], a0, b[0], b[1]);
        Half<E>::mma(acc[r], a1, b[2], b[3]);
      }
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      *reinterpret_cast<float2*>(&part[warp][g][r * 8 + c * 2]) = make_float2(acc[r][0], acc[r][1]);
      *reinterpret_cast<float2*>(&part[warp][g + 8][r * 8 + c * 2]) = make_float2(acc[r][2], acc[r][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * RP; i += kBlock) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) sum += (&part[w][0][0])[i];
      (&part[0][0][0])[i] = sum;
    }
  }
  cluster.sync();
  // the CTAs' sums, in their order; scaled to the row's largest so that both 16-bit terms keep their bits
  {
    const float scale = p.scale ? p.scale[tile.group] : 1.f;
    for (int i = threadIdx.x; i < kTile * RP; i += kBlock) {
      float sum = 0.f;
#pragma unroll
      for (int m = 0; m < kCluster; m++) sum += cluster.map_shared_rank(&part[0][0][0], m)[i];
      (&part[1][0][0])[i] = sum * scale;
    }
    __syncthreads();
    for (int m = warp; m < kTile; m += kWarps) {
      float top = 0.f;
      for (int r = lane; r < RP; r += 32) top = fmaxf(top, fabsf(part[1][m][r]));
#pragma unroll
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
      const float s = unit_scale(top);
      if (lane == 0) back[m] = 1.f / s;
      for (int r = lane * 2; r < KR; r += 64) {
        const float u0 = r < RP ? part[1][m][r] * s : 0.f, u1 = r < RP ? part[1][m][r + 1] * s : 0.f;
        const uint32_t hi = Half<E>::narrow(u0, u1);
        const float2 h = Half<E>::widen(hi);
        // what the first term leaves; nothing where the first is infinite
        const uint32_t lo = Half<E>::narrow(isinf(h.x) ? 0.f : u0 - h.x, isinf(h.y) ? 0.f : u1 - h.y);
        *reinterpret_cast<uint32_t*>(&inner[0][m][r]) = hi;
        *reinterpret_cast<uint32_t*>(&inner[1][m][r]) = lo;
      }
    }
  }
  cluster.sync();  // also: nobody leaves while its sums are being read

  // second product: every CTA a slice of out_dim, its warps 32 of it at a time.  Column 2c + b of the
  // q-th of four matrix tiles is output 8c + 2q + b, so that a lane ends with 8 consecutive outputs.
  {
    const uint16_t* up = static_cast<const uint16_t*>(p.up) + (long long)tile.group * p.up_stride;
    constexpr int KS = KR >= 32 ? KR / 32 : 1;   // steps of 32 (16) ranks
    constexpr int W = KR >= 32 ? 4 : 2;          // words a lane has of one
    uint32_t u[2][2][KS][W];                     // term, half of the tile
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int o = 0; o < 2; o++)
#pragma unroll
        for (int s = 0; s < KS; s++)
          load_words<W, true>(u[h][o][s], &inner[h][g + 8 * o][(s * 4 + c) * 2 * W], 2 * W);
    for (uint32_t n0 = n_begin + warp * 32; n0 < n_end; n0 += kWarps * 32) {
      float acc[4][4] = {};
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const uint32_t n = n0 + (g >> 1) * 8 + q * 2 + (g & 1);
#pragma unroll
        for (int s = 0; s < KS; s++) {
          uint32_t b[W] = {};
          const int at = (s * 4 + (int)c) * 2 * W, valid = (int)p.rank - at;
          if (n < n_end && valid > 0) load_words<W, VECTOR>(b, up + (size_t)n * p.rank + at, valid);
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int w = 0; w < W; w += 2) {
              const uint32_t a[4] = {u[h][0][s][w], u[h][1][s][w], u[h][0][s][w + 1], u[h][1][s][w + 1]};
              Half<E>::mma(acc[q], a, b[w], b[w + 1]);
            }
        }
      }
      const int at = (int)(n0 + c * 8), valid = (int)n_end - at;
#pragma unroll
      for (int o = 0; o < 2; o++) {
        const int t = token[g + 8 * o];
        if (t < 0 || valid <= 0) continue;
        uint32_t in[4];
        load_words<4, VECTOR>(in, base + (long long)t * p.base_stride + at, valid);
        const float s = back[g + 8 * o];
        uint32_t y[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const float2 v = Half<E>::widen(in[q]);
          y[q] = Half<E>::narrow(fmaf(acc[q][2 * o], s, v.x), fmaf(acc[q][2 * o + 1], s, v.y));
        }
        uint16_t* to = out + (long long)t * p.out_stride + at;
        if (VECTOR && valid >= 8) {
          *reinterpret_cast<uint4*>(to) = make_uint4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (i < valid) to[i] = (uint16_t)(y[i / 2] >> (i & 1 ? 16 : 0));
        }
      }
    }
  }
}

template <typename E, int RP>
cudaError_t adapter_launch(const AdapterParams& p, bool vector, cudaStream_t stream) {
  auto kern = vector ? adapter_kernel<E, RP, true> : adapter_kernel<E, RP, false>;
  constexpr size_t smem = kWarps * kTile * RP * sizeof(float) + 2 * kTile * (std::max(RP, 16) + 8) * sizeof(uint16_t);
  if (smem > 47 * 1024) {  // beside what is static
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  const uint32_t tiles = p.n_tokens / kTile + std::min(p.n_groups + 1, p.n_tokens);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * kCluster);
  cfg.blockDim = dim3(kBlock);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {kCluster, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

cudaError_t launch_adapter_add(const AdapterParams& p, int elem, cudaStream_t stream) {
  if (p.n_tokens == 0) return cudaSuccess;
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(p.base) | reinterpret_cast<uintptr_t>(p.x) |
                              reinterpret_cast<uintptr_t>(p.down) | reinterpret_cast<uintptr_t>(p.up) |
                              reinterpret_cast<uintptr_t>(p.out);
  const unsigned long long strides = (unsigned long long)p.base_stride | p.x_stride | p.down_stride | p.up_stride | p.out_stride;
  const bool vector = addresses % 16 == 0 && strides % 8 == 0 && p.dim % 8 == 0 && p.out_dim % 8 == 0 && p.rank % 8 == 0;
  auto by_rank = [&](auto e) {
    using E = decltype(e);
    if (p.rank <= 8) return adapter_launch<E, 8>(p, vector, stream);
    if (p.rank <= 16) return adapter_launch<E, 16>(p, vector, stream);
    if (p.rank <= 32) return adapter_launch<E, 32>(p, vector, stream);
    if (p.rank <= 64) return adapter_launch<E, 64>(p, vector, stream);
    return adapter_launch<E, 128>(p, vector, stream);
  };
  return elem == kElemF16 ? by_rank(__half{}) : by_rank(__nv_bfloat16{});
}

}  // namespace ugc
