// A whole routed layer for a few tokens: out[t] = sum over j of w[t, j] silu(x[t] up[e]) down[e], e the j-th expert that token t chose.  Its work is
// reading the weights of the experts that were chosen, each of them once, with all SMs.
//
//   logits   a warp has an expert's row of the router and all tokens
//   choice   egs_choice.cu's kernel
//   up       units of (an expert's up to four tokens) x (a tile of columns) x (a part of the contraction) go round the CTAs; float32 sums of parts
//   down     a cluster has a tile of the output's columns, its CTAs the contraction in parts; warps have the experts' tokens in turn.  The parts' sums
//            are joined, activated and weighted on the way into shared memory; a token's products are added in the order of its choices, the
//            CTAs' in theirs: the same bits in every run.
#include "egs_fp4.cuh"

namespace egs {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kMost = EGS_MAX_FEW_SLOTS, kRows = 4;      // slots; tokens that share a read of the weights
constexpr int kUpThreads = 256, kUpWarps = kUpThreads / 32, kUpGrid = 296, kUpPart = 1024;
constexpr int kDownThreads = 512, kDownWarps = kDownThreads / 32;
constexpr int kMostParts = 8;

struct LayerParams {
  const void* X;
  const void* router;
  const void* up;            // [E, I, J], in 4 bits [E, J, I / 2]
  const void* down;          // [E, J, I], in 4 bits [E, I, J / 2]
  const uint8_t* up_scale;
  const uint8_t* down_scale;
  void* out;
  float* weights;
  int* experts;
  float* logits;
  float* h;                  // [parts][tokens * k][J]
  long long x_row, up_row, us_row, down_row, ds_row;       // elements; in 4 bits bytes
  int tokens, E, k, I, J;
  int act_floats;            // down: room for activations
};

// An expert's tokens, up to four at a time.
struct Item {
  int expert, rows;
  short slot[kRows];
};
struct Items {
  Item item[kMost];
  int ids[kMost];
  unsigned tokens[EGS_MAX_EXPERTS];
  int count;
};
// From the chosen experts; by all threads.
__device__ __forceinline__ void list_items(const LayerParams& p, Items* s) {
  const int tid = threadIdx.x, n = p.tokens * p.k;
  for (int e = tid; e < p.E; e += blockDim.x) s->tokens[e] = 0u;
  __syncthreads();
  for (int i = tid; i < n; i += blockDim.x) {
    const int e = p.experts[i];
    s->ids[i] = e;
    atomicOr(&s->tokens[e], 1u << (i / p.k));
  }
  __syncthreads();
  if (tid < 32) {
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + tid;
      unsigned mask = e < p.E ? s->tokens[e] : 0u;
      const int own = (__popc(mask) + kRows - 1) / kRows;
      int at = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kAll, at, o);
        if (tid >= o) at += v;
      }
      const int total = __shfl_sync(kAll, at, 31);
      at += before - own;
      before += total;
      for (int i = 0; i < own; ++i) {
        Item& x = s->item[at + i];
        x.expert = e;
        x.rows = min(kRows, __popc(mask));
        for (int r = 0; r < x.rows; ++r) {
          const int t = __ffs(mask) - 1;
          mask &= mask - 1;
          int j = 0;
          while (j < p.k - 1 && s->ids[t * p.k + j] != e) ++j;
          x.slot[r] = static_cast<short>(t * p.k + j);
        }
        for (int r = x.rows; r < kRows; ++r) x.slot[r] = x.slot[0];
      }
    }
    if (tid == 0) s->count = before;
  }
  __syncthreads();
}

// Parts that the contraction of `up` is cut into: the fewest rounds of the CTAs, a unit costing as much as 128 rows beside its own.
__device__ __forceinline__ int parts_of(int units, int length) {
  int best = 1, least = 0x7fffffff;
  for (int s = 1; s <= kMostParts && (s == 1 || length / s >= 64); s *= 2) {
    const int cost = (units * s + kUpGrid - 1) / kUpGrid * ((length + s - 1) / s + 128);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

// ---- logits ---------------------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(256) few_logits_kernel(const __grid_constant__ LayerParams p) {
  using P = Packed<T, V>;
  pdl_wait();
  pdl_trigger();
  const int e = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, t0 = blockIdx.y * kRows;
  if (e >= p.E) return;
  const T* w = static_cast<const T*>(p.router) + static_cast<long long>(e) * p.I;
  const T* x[kRows];
  float acc[kRows];
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    x[m] = static_cast<const T*>(p.X) + min(t0 + m, p.tokens - 1) * p.x_row;
    acc[m] = 0.f;
  }
#pragma unroll 4
  for (int i = lane; i < p.I / V; i += 32) {
    const P a = reinterpret_cast<const P*>(w)[i];
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      const P b = reinterpret_cast<const P*>(x[m])[i];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[m] = fmaf(a.get(v), b.get(v), acc[m]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int m = 0; m < kRows; ++m) acc[m] += __shfl_xor_sync(kAll, acc[m], o);
#pragma unroll
  for (int m = 0; m < kRows; ++m)
    if (lane == m && t0 + m < p.tokens) p.logits[(t0 + m) * p.E + e] = acc[m];
}

// ---- products along rows of the weights ([contraction, columns]) -----------------------------------------------------
// A group of lanes has four neighbouring rows at a time, every `step`-th such four from c on; a[m] + c - base: the other operand, zeros up to whole
// fours.  `ready` is called when the first weights have been asked for.
template <typename T, int V, int M, int AHEAD, class Ready>
__device__ __forceinline__ void accumulate(float (&acc)[M][V], const T* W, long long w_row, int c, int step, int end, bool on, const float* const (&a)[M], int base, Ready&& ready) {
  using P = Packed<T, V>;
  P w[AHEAD][4];
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = c + i * step + r;
        w[i][r] = on && row < end ? *reinterpret_cast<const P*>(W + row * w_row) : P{};
      }
  };
  load();
  ready();
  while (c < end) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (c + i * step >= end) break;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float4 x = *reinterpret_cast<const float4*>(a[m] + c + i * step - base);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          acc[m][v] = fmaf(x.x, w[i][0].get(v), acc[m][v]);
          acc[m][v] = fmaf(x.y, w[i][1].get(v), acc[m][v]);
          acc[m][v] = fmaf(x.z, w[i][2].get(v), acc[m][v]);
          acc[m][v] = fmaf(x.w, w[i][3].get(v), acc[m][v]);
        }
      }
    }
    c += AHEAD * step;
    if (c < end) load();
  }
}
template <int LANES, int V, int M>
__device__ __forceinline__ void join_groups(float (&acc)[M][V]) {
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[m][v] += __shfl_xor_sync(kAll, acc[m][v], o);
}
__host__ __device__ constexpr int ahead_of(int V) { return V >= 4 ? 2 : 4; }

template <typename T, int V, int LANES>
struct UpShared {
  Items items;
  alignas(16) float x[kRows][kUpPart];
  float sums[kUpWarps][kRows][LANES * V];
};

template <typename T, int V, int LANES, int M>
__device__ __forceinline__ void up_unit(const LayerParams& p, UpShared<T, V, LANES>* s, const Item& item, int n0, int begin, int end, float* to) {
  constexpr int kGroups = kUpThreads / LANES, kTile = LANES * V;
  const int tid = threadIdx.x, l = tid % LANES, n = n0 + l * V;
  const T* W = static_cast<const T*>(p.up) + item.expert * (p.up_row * p.I) + n;
  float acc[M][V];
  const float* a[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    a[m] = s->x[m];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[m][v] = 0.f;
  }
  for (int c0 = begin; c0 < end; c0 += kUpPart) {
    const int c1 = min(end, c0 + kUpPart);
    accumulate<T, V, M, ahead_of(V)>(acc, W, p.up_row, c0 + tid / LANES * 4, kGroups * 4, c1, n < p.J, a, c0, [&]() {
      __syncthreads();                         // what was in shared memory has been read
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const T* x = static_cast<const T*>(p.X) + item.slot[m] / p.k * p.x_row;
        for (int i = tid; i < ((c1 - c0 + 3) & ~3); i += kUpThreads) s->x[m][i] = c0 + i < c1 ? to_f32<T>(x[c0 + i]) : 0.f;
      }
      __syncthreads();
    });
  }
  join_groups<LANES, V, M>(acc);
  if ((tid & 31) < LANES) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int v = 0; v < V; ++v) s->sums[tid >> 5][m][l * V + v] = acc[m][v];
  }
  __syncthreads();
  for (int i = tid; i < M * kTile; i += kUpThreads) {
    const int m = i / kTile, col = i % kTile;
    if (m >= item.rows || n0 + col >= p.J) continue;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kUpWarps; ++w) t += s->sums[w][m][col];
    to[static_cast<long long>(item.slot[m]) * p.J + n0 + col] = t;
  }
}

template <typename T, int V, int LANES>
__global__ void __launch_bounds__(kUpThreads, 2) few_up_kernel(const __grid_constant__ LayerParams p) {
  constexpr int kTile = LANES * V;
  __shared__ UpShared<T, V, LANES> s;
  pdl_wait();
  pdl_trigger();
  list_items(p, &s.items);
  const int tiles = (p.J + kTile - 1) / kTile, all = s.items.count * tiles, parts = parts_of(all, p.I), length = ((p.I + parts - 1) / parts + 3) & ~3;
  for (int u = blockIdx.x; u < all * parts; u += gridDim.x) {
    const int part = u / all, x = u - part * all, i = x / tiles, n0 = (x - i * tiles) * kTile, begin = min(p.I, part * length), end = min(p.I, begin + length);
    const Item item = s.items.item[i];
    float* to = p.h + static_cast<long long>(part) * p.tokens * p.k * p.J;
    if (item.rows == 1) up_unit<T, V, LANES, 1>(p, &s, item, n0, begin, end, to);
    else up_unit<T, V, LANES, kRows>(p, &s, item, n0, begin, end, to);
  }
}

// Sum of a slot's parts, activated.
__device__ __forceinline__ float activation(const LayerParams& p, int parts, long long at) {
  float v = p.h[at];
  for (int s = 1; s < parts; ++s) v += p.h[at + static_cast<long long>(s) * p.tokens * p.k * p.J];
  return v / (1.f + expf(-v));
}

__device__ __forceinline__ int cluster_rank() {
  int r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ int cluster_size() {
  int r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float of_cta(const float* mine, int rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// out[t, n0 + n] from the slots' products: part [shares][slots][tile]; `sums` [tokens][tile] of shared memory
template <typename T>
__device__ __forceinline__ void put_out(const LayerParams& p, const float* part, float* sums, int shares, int tile, int n0) {
  const int slots = p.tokens * p.k, rank = cluster_rank(), size = cluster_size();
  for (int i = threadIdx.x; i < p.tokens * tile; i += kDownThreads) {
    const int t = i / tile, n = i - t * tile;
    float v = 0.f;
    for (int j = 0; j < p.k; ++j)
      for (int s = 0; s < shares; ++s) v += part[(s * slots + t * p.k + j) * tile + n];
    sums[i] = v;
  }
  cluster_sync();
  for (int i = threadIdx.x + rank * kDownThreads; i < p.tokens * tile; i += kDownThreads * size) {
    const int t = i / tile, n = i - t * tile;
    float v = of_cta(sums + i, 0);
    for (int r = 1; r < size; ++r) v += of_cta(sums + i, r);
    if (n0 + n < p.I) static_cast<T*>(p.out)[static_cast<long long>(t) * p.I + n0 + n] = from_f32<T>(v);
  }
  cluster_sync();
}

template <typename T, int V, int LANES, int M>
__device__ __forceinline__ void down_item(const LayerParams& p, const Item& item, const float* act, int pitch, int base, int begin, int end, int n0, float* part, bool first) {
  constexpr int kTile = LANES * V;
  const int lane = threadIdx.x & 31, l = lane % LANES, n = n0 + l * V;
  float acc[M][V];
  const float* a[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    a[m] = act + item.slot[m] * pitch;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[m][v] = 0.f;
  }
  accumulate<T, V, M, ahead_of(V)>(acc, static_cast<const T*>(p.down) + item.expert * (p.down_row * p.J) + n, p.down_row, begin + lane / LANES * 4, 32 / LANES * 4, end, n < p.I, a, base, []() {});
  join_groups<LANES, V, M>(acc);
  if (lane < LANES) {
#pragma unroll
    for (int m = 0; m < M; ++m)
      if (m < item.rows) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float* to = part + item.slot[m] * kTile + l * V + v;
          *to = first ? acc[m][v] : *to + acc[m][v];
        }
      }
  }
}

template <typename T, int V, int LANES>
__global__ void __launch_bounds__(kDownThreads, 1) few_down_kernel(const __grid_constant__ LayerParams p) {
  constexpr int kTile = LANES * V;
  extern __shared__ __align__(16) float layer_smem[];
  __shared__ Items items;
  pdl_wait();
  pdl_trigger();
  list_items(p, &items);
  const int slots = p.tokens * p.k, rank = cluster_rank(), size = cluster_size(), tid = threadIdx.x, warp = tid >> 5;
  const int n0 = blockIdx.x / size * kTile;
  float* act = layer_smem;
  float* part = layer_smem + p.act_floats;
  const int up_tiles = (p.J + kTile - 1) / kTile, parts = parts_of(items.count * up_tiles, p.I);
  const int length = ((p.J + size - 1) / size + 3) & ~3, begin = min(p.J, rank * length), end = min(p.J, begin + length);
  const int room = min(length, p.act_floats / slots & ~3);
  int shares = 1;                              // warps that have an item's contraction in turn
  while (items.count * shares * 2 <= kDownWarps && length / shares >= 64) shares *= 2;
  for (int c0 = begin; c0 == begin || c0 < end; c0 += room) {
    const int c1 = min(end, c0 + room), width = (c1 - c0 + 3) & ~3;
    __syncthreads();
    for (int slot = warp; slot < slots; slot += kDownWarps) {
      const float w = p.weights[slot];
      for (int i = tid & 31; i < width; i += 32) act[slot * room + i] = c0 + i < c1 ? w * activation(p, parts, static_cast<long long>(slot) * p.J + c0 + i) : 0.f;
    }
    __syncthreads();
    const int each = (width / 4 + shares - 1) / shares * 4;
    for (int x = warp; x < items.count * shares; x += kDownWarps) {
      const int i = x / shares, share = x - i * shares, b = min(c1, c0 + share * each), e = min(c1, b + each);
      const Item item = items.item[i];
      float* to = part + share * slots * kTile;
      if (item.rows == 1) down_item<T, V, LANES, 1>(p, item, act, room, c0, b, e, n0, to, c0 == begin);
      else down_item<T, V, LANES, kRows>(p, item, act, room, c0, b, e, n0, to, c0 == begin);
    }
  }
  __syncthreads();
  put_out<T>(p, part, act, shares, kTile, n0);
}

// ---- products along the contraction, weights in 4 bits ([columns, contraction]) ---------------------------------------
constexpr int kChannels = 8;                   // columns of a warp
constexpr int kTile4 = 64;

// Eight columns of an expert from n0 on times M rows, blocks [begin, end): a[m] + b * 32: twice the rows' 4 bits as bytes, f[m] + b: their scales.  Lanes
// go along the blocks, 4 to 32 of them; those that are left have other columns.  emit(column, row, sum) for the lanes that have the sums.
template <int M, class Emit>
__device__ __forceinline__ void columns4(const uint8_t* W, long long w_row, const uint8_t* S, long long s_row, int C, int N, int n0, int begin, int end, const uint8_t* const (&a)[M],
                                         const float* const (&f)[M], int base, Emit&& emit) {
  const int lane = threadIdx.x & 31;
  int lanes_log2 = 2;
  while (lanes_log2 < 5 && (1 << lanes_log2) < end - begin) ++lanes_log2;
  const int along = lane & ((1 << lanes_log2) - 1), group = lane >> lanes_log2, groups = 32 >> lanes_log2;
  constexpr int kAtOnce = 2;
  for (int j0 = 0; j0 < kChannels / groups; j0 += kAtOnce) {
    float acc[kAtOnce][M];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
      for (int m = 0; m < M; ++m) acc[j][m] = 0.f;
#pragma unroll 2
    for (int b = begin + along; b < end; b += 1 << lanes_log2) {
      Block4 w[kAtOnce];
      uint32_t s[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const long long n = min(n0 + (j0 + j) * groups + group, N - 1);
        w[j] = load_block(W + n * w_row, b, C);
        s[j] = S[n * s_row + b];
      }
      uint32_t x[M][8];
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 y = *reinterpret_cast<const uint4*>(a[m] + (b - base) * 32 + i * 16);
          x[m][4 * i] = y.x; x[m][4 * i + 1] = y.y; x[m][4 * i + 2] = y.z; x[m][4 * i + 3] = y.w;
        }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        int sum[M];
#pragma unroll
        for (int m = 0; m < M; ++m) sum[m] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t low, high;
          fp4_integers(w[j].w[i], low, high);
#pragma unroll
          for (int m = 0; m < M; ++m) sum[m] = __dp4a(static_cast<int>(x[m][2 * i + 1]), static_cast<int>(high), __dp4a(static_cast<int>(x[m][2 * i]), static_cast<int>(low), sum[m]));
        }
        const float power = fp4_power(s[j]);
#pragma unroll
        for (int m = 0; m < M; ++m) acc[j][m] = fmaf(static_cast<float>(sum[m]) * f[m][b - base], power, acc[j][m]);
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
      for (int m = 0; m < M; ++m)
        for (int o = 1; o < 1 << lanes_log2; o <<= 1) acc[j][m] += __shfl_xor_sync(kAll, acc[j][m], o);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int c = (j0 + j) * groups + group;
      if (j0 + j < kChannels / groups && along == 0 && n0 + c < N) {
#pragma unroll
        for (int m = 0; m < M; ++m) emit(n0 + c, m, acc[j][m]);
      }
    }
  }
}

// A block of 32 values in 4 bits, as twice their values in bytes; a quarter of its scale.
__device__ __forceinline__ float block4(float (&v)[32], uint8_t* to) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  const uint32_t byte = fp4_scale(top);
  const float inverse = fp4_inverse(byte);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fp4_scaled(v[8 * i + j], inverse);
    uint2 w;
    fp4_integers(fp4_pack8(x), w.x, w.y);
    *reinterpret_cast<uint2*>(to + 8 * i) = w;
  }
  return 0.25f * fp4_power(byte);
}

struct Up4Shared {
  Items items;
  alignas(16) uint8_t x[kRows][2 * kUpPart];
  float f[kRows][2 * kUpPart / kFp4Block];
};

template <typename T, int M>
__device__ __forceinline__ void up4_unit(const LayerParams& p, Up4Shared* s, const Item& item, int n0, int begin, int end, float* to) {
  const int tid = threadIdx.x;
  const uint8_t* a[M];
  const float* f[M];
  const T* x[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    a[m] = s->x[m];
    f[m] = s->f[m];
    x[m] = static_cast<const T*>(p.X) + item.slot[m] / p.k * p.x_row;
  }
  const int C = (p.I + 1) / 2 * 2, chunk = 2 * kUpPart / kFp4Block;
  for (int b0 = begin; b0 < end; b0 += chunk) {
    const int b1 = min(end, b0 + chunk), n = b1 - b0;
    __syncthreads();
    for (int i = tid; i < M * n; i += kUpThreads) {
      const int m = i / n, b = b0 + i - m * n;
      float v[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = b * 32 + c < p.I ? to_f32<T>(x[m][b * 32 + c]) : 0.f;
      s->f[m][b - b0] = block4(v, s->x[m] + (b - b0) * 32);
    }
    __syncthreads();
    const bool first = b0 == begin;
    columns4<M>(static_cast<const uint8_t*>(p.up) + item.expert * (p.up_row * p.J), p.up_row, p.up_scale + item.expert * (p.us_row * p.J), p.us_row, C, p.J,
                n0 + (tid >> 5) * kChannels, b0, b1, a, f, b0, [&](int col, int m, float v) {
                  if (m >= item.rows) return;
                  float* o = to + static_cast<long long>(item.slot[m]) * p.J + col;
                  *o = first ? v : *o + v;
                });
  }
}

template <typename T>
__global__ void __launch_bounds__(kUpThreads, 2) few_up4_kernel(const __grid_constant__ LayerParams p) {
  __shared__ Up4Shared s;
  pdl_wait();
  pdl_trigger();
  list_items(p, &s.items);
  const int tiles = (p.J + kTile4 - 1) / kTile4, all = s.items.count * tiles, parts = parts_of(all, p.I), blocks = fp4_blocks(p.I), length = (blocks + parts - 1) / parts;
  for (int u = blockIdx.x; u < all * parts; u += gridDim.x) {
    const int part = u / all, x = u - part * all, i = x / tiles, n0 = (x - i * tiles) * kTile4, begin = min(blocks, part * length), end = min(blocks, begin + length);
    const Item item = s.items.item[i];
    float* to = p.h + static_cast<long long>(part) * p.tokens * p.k * p.J;
    if (begin == end) {                        // (nothing is left for the last parts of a short contraction)
      for (int c = threadIdx.x; c < item.rows * kTile4; c += kUpThreads)
        if (n0 + c % kTile4 < p.J) to[static_cast<long long>(item.slot[c / kTile4]) * p.J + n0 + c % kTile4] = 0.f;
    } else if (item.rows == 1) {
      up4_unit<T, 1>(p, &s, item, n0, begin, end, to);
    } else {
      up4_unit<T, kRows>(p, &s, item, n0, begin, end, to);
    }
  }
}

template <int M>
__device__ __forceinline__ void down4_item(const LayerParams& p, const Item& item, const uint8_t* act, const float* scale, int pitch, int b0, int b1, int n0, int base_n, float* part, bool first) {
  const uint8_t* a[M];
  const float* f[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    a[m] = act + item.slot[m] * pitch * 32;
    f[m] = scale + item.slot[m] * pitch;
  }
  columns4<M>(static_cast<const uint8_t*>(p.down) + item.expert * (p.down_row * p.I), p.down_row, p.down_scale + item.expert * (p.ds_row * p.I), p.ds_row, (p.J + 1) / 2 * 2, p.I, n0, b0, b1, a, f,
              b0, [&](int col, int m, float v) {
                if (m >= item.rows) return;
                float* o = part + item.slot[m] * kTile4 + col - base_n;
                *o = first ? v : *o + v;
              });
}

template <typename T>
__global__ void __launch_bounds__(kDownThreads, 1) few_down4_kernel(const __grid_constant__ LayerParams p) {
  extern __shared__ __align__(16) float layer_smem[];
  __shared__ Items items;
  pdl_wait();
  pdl_trigger();
  list_items(p, &items);
  const int slots = p.tokens * p.k, rank = cluster_rank(), size = cluster_size(), tid = threadIdx.x, warp = tid >> 5;
  const int n0 = blockIdx.x / size * kTile4;
  float* part = layer_smem + p.act_floats;
  const int up_tiles = (p.J + kTile4 - 1) / kTile4, parts = parts_of(items.count * up_tiles, p.I), blocks = fp4_blocks(p.J);
  const int length = (blocks + size - 1) / size, begin = min(blocks, rank * length), end = min(blocks, begin + length);
  const int room = min(length, p.act_floats / (9 * slots));            // blocks: eight words of bytes and a scale
  uint8_t* act = reinterpret_cast<uint8_t*>(layer_smem);
  float* scale = layer_smem + static_cast<long long>(slots) * room * 8;
  for (int b0 = begin; b0 == begin || b0 < end; b0 += room) {
    const int b1 = min(end, b0 + room), n = b1 - b0;
    __syncthreads();
    for (int i = tid; i < slots * n; i += kDownThreads) {
      const int slot = i / n, b = b0 + i - slot * n;
      float v[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = b * 32 + c < p.J ? activation(p, parts, static_cast<long long>(slot) * p.J + b * 32 + c) : 0.f;
      scale[slot * room + b - b0] = p.weights[slot] * block4(v, act + (slot * room + b - b0) * 32);
    }
    __syncthreads();
    constexpr int kSets = kTile4 / kChannels;
    for (int x = warp; x < items.count * kSets; x += kDownWarps) {
      const Item item = items.item[x / kSets];
      const int first_n = n0 + x % kSets * kChannels;
      if (item.rows == 1) down4_item<1>(p, item, act, scale, room, b0, b1, first_n, n0, part, b0 == begin);
      else down4_item<kRows>(p, item, act, scale, room, b0, b1, first_n, n0, part, b0 == begin);
    }
  }
  __syncthreads();
  put_out<T>(p, part, layer_smem, 1, kTile4, n0);
}

// ---- launches ----------------------------------------------------------------------------------------------------------
constexpr size_t kDownSmem = 200 * 1024;

template <class... Params, class... Args>
cudaError_t launch_cluster(void (*kernel)(Params...), unsigned grid, unsigned block, unsigned cluster, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// CTAs of a cluster: as many as leave a CTA for every SM at most, each with 32 contraction elements at least.
unsigned cluster_of(int tiles, int J) {
  unsigned size = 8;
  while (size > 1 && (tiles * static_cast<int>(size) > 148 || J / static_cast<int>(size) < 32)) size /= 2;
  return size;
}

template <auto kernel, typename T>
cudaError_t down_launch(LayerParams p, int tile, cudaStream_t st) {
  const int tiles = (p.I + tile - 1) / tile, slots = p.tokens * p.k;
  cudaError_t err = ensure_smem_optin<kernel>(static_cast<int>(kDownSmem));
  if (err != cudaSuccess) return err;
  const size_t part = static_cast<size_t>(slots < 4 * kDownWarps ? 4 * kDownWarps : slots) * tile * sizeof(float);
  const unsigned size = cluster_of(tiles, p.J);
  size_t act = static_cast<size_t>(slots) * (p.J / size + 36) * sizeof(float);
  if (act < static_cast<size_t>(p.tokens) * tile * sizeof(float)) act = static_cast<size_t>(p.tokens) * tile * sizeof(float);
  act = (act + 15) & ~static_cast<size_t>(15);
  if (act > kDownSmem - part) act = kDownSmem - part;
  p.act_floats = static_cast<int>(act / sizeof(float));
  count_launch();
  return launch_cluster(kernel, tiles * size, kDownThreads, size, act + part, st, p);
}

bool on(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T>
cudaError_t layer_t(const LayerParams& p, bool fp4, const egs_route& r, const float* bias, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T), kLanes = 8;
  const dim3 grid((p.E + 7) / 8, (p.tokens + kRows - 1) / kRows);
  const bool vectors = p.I % V == 0 && p.x_row % V == 0 && on(p.X, 16) && on(p.router, 16);
  count_launch();
  cudaError_t err = vectors ? launch_kernel(few_logits_kernel<T, V>, grid, 256, 0, st, true, p) : launch_kernel(few_logits_kernel<T, 1>, grid, 256, 0, st, true, p);
  if (err != cudaSuccess) return err;
  if ((err = launch_route_tokens(p.logits, bias, p.weights, p.experts, r, p.E, EGS_F32, st)) != cudaSuccess) return err;
  count_launch();
  if (fp4) {
    if ((err = launch_kernel(few_up4_kernel<T>, kUpGrid, kUpThreads, 0, st, true, p)) != cudaSuccess) return err;
    return down_launch<few_down4_kernel<T>, T>(p, kTile4, st);
  }
  // (one width for both: the parts of `up` are counted by it)
  const bool wide = p.I % V == 0 && p.J % V == 0 && on(p.up, 16) && on(p.down, 16);
  if (wide) {
    if ((err = launch_kernel(few_up_kernel<T, V, kLanes>, kUpGrid, kUpThreads, 0, st, true, p)) != cudaSuccess) return err;
    return down_launch<few_down_kernel<T, V, kLanes>, T>(p, V * kLanes, st);
  }
  if ((err = launch_kernel(few_up_kernel<T, 1, 32>, kUpGrid, kUpThreads, 0, st, true, p)) != cudaSuccess) return err;
  return down_launch<few_down_kernel<T, 1, 32>, T>(p, 32, st);
}

}  // namespace

size_t few_layer_workspace(const egs_route& r, long long J) {
  const size_t logits = (static_cast<size_t>(r.tokens) * r.E + 3) / 4 * 4;
  return (logits + static_cast<size_t>(kMostParts) * r.tokens * r.top_k * J) * sizeof(float);
}

cudaError_t launch_few_layer(const FewLayer& f, const egs_route& r, int dtype, void* workspace, cudaStream_t st) {
  LayerParams p{};
  p.X = f.X; p.router = f.router; p.up = f.up; p.down = f.down; p.up_scale = f.up_scale; p.down_scale = f.down_scale;
  p.out = f.out; p.weights = f.weights; p.experts = f.experts;
  p.logits = static_cast<float*>(workspace);
  p.h = p.logits + (static_cast<size_t>(r.tokens) * r.E + 3) / 4 * 4;
  p.x_row = f.x_row;
  p.tokens = static_cast<int>(r.tokens); p.E = r.E; p.k = r.top_k; p.I = f.I; p.J = f.J;
  const bool fp4 = f.up_scale != nullptr;
  p.up_row = fp4 ? f.up_row : p.J; p.us_row = f.us_row; p.down_row = fp4 ? f.down_row : p.I; p.ds_row = f.ds_row;
  return dtype == EGS_F16 ? layer_t<__half>(p, fp4, r, f.bias, st) : dtype == EGS_BF16 ? layer_t<__nv_bfloat16>(p, fp4, r, f.bias, st) : layer_t<float>(p, fp4, r, f.bias, st);
}

}  // namespace egs
