// A whole routed layer for a few tokens: out[t] = sum over j of w[t, j] silu(x[t] up[e]) down[e], e the j-th expert that token t chose.  Its work is
// reading the weights of the experts that were chosen, each of them once, with all SMs.
//
//   choice   two kernels: the logits, a warp two experts' rows of the router and four tokens, and egs_choice.cu's.  (In one kernel with `up`, each CTA
//            choosing for itself, or in one with each other, by a cluster of eight CTAs or one, they took 0.5 to 6 us more.)
//   up       units of (an expert's up to four tokens) x (a tile of columns) x (a part of the contraction) go round
//            the CTAs; float32 sums of parts
//   down     a cluster has a tile of the output's columns, its CTAs the contraction in parts; warps have the experts' tokens in turn.  The parts' sums
//            are joined, activated and weighted on the way into shared memory; a token's products are added in the order of its choices, the
//            CTAs' in theirs: the same bits in every run.
//
// us a call in a graph, new weights each time: 1 token, 8 of 64 experts, 2048 x 512 bf16 (33.8 MB, 5.2 at the copy's rate) 17.2, of which logits 2, choice 2, `up` 4.2 and `down`
// 6.7 on the device, the rest between them; 16 tokens, 4 of 64, 1024 x 256 (43 MB) 26.0
// (28.2 with a last product that waited before it listed the items and asked for weights).  Products run at 4 to 5 TB/s once weights come; what is left is latency: four
// launches, the list, the first weights, the join of a cluster.  Tried: the other product's weights to the L2 ahead (no gain), 16-bit products on mma.sync (1 us more: float32 sums by
// packed FMA are not what bounds it), weights through registers (3.4 TB/s), rings of 2, 4 and 6 steps (equal, equal, slower), tiles of 128 columns (20 us -> 24.6).
#include "egs_fp4.cuh"

namespace egs {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kMost = EGS_MAX_FEW_SLOTS, kRows = 4;      // slots; tokens that share a read of the weights
constexpr int kUpThreads = 256, kUpWarps = kUpThreads / 32, kUpGrid = 296, kUpPart = 1024;
constexpr int kDownThreads = 512, kDownWarps = kDownThreads / 32;
constexpr int kMostParts = 8, kMostSplits = 4;
constexpr int kFixedRows = 128;              // of a unit, in rows of its tile: 16 KB of weights

struct Items;
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
  Items* list;               // in 4 bits: from `up`
  long long x_row, up_row, us_row, down_row, ds_row;       // elements; in 4 bits bytes
  long long up_far, down_far;      // in 4 bits: bytes from one expert to the next
  int tokens, E, k, I, J;
  int x_vectors;             // rows of X and of the router begin on 16 bytes and are whole 16 bytes
  long long weight_bytes;    // of all experts' matrices, of either product
  uint32_t up_first, down_first;   // shifted rows: `up` and `down` are the 16 bytes that the weights begin in, this many elements on
  int ring_words;            // of weights on their way, in shared memory
  int act_floats;            // down: room for activations
  int splits;                // ... clusters that a tile's contraction is cut into beside their CTAs
  float* sums;               // ... theirs, [splits][tokens][I], where there are several
  Div by_tiles, by_k, by_stages;
};

// An expert's tokens, up to four at a time.
struct alignas(16) Item {
  int expert, rows;
  short slot[kRows];
};
struct alignas(16) Items {
  Item item[kMost];
  int count;
};
// What is needed while they are listed.
struct Scratch {
  int ids[kMost];
  unsigned tokens[EGS_MAX_EXPERTS];
  int first[EGS_MAX_EXPERTS];    // an expert's first item
};
// From the chosen experts (w->ids); by all threads, which have synchronised behind the ids and w->tokens = 0.
__device__ __forceinline__ void list_chosen(const LayerParams& p, Items* s, Scratch* w) {
  const int tid = threadIdx.x, n = p.tokens * p.k;
  for (int i = tid; i < n; i += blockDim.x) atomicOr(&w->tokens[w->ids[i]], 1u << p.by_k.quotient(i));
  __syncthreads();
  if (tid < 32) {
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + tid, own = e < p.E ? (__popc(w->tokens[e]) + kRows - 1) / kRows : 0;
      int at = before;
#pragma unroll
      for (int bit = 0; bit < 4; ++bit) {        // (eight items at most)
        const unsigned has = __ballot_sync(kAll, own >> bit & 1);
        at += __popc(has & ((1u << tid) - 1u)) << bit;
        before += __popc(has) << bit;
      }
      if (e < p.E) w->first[e] = at;
    }
    if (tid == 0) s->count = before;
  }
  __syncthreads();
  for (int i = tid; i < n; i += blockDim.x) {
    const int e = w->ids[i];
    const unsigned tokens = w->tokens[e];
    const int place = __popc(tokens & ((1u << p.by_k.quotient(i)) - 1u)), rows = min(kRows, __popc(tokens) - place / kRows * kRows);
    Item& x = s->item[w->first[e] + place / kRows];
    x.slot[place % kRows] = static_cast<short>(i);
    if (place % kRows == 0) {
      x.expert = e;
      x.rows = rows;
      for (int r = rows; r < kRows; ++r) x.slot[r] = static_cast<short>(i);
    }
  }
  __syncthreads();
}

// The items of the choice; by all threads.
__device__ __forceinline__ void list_items(const LayerParams& p, Items* s, Scratch* w) {
  if (p.tokens == 1) {                         // its experts differ
    const int i = threadIdx.x;
    if (i < p.k) {
      Item x{__ldcg(p.experts + i), 1};
#pragma unroll
      for (int r = 0; r < kRows; ++r) x.slot[r] = static_cast<short>(i);
      s->item[i] = x;
    }
    if (i == 0) s->count = p.k;
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) w->tokens[e] = 0u;
  for (int i = threadIdx.x; i < p.tokens * p.k; i += blockDim.x) w->ids[i] = __ldcg(p.experts + i);
  __syncthreads();
  list_chosen(p, s, w);
}

// Parts that the contraction of `up` is cut into: the fewest rounds of the CTAs, a unit costing as much as kFixedRows beside its own.
__device__ __forceinline__ int parts_of(int units, int length) {
  int best = 1, least = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = 1 << i, cost = (units * s + kUpGrid - 1) / kUpGrid * (((length + s - 1) >> i) + kFixedRows);
    if (cost < least && (i == 0 || length >> i >= 64)) {
      least = cost;
      best = s;
    }
  }
  return best;
}

// ---- clusters -----------------------------------------------------------------------------------------------------------
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
__device__ __forceinline__ uint32_t in_cta(const void* mine, int rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
  return at;
}
// Dot products of two experts' rows of the router with M tokens' rows from t0 on (the last ones' for those that are not there); all lanes have them.  Loads
// of AHEAD steps go out together.
template <typename T, int V, int M, int AHEAD>
__device__ __forceinline__ void dots(const LayerParams& p, int e0, int e1, int t0, float (&acc)[2][M]) {
  using P = Packed<T, V>;
  const int lane = threadIdx.x & 31, n = p.I / V;
  const P* w0 = reinterpret_cast<const P*>(static_cast<const T*>(p.router) + static_cast<long long>(e0) * p.I);
  const P* w1 = reinterpret_cast<const P*>(static_cast<const T*>(p.router) + static_cast<long long>(min(e1, p.E - 1)) * p.I);
  const P* x[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    x[m] = reinterpret_cast<const P*>(static_cast<const T*>(p.X) + min(t0 + m, p.tokens - 1) * p.x_row);
    acc[0][m] = acc[1][m] = 0.f;
  }
  for (int i0 = lane; i0 < n; i0 += 32 * AHEAD) {
    P a[2][AHEAD], b[M][AHEAD];
#pragma unroll
    for (int h = 0; h < AHEAD; ++h) {
      const bool there = i0 + h * 32 < n;
      a[0][h] = there ? w0[i0 + h * 32] : P{};
      a[1][h] = there ? w1[i0 + h * 32] : P{};
#pragma unroll
      for (int m = 0; m < M; ++m) b[m][h] = there ? x[m][i0 + h * 32] : P{};
    }
#pragma unroll
    for (int h = 0; h < AHEAD; ++h)
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          acc[0][m] = fmaf(a[0][h].get(v), b[m][h].get(v), acc[0][m]);
          acc[1][m] = fmaf(a[1][h].get(v), b[m][h].get(v), acc[1][m]);
        }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      acc[0][m] += __shfl_xor_sync(kAll, acc[0][m], o);
      acc[1][m] += __shfl_xor_sync(kAll, acc[1][m], o);
    }
}
// ... of the up to four tokens from t0 on, by a warp
template <typename T>
__device__ __forceinline__ void logits_by_warps(const LayerParams& p, int e, int t0) {
  constexpr int V = 16 / sizeof(T);
  if (e >= p.E) return;
  auto put = [&](int t, const auto& acc, int m) {
    if (threadIdx.x & 31) return;
    p.logits[t * p.E + e] = acc[0][m];
    if (e + 1 < p.E) p.logits[t * p.E + e + 1] = acc[1][m];
  };
  if (p.tokens - t0 == 1) {
    float acc[2][1];
    if (p.x_vectors) dots<T, V, 1, 8>(p, e, e + 1, t0, acc);
    else dots<T, 1, 1, 16>(p, e, e + 1, t0, acc);
    put(t0, acc, 0);
  } else {
    float acc[2][kRows];
    if (p.x_vectors) dots<T, V, kRows, 2>(p, e, e + 1, t0, acc);
    else dots<T, 1, kRows, 8>(p, e, e + 1, t0, acc);
#pragma unroll
    for (int m = 0; m < kRows; ++m)
      if (t0 + m < p.tokens) put(t0 + m, acc, m);
  }
}
// The logits in float32; 2.0 to 2.6 us, the latency of a router's row.
template <typename T>
__global__ void __launch_bounds__(128) few_logits_kernel(const __grid_constant__ LayerParams p) {
  pdl_wait();
  pdl_trigger();
  logits_by_warps<T>(p, (blockIdx.x * 4 + (threadIdx.x >> 5)) * 2, blockIdx.y * kRows);
}

// ---- products along rows of the weights ([contraction, columns]) -----------------------------------------------------
// Sums of V columns, two to a 64-bit register where V is even: one instruction adds two products.
template <int V> struct Sums {
  static constexpr bool kPairs = V % 2 == 0;
  using Word = typename std::conditional<kPairs, unsigned long long, float>::type;
  Word raw[kPairs ? V / 2 : V];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (auto& x : raw) x = 0;
  }
  __device__ __forceinline__ float get(int v) const {
    if constexpr (kPairs) return __uint_as_float(static_cast<uint32_t>(v & 1 ? raw[v / 2] >> 32 : raw[v / 2]));
    else return raw[v];
  }
  static __device__ __forceinline__ unsigned long long pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
  }
  template <class P>
  __device__ __forceinline__ void add(float x, const P& w) {
    if constexpr (kPairs) {
      const unsigned long long xx = pair(x, x);
#pragma unroll
      for (int v = 0; v < V; v += 2) asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(raw[v / 2]) : "l"(xx), "l"(pair(w.get(v), w.get(v + 1))));
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) raw[v] = fmaf(x, w.get(v), raw[v]);
    }
  }
};

// A group of lanes has four neighbouring rows at a time, every `step`-th such four from c on; a[m] + c - base: the other operand, zeros up to whole
// fours.  `ready` is called when the first weights have been asked for.
template <typename T, int V, int M, int AHEAD, class Ready>
__device__ __forceinline__ void accumulate(Sums<V> (&acc)[M], const T* W, int w_row, int c, int step, int end, bool on, const float* const (&a)[M], int base, Ready&& ready) {
  using P = Packed<T, V>;
  P w[AHEAD][4];
  auto load = [&]() {
    const T* from = W + static_cast<long long>(c) * w_row;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        w[i][r] = on && c + i * step + r < end ? *reinterpret_cast<const P*>(from + static_cast<long long>(i * step + r) * w_row) : P{};
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
        acc[m].add(x.x, w[i][0]);
        acc[m].add(x.y, w[i][1]);
        acc[m].add(x.z, w[i][2]);
        acc[m].add(x.w, w[i][3]);
      }
    }
    c += AHEAD * step;
    if (c < end) load();
  }
}
// Weights on their way to shared memory, DEPTH pieces of 64 bytes a thread, each thread's its own: what it asked for it reads, so that nobody waits for
// others, and the next unit's weights come while this one's sums are joined.  (Into registers, with a wait for all that had been asked for before
// more was, 43 MB came at 3.4 TB/s.)
// SHIFT: rows that begin anywhere.  What comes are the 16-byte pieces of memory that a row's tile lies in, one more than it has, and a thread shifts its elements
// together from its piece and the next thread's.
template <int THREADS, int DEPTH, int LANES, bool SHIFT>
struct Ring {
  enum : bool { kShift = SHIFT };
  uint32_t base;
  int slot = 0;
  __device__ __forceinline__ explicit Ring(const void* smem) : base(static_cast<uint32_t>(__cvta_generic_to_shared(smem))) {}
  __device__ __forceinline__ uint32_t at(int r) const { return base + static_cast<uint32_t>(slot * 4 + r) * (THREADS * 16u) + threadIdx.x * 16u; }
  __device__ __forceinline__ uint32_t behind(int r) const {        // the piece that a group of threads has beyond theirs
    return base + static_cast<uint32_t>(DEPTH * THREADS * 64) + (static_cast<uint32_t>(slot * 4 + r) * (THREADS / LANES) + threadIdx.x / LANES) * 16u;
  }
  __device__ __forceinline__ void ask(uint32_t to, const void* from, int bytes) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
  }
  __device__ __forceinline__ void asked() {        // (the slot that has been read is the one that is asked for anew)
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++slot == DEPTH) slot = 0;
  }
  __device__ __forceinline__ void wait() const {
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
    if constexpr (SHIFT) __syncwarp();
  }
  __device__ __forceinline__ void read() const {   // all that is in the slot
    if constexpr (SHIFT) __syncwarp();
  }
  __device__ __forceinline__ static uint4 load(uint32_t from) {
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(from) : "memory");
    return x;
  }
  // first: bytes of this thread's piece that are before its elements
  template <class P>
  __device__ __forceinline__ P get(int r, uint32_t first) const {
    static_assert(sizeof(P) == 16, "pieces are of 16 bytes");
    union {
      uint4 raw;
      P value;
    } x{};
    x.raw = load(at(r));
    if constexpr (SHIFT) {
      const uint4 y = load(threadIdx.x % LANES == LANES - 1 ? behind(r) : at(r) + 16u);
      uint32_t w[8] = {x.raw.x, x.raw.y, x.raw.z, x.raw.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = first & 8u ? w[i + 2] : w[i];
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = first & 4u ? w[i + 1] : w[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (first & 2u) * 8u);
      x.raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return x.value;
  }
};
// Shifted rows: `left` of four from `row` on (of all experts' rows), from column n0 on; all: bytes of the weights, which begin `first` elements behind W.
template <typename T, int LANES, class R>
__device__ __forceinline__ void ask_shifted(const R& ring, const void* W, uint32_t first, int N, long long row, int left, int n0, long long all) {
  const int lane = threadIdx.x % LANES;
  long long begin = (row * N + n0 + first) * static_cast<long long>(sizeof(T));
  all += first * static_cast<long long>(sizeof(T));
  auto ask = [&](uint32_t to, long long at, int r) {
    const int there = r < left ? static_cast<int>(max(min(all - at, 16ll), 0ll)) : 0;
    ring.ask(to, there ? static_cast<const char*>(W) + at : W, there);
  };
#pragma unroll
  for (int r = 0; r < 4; ++r, begin += N * static_cast<long long>(sizeof(T))) {
    ask(ring.at(r), (begin & ~15ll) + lane * 16, r);
    if (lane == r) ask(ring.behind(r), (begin & ~15ll) + LANES * 16, r);
  }
}
// Four rows of weights times M rows of the other operand at `at`.  Shifted rows: element `first` of all is the first row's first, they are N apart.
template <typename T, int V, int M, class R>
__device__ __forceinline__ void add_four(Sums<V> (&acc)[M], const R& ring, const float* const (&a)[M], int at, uint32_t first, uint32_t N) {
  Packed<T, V> w[4];
#pragma unroll
  for (int r = 0; r < 4; ++r, first += N) w[r] = ring.template get<Packed<T, V>>(r, first * sizeof(T));
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const float4 x = *reinterpret_cast<const float4*>(a[m] + at);
    acc[m].add(x.x, w[0]);
    acc[m].add(x.y, w[1]);
    acc[m].add(x.z, w[2]);
    acc[m].add(x.w, w[3]);
  }
}
// Sums over the groups of lanes: all lanes have them.
template <int LANES, int V, int M>
__device__ __forceinline__ void join_groups(const Sums<V> (&acc)[M], float (&sum)[M][V]) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float x = acc[m].get(v);
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) x += __shfl_xor_sync(kAll, x, o);
      sum[m][v] = x;
    }
}
constexpr int kAhead = 4;                    // steps of single elements whose loads go out together

template <typename T, int V, int LANES>
struct UpShared {
  Items items;
  Scratch scratch;
  alignas(16) float x[kRows][kUpPart];
  float sums[kUpWarps][kRows][LANES * V];
};

struct UpUnit {
  int item, part, n0, begin, end;
};
__device__ __forceinline__ UpUnit up_unit_of(const LayerParams& p, int u, int all, int length, int whole, int tile) {
  UpUnit x;
  x.part = u / all;
  const int rest = u - x.part * all;
  x.item = p.by_tiles.quotient(rest);
  x.n0 = (rest - x.item * p.by_tiles.d) * tile;
  x.begin = min(whole, x.part * length);
  x.end = min(whole, x.begin + length);
  return x;
}

// A unit's products; ring: has its weights (16-byte vectors), `next` asks for more; without it (narrow ones) they are asked for here.
template <typename T, int V, int LANES, int M, class R, class Next>
__device__ __forceinline__ void up_unit(const LayerParams& p, UpShared<T, V, LANES>* s, const UpUnit& u, float* to, R& ring, Next&& next) {
  constexpr int kStep = kUpThreads / LANES * 4, kTile = LANES * V;
  const int tid = threadIdx.x, l = tid % LANES, n = u.n0 + l * V;
  const Item item = s->items.item[u.item];
  const T* W = static_cast<const T*>(p.up) + item.expert * (p.up_row * p.I) + n;
  Sums<V> acc[M];
  const float* a[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    a[m] = s->x[m];
    acc[m].zero();
  }
  for (int c0 = u.begin; c0 < u.end; c0 += kUpPart) {
    const int c1 = min(u.end, c0 + kUpPart), first = c0 + tid / LANES * 4;
    auto stage = [&]() {
      __syncthreads();                         // what was in shared memory has been read
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const T* x = static_cast<const T*>(p.X) + p.by_k.quotient(item.slot[m]) * p.x_row;
        for (int i = tid; i < ((c1 - c0 + 3) & ~3); i += kUpThreads) s->x[m][i] = c0 + i < c1 ? to_f32<T>(x[c0 + i]) : 0.f;
      }
      __syncthreads();
    };
    if constexpr (V == 16 / sizeof(T)) {
      stage();
      for (int c = first, left = (c1 - c0 + kStep - 1) / kStep; left; --left, c += kStep) {
        ring.wait();
        if (c < c1) add_four<T, V, M>(acc, ring, a, c - c0, R::kShift ? (static_cast<uint32_t>(item.expert) * p.I + c) * p.J + u.n0 + p.up_first : 0u, p.J);
        ring.read();
        next();
      }
    } else {
      accumulate<T, V, M, kAhead>(acc, W, static_cast<int>(p.up_row), first, kStep, c1, n < p.J, a, c0, stage);
    }
  }
  float sum[M][V];
  join_groups<LANES, V, M>(acc, sum);
  if ((tid & 31) < LANES) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int v = 0; v < V; ++v) s->sums[tid >> 5][m][l * V + v] = sum[m][v];
  }
  __syncthreads();
  for (int i = tid; i < M * kTile; i += kUpThreads) {
    const int m = i / kTile, col = i % kTile;
    if (m >= item.rows || u.n0 + col >= p.J) continue;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kUpWarps; ++w) t += s->sums[w][m][col];
    to[static_cast<long long>(item.slot[m]) * p.J + u.n0 + col] = t;
  }
}

constexpr int kUpDepth = 4, kDownDepth = 3;
constexpr size_t ring_bytes(int threads, int depth, int lanes) { return static_cast<size_t>(threads) * depth * 64 + (lanes ? static_cast<size_t>(threads / lanes) * depth * 64 : 0); }

// Parts of the first product.  Two CTAs an SM, so that one loads while the other joins its sums; a tile is 128 bytes of a row (eight lanes), of which 32 rows come at a time.
template <typename T, int V, int LANES, bool SHIFT>
__global__ void __launch_bounds__(kUpThreads, 2) few_up_kernel(const __grid_constant__ LayerParams p) {
  constexpr int kTile = LANES * V, kStep = kUpThreads / LANES * 4;
  constexpr bool kRing = V == 16 / sizeof(T);
  extern __shared__ __align__(16) uint32_t layer_table[];
  __shared__ UpShared<T, V, LANES> s;
  pdl_wait();
  pdl_trigger();
  list_items(p, &s.items, &s.scratch);
  const int parts = parts_of(s.items.count * p.by_tiles.d, p.I);
  const int all = s.items.count * p.by_tiles.d, units = all * parts, length = ((p.I + parts - 1) / parts + 3) & ~3;
  Ring<kUpThreads, kUpDepth, LANES, SHIFT> ring(layer_table);
  // what is asked for next: rows c .. c + 3 of unit `coming`
  int coming = blockIdx.x, c = 0, end = 0, left = 0;
  bool on = false;
  const T* from = static_cast<const T*>(p.up);
  long long first_row = 0;
  int n0 = 0;
  auto next = [&]() {
    if (left == 0 && coming < units) {
      const UpUnit x = up_unit_of(p, coming, all, length, p.I, kTile);
      const int n = x.n0 + threadIdx.x % LANES * V;
      on = n < p.J;
      c = x.begin + threadIdx.x / LANES * 4;
      end = x.end;
      left = (x.end - x.begin + kStep - 1) / kStep;
      from = static_cast<const T*>(p.up) + s.items.item[x.item].expert * (p.up_row * p.I) + c * p.up_row + n;
      first_row = static_cast<long long>(s.items.item[x.item].expert) * p.I;
      n0 = x.n0;
      coming += gridDim.x;
    }
    if (left) {
      if constexpr (SHIFT) {
        ask_shifted<T, LANES>(ring, p.up, p.up_first, p.J, first_row + c, end - c, n0, p.weight_bytes);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool there = on && c + r < end;
          ring.ask(ring.at(r), there ? from + r * p.up_row : static_cast<const T*>(p.up), there ? 16 : 0);
        }
      }
      c += kStep;
      from += kStep * p.up_row;
      --left;
    }
    ring.asked();
  };
  if constexpr (kRing) {
#pragma unroll 1
    for (int d = 0; d < kUpDepth; ++d) next();
  }
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const UpUnit x = up_unit_of(p, u, all, length, p.I, kTile);
    float* to = p.h + static_cast<long long>(x.part) * p.tokens * p.k * p.J;
    const int rows = s.items.item[x.item].rows;
    if (rows == 1) up_unit<T, V, LANES, 1>(p, &s, x, to, ring, next);
    else if (rows == 2) up_unit<T, V, LANES, 2>(p, &s, x, to, ring, next);
    else up_unit<T, V, LANES, kRows>(p, &s, x, to, ring, next);
  }
}

// The items and the choice's weights, in shared memory.  `down` calls this ahead of its wait: what the choice has written is there, since `up` lets its dependents begin when all of its
// CTAs have waited for the choice, and with it for all that came before.  So are weights of the layer.
struct DownShared : Items {
  float weights[kMost];
};
__device__ __forceinline__ void begin_down(const LayerParams& p, DownShared* s, void* scratch) {
  for (int i = threadIdx.x; i < p.tokens * p.k; i += blockDim.x) s->weights[i] = __ldcg(p.weights + i);
  list_items(p, s, static_cast<Scratch*>(scratch));
  __syncthreads();                             // (and the scratch is free)
}

// N neighbouring sums of a slot's parts from h[at] on (those that exist: left), activated.  All loads go out before the first sum.
template <int N>
__device__ __forceinline__ void activation(const LayerParams& p, int parts, long long at, int left, float (&v)[N]) {
  const long long far = static_cast<long long>(p.tokens) * p.k * p.J;
  float x[kMostParts][N];
  const bool vectors = N % 4 == 0 && left >= N && p.J % 4 == 0;
#pragma unroll
  for (int s = 0; s < kMostParts; ++s) {
    const float* h = p.h + at + s * far;
    if (vectors) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const float4 y = s < parts ? reinterpret_cast<const float4*>(h)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
        x[s][4 * i] = y.x; x[s][4 * i + 1] = y.y; x[s][4 * i + 2] = y.z; x[s][4 * i + 3] = y.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[s][i] = s < parts && i < left ? h[i] : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float sum = x[0][i];
#pragma unroll
    for (int s = 1; s < kMostParts; ++s) sum += x[s][i];
    v[i] = i < left ? sum / (1.f + expf(-sum)) : 0.f;
  }
}

// out[t, n0 + n] from this CTA's sums: sum(t, n, v) adds four of them to v.  Every CTA of a cluster has a share of the outputs, and the others hand it their
// sums: to, room for them, [CTAs][outputs of a share] of shared memory.
template <typename T, int TILE, class Sum>
__device__ __forceinline__ void put_out(const LayerParams& p, float* to, int n0, int split, Sum&& sum) {
  const int rank = cluster_rank(), size = cluster_size(), all = p.tokens * TILE, own = (all / 4 + size - 1) / size * 4;
  auto put = [&](int t, int n, float v) {
    if (n0 + n >= p.I) return;
    const long long at = static_cast<long long>(t) * p.I + n0 + n;
    if (gridDim.y > 1) p.sums[split * (static_cast<long long>(p.tokens) * p.I) + at] = v;
    else static_cast<T*>(p.out)[at] = from_f32<T>(v);
  };
  if (size > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // all have begun
  for (int i = threadIdx.x * 4; i < all; i += blockDim.x * 4) {
    const int t = i / TILE, n = i % TILE;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    sum(t, n, v);
    if (size == 1) {
      put(t, n, v.x);
      put(t, n + 1, v.y);
      put(t, n + 2, v.z);
      put(t, n + 3, v.w);
    } else {
      const int owner = i / own;
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(in_cta(to + rank * own + i - owner * own, owner)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
    }
  }
  if (size == 1) return;
  cluster_sync();
  for (int i = threadIdx.x; i < min(own, all - rank * own); i += blockDim.x) {
    const int x = rank * own + i, t = x / TILE, n = x % TILE;
    float v = to[i];
    for (int r = 1; r < size; ++r) v += to[r * own + i];
    put(t, n, v);
  }
}

template <typename T, int V, int LANES, int M, class R, class Next>
__device__ __forceinline__ void down_item(const LayerParams& p, const Item& item, const float* act, int pitch, int base, int begin, int end, int n0, float* part, bool first, R& ring, Next&& next) {
  constexpr int kTile = LANES * V, kStep = 32 / LANES * 4;
  const int lane = threadIdx.x & 31, l = lane % LANES, n = n0 + l * V;
  Sums<V> acc[M];
  const float* a[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    a[m] = act + item.slot[m] * pitch;
    acc[m].zero();
  }
  if constexpr (V == 16 / sizeof(T)) {
    for (int c = begin + lane / LANES * 4, left = (end - begin + kStep - 1) / kStep; left; --left, c += kStep) {
      ring.wait();
      if (c < end) add_four<T, V, M>(acc, ring, a, c - base, R::kShift ? (static_cast<uint32_t>(item.expert) * p.J + c) * p.I + n0 + p.down_first : 0u, p.I);
      ring.read();
      next();
    }
  } else {
    accumulate<T, V, M, kAhead>(acc, static_cast<const T*>(p.down) + item.expert * (p.down_row * p.J) + n, static_cast<int>(p.down_row), begin + lane / LANES * 4, kStep, end, n < p.I, a, base, []() {});
  }
  float sum[M][V];
  join_groups<LANES, V, M>(acc, sum);
  if (lane < LANES) {
#pragma unroll
    for (int m = 0; m < M; ++m)
      if (m < item.rows) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float* to = part + item.slot[m] * kTile + l * V + v;
          *to = first ? sum[m][v] : *to + sum[m][v];
        }
      }
  }
}

// The second product and the sum over the choices.  Clusters, because the contraction is short and the columns are few: a token's sums of all CTAs meet in shared memory instead of
// in another launch.  16 warps have items of their own, so that no two write the same sums.
template <typename T, int V, int LANES, bool SHIFT>
__global__ void __launch_bounds__(kDownThreads, 1) few_down_kernel(const __grid_constant__ LayerParams p) {
  constexpr int kTile = LANES * V, kStep = 32 / LANES * 4;
  constexpr bool kRing = V == 16 / sizeof(T);
  extern __shared__ __align__(16) float layer_smem[];
  __shared__ DownShared items;
  if (cluster_size() > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  begin_down(p, &items, layer_smem);
  const int slots = p.tokens * p.k, rank = cluster_rank(), size = cluster_size(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.y, n0 = blockIdx.x / size * kTile;
  float* act = layer_smem + p.ring_words;
  float* part = act + p.act_floats;
  const int parts = parts_of(items.count * p.by_tiles.d, p.I);
  const int ctas = size * p.splits, length = ((p.J + ctas - 1) / ctas + 3) & ~3, begin = min(p.J, (split * size + rank) * length), end = min(p.J, begin + length);
  const int room = min(length, p.act_floats / slots & ~3);
  int shares_log2 = 0;                         // warps that have an item's contraction in turn
  while (items.count << (shares_log2 + 1) <= kDownWarps && length >> shares_log2 >= 64) ++shares_log2;
  const int turns = items.count << shares_log2;
  Ring<kDownThreads, kDownDepth, LANES, SHIFT> ring(layer_smem);
  for (int c0 = begin; c0 == begin || c0 < end; c0 += room) {
    const int c1 = min(end, c0 + room), width = (c1 - c0 + 3) & ~3, each = ((width / 4 + (1 << shares_log2) - 1) >> shares_log2) * 4;
    auto share_of = [&](int x, int* to) {      // first row, and the one behind the last
      const int b = min(c1, c0 + (x & ((1 << shares_log2) - 1)) * each);
      *to = min(c1, b + each);
      return b;
    };
    // what is asked for next: rows c .. c + 3 of turn `coming`
    int coming = warp, c = 0, stop = 0, left = 0;
    const T* from = static_cast<const T*>(p.down);
    const bool on = n0 + lane % LANES * V < p.I;
    long long first_row = 0;
    auto next = [&]() {
      while (left == 0 && coming < turns) {
        const int b = share_of(coming, &stop);
        c = b + lane / LANES * 4;
        left = (stop - b + kStep - 1) / kStep;
        from = static_cast<const T*>(p.down) + items.item[coming >> shares_log2].expert * (p.down_row * p.J) + c * p.down_row + n0 + lane % LANES * V;
        first_row = static_cast<long long>(items.item[coming >> shares_log2].expert) * p.J;
        coming += kDownWarps;
      }
      if (left) {
        if constexpr (SHIFT) {
          ask_shifted<T, LANES>(ring, p.down, p.down_first, p.I, first_row + c, stop - c, n0, p.weight_bytes);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool there = on && c + r < stop;
            ring.ask(ring.at(r), there ? from + r * p.down_row : static_cast<const T*>(p.down), there ? 16 : 0);
          }
        }
        c += kStep;
        from += kStep * p.down_row;
        --left;
      }
      ring.asked();
    };
    if constexpr (kRing) {
#pragma unroll 1
      for (int d = 0; d < kDownDepth; ++d) next();
    }
    if (c0 == begin) {                         // the first weights are on their way
      pdl_wait();
      pdl_trigger();
    }
    // activations, four at a time
    __syncthreads();
    for (int i = tid; i < slots * (width / 4); i += kDownThreads) {
      const int slot = i / (width / 4), at = (i - slot * (width / 4)) * 4;
      const float w = items.weights[slot];
      float v[4];
      activation<4>(p, parts, static_cast<long long>(slot) * p.J + c0 + at, c1 - c0 - at, v);
      *reinterpret_cast<float4*>(act + slot * room + at) = make_float4(w * v[0], w * v[1], w * v[2], w * v[3]);
    }
    __syncthreads();
    for (int x = warp; x < turns; x += kDownWarps) {
      int e;
      const int b = share_of(x, &e);
      const Item item = items.item[x >> shares_log2];
      float* to = part + (x & ((1 << shares_log2) - 1)) * slots * kTile;
      if (item.rows == 1) down_item<T, V, LANES, 1>(p, item, act, room, c0, b, e, n0, to, c0 == begin, ring, next);
      else if (item.rows == 2) down_item<T, V, LANES, 2>(p, item, act, room, c0, b, e, n0, to, c0 == begin, ring, next);
      else down_item<T, V, LANES, kRows>(p, item, act, room, c0, b, e, n0, to, c0 == begin, ring, next);
    }
  }
  __syncthreads();
  put_out<T, kTile>(p, part + max(4 * kDownWarps, slots) * kTile, n0, split, [&](int t, int n, float4& v) {
    for (int j = 0; j < p.k << shares_log2; ++j) {
      const float4 x = *reinterpret_cast<const float4*>(part + ((j & ((1 << shares_log2) - 1)) * slots + t * p.k + (j >> shares_log2)) * kTile + n);
      v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    }
  });
}

// The splits' sums, in their order.
template <typename T>
__global__ void __launch_bounds__(256) few_join_kernel(const __grid_constant__ LayerParams p) {
  pdl_wait();
  pdl_trigger();
  const long long all = static_cast<long long>(p.tokens) * p.I, i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= all) return;
  float v[kMostSplits];
#pragma unroll
  for (int s = 0; s < kMostSplits; ++s) v[s] = s < p.splits ? p.sums[s * all + i] : 0.f;
#pragma unroll
  for (int s = 1; s < kMostSplits; ++s) v[0] += v[s];
  static_cast<T*>(p.out)[i] = from_f32<T>(v[0]);
}

// ---- weights in 4 bits -------------------------------------------------------------------------------------------------
// Rows and weights become 16-bit floats, which hold them exactly, and go through the tensor cores (mma.sync: 16 columns, 16 contraction elements, up to eight
// rows); a block's sums are exact, then times both scales into float32 sums.  (As integers through dp4a four columns and a block took 980
// instructions a warp: 83 us a call, 8 tokens, 8 of 64 experts, 2048 x 512, 47 MB.  Now 35 to 38: 4.3 (NC) to 5.1 million warp instructions a product, a third of which ask for
// weights; with cold caches a product took 20 us, 16 without its arithmetic and 12 without its loads, and takes 14 (NC) to 17 now.)  The weights' bytes lie along the contraction (NC) or along the columns (CN).
// A warp's stage: 4 blocks of the contraction x a tile of 32 columns, 2 KB of weights; kDepth4 stages are on their way, each warp's its own.  Lane (g, q) = (lane / 4,
// lane % 4) multiplies columns 4 g .. 4 g + 3 and of each block the eight elements from 8 q on; their order is the same in both operands.
constexpr int kTile4 = 32, kStage4 = 4, kDepth4 = 3, kThreads4 = 256, kWarps4 = kThreads4 / 32;
constexpr int kRowPitch4 = 320;                // a row's 256 bytes, in other banks than the next one's
constexpr int kStageRows4 = 2048, kStageScale4 = kStageRows4 + kRows * kRowPitch4, kStageF4 = kStageScale4 + 128, kStageBytes4 = kStageF4 + kRows * 16;
constexpr int kWarpBytes4 = kDepth4 * kStageBytes4 + 512;      // ... and the scales of a stage as floats
constexpr size_t kRing4 = static_cast<size_t>(kWarps4) * kWarpBytes4;
__host__ __device__ constexpr int stages_of(int C) { return (fp4_blocks(C) + kStage4 - 1) / kStage4; }
enum Layout4 { kNC, kCN16, kCN4, kCN1 };       // CN: rows, counted from the tensor's begin, are whole pieces of so many bytes

struct Matrix4 {
  const uint8_t *w, *s;
  long long far, s_far;        // bytes from one expert to the next
  uint32_t row;                // NC: from one column to the next, CN: from one pair of contraction elements to the next
  uint32_t s_row;              // from one column's scales to the next
  int C, N;
  bool words;                  // scales can be read four at a time
};
__device__ __forceinline__ unsigned long long wide(uint32_t a, uint32_t b) { return static_cast<unsigned long long>(a) * b; }
// Rows in 16-bit floats, whole blocks, and their scales, whole stages.
struct Rows4 {
  __half* x;
  float* f;
  int C;
  __device__ __forceinline__ const __half* row(int i) const { return x + static_cast<long long>(i) * fp4_blocks(C) * kFp4Block; }
  __device__ __forceinline__ const float* scale(int i) const { return f + i * stages_of(C) * kStage4; }
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t word_at(uint32_t at) {
  uint32_t x;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ uint4 words_at(uint32_t at) {
  uint4 x;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
  return x;
}
// Eight floats to the nearest of 4 bits, as 16-bit floats.  (By way of integers: see fp4_halves.)
__device__ __forceinline__ uint4 fp4_rounded(const float (&v)[8]) {
  uint32_t twice[2];
  fp4_integers(fp4_pack8(v), twice[0], twice[1]);
  alignas(16) __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int two = static_cast<int>(twice[i / 2] >> (i % 2 * 16));
    h[i] = __floats2half2_rn(0.5f * static_cast<signed char>(two), 0.5f * static_cast<signed char>(two >> 8));
  }
  return *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// acc += d * low * power * high of two rows, in this order (see fp4_factors).
__device__ __forceinline__ void add_scaled(float2& acc, float2 d, float2 low, float power, float2 high) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 b, {%6, %6};\n\tmul.rn.f32x2 a, a, b;\n\t"
      "mov.b64 b, {%7, %8};\n\tmov.b64 c, {%0, %1};\n\tfma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "+f"(acc.x), "+f"(acc.y) : "f"(d.x), "f"(d.y), "f"(low.x), "f"(low.y), "f"(power), "f"(high.x), "f"(high.y));
}

template <int LAYOUT>
struct Stages {
  const Matrix4& t;
  uint32_t base;
  int ask_slot = 0, get_slot = 0;
  uint32_t late[kStage4];      // scales that are read byte by byte, stored when the next stage is asked for
  uint32_t late_at = 0;
  uint32_t own;                // where this lane's first piece of a stage goes
  // of the unit that is asked for: where this lane's pieces of its first stage are
  const uint8_t *w, *s;
  const char *x0, *x1, *f;
  int n0, rows, whole;         // whole: stages that need no bounds

  __device__ __forceinline__ Stages(const void* smem, const Matrix4& m) : t(m), base(static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + (threadIdx.x >> 5) * kWarpBytes4) {
    const int lane = threadIdx.x & 31, i = lane >> 1, col = lane >> 2;
    own = LAYOUT == kNC ? (((col & 3) * 8 + (col >> 2)) * 4) * 16 : ((i & 3) * 4 + (i >> 2)) * 32 + (lane & 1) * 16;
  }
  // Columns [column, column + 32) of an expert and `m` rows; which(i): the i-th one's place in x.
  template <class Which>
  __device__ __forceinline__ void begin(int expert, int column, const Rows4& x, int m, Which&& which) {
    const int lane = threadIdx.x & 31;
    n0 = column;
    rows = m;
    w = t.w + expert * t.far;
    if constexpr (LAYOUT == kNC) w += wide(n0 + (lane >> 2), t.row) + (lane & 3) * 16;
    else if constexpr (LAYOUT == kCN1) w += n0 + lane;
    else w += n0 + (lane & 1) * 16 + wide(lane >> 1, t.row);
    s = t.s + expert * t.s_far + wide(n0 + lane, t.s_row);
    const uint32_t pitch = fp4_blocks(x.C) * kFp4Block * 2, piece = (lane & 15) * 16;
    x0 = reinterpret_cast<const char*>(x.x) + wide(which(lane >> 4), pitch) + piece;
    x1 = reinterpret_cast<const char*>(x.x) + wide(which(2 + (lane >> 4)), pitch) + piece;
    f = reinterpret_cast<const char*>(x.f) + wide(which(lane & 3), stages_of(x.C) * kStage4 * 4);
    whole = t.words && LAYOUT != kCN1 && n0 + kTile4 <= t.N ? (t.C + 1) / 2 / (kStage4 * 16) : 0;
  }
  __device__ __forceinline__ void store_late() {
    if (late_at == 0) return;
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(late_at), "r"(late[0] | late[1] << 8 | late[2] << 16 | late[3] << 24) : "memory");
    late_at = 0;
  }
  __device__ __forceinline__ void ask(int stage) {
    const int lane = threadIdx.x & 31;
    const uint32_t to = base + ask_slot * kStageBytes4;
    const uint8_t* from = w + (LAYOUT == kNC ? wide(stage, kStage4 * 16) : wide(stage * (kStage4 * 16), t.row));
    const unsigned long long step = wide(LAYOUT == kNC ? 8 : 16, t.row);
    const uint32_t x_to = to + kStageRows4 + (lane >> 4) * kRowPitch4 + (lane & 15) * 16, x_from = stage * (kStage4 * kFp4Block * 2);
    if (stage < whole) {
#pragma unroll
      for (int r = 0; r < 4; ++r, from += step) {
        if constexpr (LAYOUT == kNC) copy16(to + own + r * 128 + (((lane & 3) ^ r) << 4), from, 16);
        else if constexpr (LAYOUT == kCN16) copy16(to + own + r * 512, from, 16);
        else
#pragma unroll
          for (int j = 0; j < 4; ++j) copy4(to + own + r * 512 + 4 * j, from + 4 * j, 4);
      }
      copy4(to + kStageScale4 + lane * 4, s + stage * kStage4, 4);
      if ((lane >> 4) < rows) copy16(x_to, x0 + x_from, 16);
      if (2 + (lane >> 4) < rows) copy16(x_to + 2 * kRowPitch4, x1 + x_from, 16);
      if (lane < rows) copy16(to + kStageF4 + lane * 16, f + stage * (kStage4 * 4), 16);
      return;
    }
    store_late();
    const int b0 = stage * kStage4, half = (t.C + 1) / 2, left_blocks = min(fp4_blocks(t.C) - b0, kStage4);
    if constexpr (LAYOUT == kNC) {
      const int left = half - (b0 + (lane & 3)) * 16;
#pragma unroll
      for (int r = 0; r < 4; ++r, from += step) {       // column c = 8 r + lane / 4 to the place (c % 4, c / 4), its pieces in turns
        const int bytes = n0 + r * 8 + (lane >> 2) < t.N ? max(min(left, 16), 0) : 0;
        copy16(to + own + r * 128 + (((lane & 3) ^ r) << 4), bytes ? from : t.w, bytes);
      }
    } else if constexpr (LAYOUT == kCN1) {
#pragma unroll 1
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i, from += t.row) {
          const uint32_t v = (b0 + r) * 16 + i < half && n0 + lane < t.N ? *from : 0u;
          asm volatile("st.shared.u8 [%0], %1;" ::"r"(to + (r * 16 + (i & 3) * 4 + (i >> 2)) * 32 + lane), "r"(v) : "memory");
        }
    } else {
      const int left = t.N - n0 - (lane & 1) * 16;
#pragma unroll
      for (int r = 0; r < 4; ++r, from += step) {
        const int bytes = (b0 + r) * 16 + (lane >> 1) < half ? max(min(left, 16), 0) : 0;
        if constexpr (LAYOUT == kCN16) {
          copy16(to + own + r * 512, bytes ? from : t.w, bytes);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) copy4(to + own + r * 512 + 4 * j, j * 4 < bytes ? from + 4 * j : t.w, max(min(bytes - j * 4, 4), 0));
        }
      }
    }
    const int blocks = n0 + lane < t.N ? left_blocks : 0;
    if (t.words) {
      copy4(to + kStageScale4 + lane * 4, blocks ? s + b0 : t.s, blocks);
    } else {
#pragma unroll
      for (int i = 0; i < kStage4; ++i) late[i] = i < blocks ? s[b0 + i] : 0;
      late_at = to + kStageScale4 + lane * 4;
    }
    const bool there = (lane & 15) / 4 < left_blocks;
    if ((lane >> 4) < rows) copy16(x_to, there ? x0 + x_from : x0, there ? 16 : 0);
    if (2 + (lane >> 4) < rows) copy16(x_to + 2 * kRowPitch4, there ? x1 + x_from : x1, there ? 16 : 0);
    if (lane < rows) copy16(to + kStageF4 + lane * 16, f + b0 * 4, left_blocks * 4);
  }
  __device__ __forceinline__ void asked() {
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++ask_slot == kDepth4) ask_slot = 0;
  }
  // acc[i]: columns 4 g + i of `count` rows, 2 q and 2 q + 1 (of q < 2)
  __device__ __forceinline__ void add(float2 (&acc)[4], int count) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const uint32_t from = base + get_slot * kStageBytes4, powers = base + kDepth4 * kStageBytes4;
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth4 - 1) : "memory");
    __syncwarp();
    const uint32_t bytes = word_at(from + kStageScale4 + lane * 4);
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(powers + ((lane & 3) * 8 + g) * 16), "f"(fp4_power(bytes & 255u)), "f"(fp4_power(bytes >> 8 & 255u)), "f"(fp4_power(bytes >> 16 & 255u)),
                 "f"(fp4_power(bytes >> 24)) : "memory");
    __syncwarp();
    float power[4][kStage4], scale[2][kStage4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = words_at(powers + (i * 8 + g) * 16);
      power[i][0] = __uint_as_float(v.x); power[i][1] = __uint_as_float(v.y); power[i][2] = __uint_as_float(v.z); power[i][3] = __uint_as_float(v.w);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 v = words_at(from + kStageF4 + ((q & 1) * 2 + i) * 16);
      scale[i][0] = __uint_as_float(v.x); scale[i][1] = __uint_as_float(v.y); scale[i][2] = __uint_as_float(v.z); scale[i][3] = __uint_as_float(v.w);
    }
#pragma unroll
    for (int kk = 0; kk < kStage4; ++kk) {
      uint32_t w[4];
      if constexpr (LAYOUT == kNC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = word_at(from + ((i * 8 + g) * 4 + (kk ^ (g >> 1))) * 16 + q * 4);
      } else {
        uint32_t r[4];                         // four columns of a pair of elements each: to four pairs of a column each
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = word_at(from + (kk * 16 + i * 4 + q) * 32 + g * 4);
        const uint32_t p0 = __byte_perm(r[0], r[1], 0x5140), p1 = __byte_perm(r[2], r[3], 0x5140), p2 = __byte_perm(r[0], r[1], 0x7362), p3 = __byte_perm(r[2], r[3], 0x7362);
        w[0] = __byte_perm(p0, p1, 0x5410);
        w[1] = __byte_perm(p0, p1, 0x7632);
        w[2] = __byte_perm(p2, p3, 0x5410);
        w[3] = __byte_perm(p2, p3, 0x7632);
      }
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (g < count) x = words_at(from + kStageRows4 + g * kRowPitch4 + kk * 64 + q * 16);
      float low0, low1, high0, high1;
      fp4_factors(scale[0][kk], low0, high0);
      fp4_factors(scale[1][kk], low1, high1);
      const float2 low = make_float2(low0, low1), high = make_float2(high0, high1);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        uint32_t a[4], b[4];
        fp4_halves(w[i], a);
        fp4_halves(w[i + 1], b);
        float d[4];
        mma16(d, a[0], b[0], a[1], b[1], x.x, x.y, 0.f, 0.f, 0.f, 0.f);
        mma16(d, a[2], b[2], a[3], b[3], x.z, x.w, d[0], d[1], d[2], d[3]);
        add_scaled(acc[i], make_float2(d[0], d[1]), low, power[i][kk], high);
        add_scaled(acc[i + 1], make_float2(d[2], d[3]), low, power[i + 1][kk], high);
      }
    }
    __syncwarp();                              // the slot may be asked for anew, the powers written
    if (++get_slot == kDepth4) get_slot = 0;
  }
};

// Eight of a block's 32 values by each of four neighbouring lanes, in 4 bits, as 16-bit floats; the block's scale.
__device__ __forceinline__ float block4(const float (&v)[8], __half* to) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(kAll, top, 1));
  top = max(top, __shfl_xor_sync(kAll, top, 2));
  const uint32_t byte = fp4_scale(top);
  const float inverse = fp4_inverse(byte);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fp4_scaled(v[i], inverse);
  if (to) *reinterpret_cast<uint4*>(to) = fp4_rounded(x);
  return fp4_power(byte);
}

// The logits, as few_logits_kernel's, and behind their CTAs those that bring X into 4 bits.
template <typename T>
__global__ void __launch_bounds__(128) few_logits4_kernel(const __grid_constant__ LayerParams p, const Rows4 to, int logits_ctas) {
  pdl_wait();
  pdl_trigger();
  const int t0 = blockIdx.y * kRows;
  if (blockIdx.x < logits_ctas) {
    logits_by_warps<T>(p, (blockIdx.x * 4 + (threadIdx.x >> 5)) * 2, t0);
    return;
  }
  constexpr int kVec = 16 / sizeof(T);
  const int blocks = fp4_blocks(p.I), i = (blockIdx.x - logits_ctas) * 128 + threadIdx.x, c = i * 8;
  float v[kRows][8];
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    const T* from = static_cast<const T*>(p.X) + min(t0 + m, p.tokens - 1) * p.x_row + c;
    if (p.x_vectors && c + 8 <= p.I) {
#pragma unroll
      for (int h = 0; h < 8 / kVec; ++h) {
        const Packed<T, kVec> y = reinterpret_cast<const Packed<T, kVec>*>(from)[h];
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[m][h * kVec + j] = y.get(j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[m][j] = c + j < p.I ? to_f32<T>(from[j]) : 0.f;
    }
  }
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    const bool there = i / 4 < blocks && t0 + m < p.tokens;
    const float f = block4(v[m], there ? const_cast<__half*>(to.row(t0 + m)) + c : nullptr);
    if (there && i % 4 == 0) const_cast<float*>(to.scale(t0 + m))[i / 4] = f;
  }
}

// Units go round the CTAs: an item's products with a tile of columns, its warps the contraction in turn.  What the warps' sums add up to is activated and, one block of
// the other product's contraction, brought into 4 bits.
struct Up4Shared {
  Items items;
  Scratch scratch;
  float sums[2][kWarps4][kRows][kTile4];
};
template <int LAYOUT>
__global__ void __launch_bounds__(kThreads4, 2) few_up4_kernel(const __grid_constant__ LayerParams p, const __grid_constant__ Matrix4 t, const Rows4 x, const Rows4 to) {
  extern __shared__ __align__(16) uint32_t layer_table[];
  __shared__ Up4Shared s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  list_items(p, &s.items, &s.scratch);
  if (blockIdx.x == 0) {
    for (int i = tid; i < s.items.count; i += kThreads4) p.list->item[i] = s.items.item[i];
    if (tid == 0) p.list->count = s.items.count;
  }
  const int tiles = p.by_tiles.d, units = s.items.count * tiles, stages = stages_of(p.I);
  Stages<LAYOUT> ring(layer_table, t);
  int coming = warp < stages ? blockIdx.x : units, stage = stages;       // of what is asked for next; (a contraction of few stages leaves warps idle)
  auto next = [&]() {
    if (stage >= stages && coming < units) {
      const int which = p.by_tiles.quotient(coming);
      const Item& item = s.items.item[which];
      ring.begin(item.expert, (coming - which * tiles) * kTile4, x, item.rows, [&](int m) { return p.by_k.quotient(item.slot[m]); });
      stage = warp;
      coming += gridDim.x;
    }
    if (stage < stages) {
      ring.ask(stage);
      stage += kWarps4;
    } else {
      ring.store_late();
    }
    ring.asked();
  };
#pragma unroll 1
  for (int d = 0; d < kDepth4 - 1; ++d) next();
  int buffer = 0;
  for (int u = blockIdx.x; u < units; u += gridDim.x, buffer ^= 1) {
    const int which = p.by_tiles.quotient(u), n0 = (u - which * tiles) * kTile4;
    const Item item = s.items.item[which];
    float2 acc[4] = {};
    for (int i = warp; i < stages; i += kWarps4) {
      next();
      ring.add(acc, item.rows);
    }
    const int g = lane >> 2, q = lane & 3;
    if (q < 2) {
      *reinterpret_cast<float4*>(&s.sums[buffer][warp][2 * q][4 * g]) = make_float4(acc[0].x, acc[1].x, acc[2].x, acc[3].x);
      *reinterpret_cast<float4*>(&s.sums[buffer][warp][2 * q + 1][4 * g]) = make_float4(acc[0].y, acc[1].y, acc[2].y, acc[3].y);
    }
    __syncthreads();                           // (and when all have come here again the other buffer has been read)
    if (warp < item.rows) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps4; ++w) v += s.sums[buffer][w][warp][lane];
      v = n0 + lane < p.J ? v / (1.f + expf(-v)) : 0.f;
      const uint32_t byte = fp4_scale(__reduce_max_sync(kAll, __float_as_uint(v) & 0x7fffffffu));
      const float y[8] = {fp4_scaled(v, fp4_inverse(byte))};
      const_cast<__half*>(to.row(item.slot[warp]))[n0 + lane] = __ushort_as_half(static_cast<unsigned short>(fp4_rounded(y).x));
      if (lane == 0) const_cast<float*>(to.scale(item.slot[warp]))[n0 / kTile4] = fp4_power(byte);
    }
  }
}

// A cluster has a tile of the output's columns, its warps the items' stages in turn; each warp adds up the tokens' outputs for itself, then they are joined.
template <typename T, int LAYOUT>
__global__ void __launch_bounds__(kThreads4, 2) few_down4_kernel(const __grid_constant__ LayerParams p, const __grid_constant__ Matrix4 t, const Rows4 x) {
  extern __shared__ __align__(16) float layer_smem[];
  __shared__ DownShared items;
  const int rank = cluster_rank(), size = cluster_size(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n0 = blockIdx.x / size * kTile4;
  if (size > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  float* part = layer_smem + kRing4 / 4;       // [warp][token][column]
  for (int i = tid; i < kWarps4 * p.tokens * kTile4; i += kThreads4) part[i] = 0.f;
  pdl_wait();
  pdl_trigger();
  for (int i = tid; i < p.tokens * p.k; i += kThreads4) {       // (items are no more than slots)
    items.item[i] = p.list->item[i];
    items.weights[i] = p.weights[i];
  }
  if (tid == 0) items.count = p.list->count;
  __syncthreads();
  const int stages = stages_of(p.J), all = items.count * stages, step = size * kWarps4;
  Stages<LAYOUT> ring(layer_smem, t);
  int coming = rank * kWarps4 + warp;
  auto next = [&]() {
    if (coming < all) {
      const int which = p.by_stages.quotient(coming);
      const Item& item = items.item[which];
      ring.begin(item.expert, n0, x, item.rows, [&](int m) { return static_cast<int>(item.slot[m]); });
      ring.ask(coming - which * stages);
      coming += step;
    } else {
      ring.store_late();
    }
    ring.asked();
  };
#pragma unroll 1
  for (int d = 0; d < kDepth4 - 1; ++d) next();
  const int g = lane >> 2, q = lane & 3;
  for (int i = rank * kWarps4 + warp; i < all; i += step) {
    const Item item = items.item[p.by_stages.quotient(i)];
    const int slot0 = item.slot[(q & 1) * 2], slot1 = item.slot[(q & 1) * 2 + 1];
    float2 acc[4] = {};
    next();
    ring.add(acc, item.rows);
    const float w0 = items.weights[slot0], w1 = items.weights[slot1];
    float4* to = reinterpret_cast<float4*>(part + (warp * p.tokens + p.by_k.quotient(slot0)) * kTile4 + 4 * g);
    if (q * 2 < item.rows) {
      const float4 o = *to;
      *to = make_float4(fmaf(w0, acc[0].x, o.x), fmaf(w0, acc[1].x, o.y), fmaf(w0, acc[2].x, o.z), fmaf(w0, acc[3].x, o.w));
    }
    to = reinterpret_cast<float4*>(part + (warp * p.tokens + p.by_k.quotient(slot1)) * kTile4 + 4 * g);
    if (q * 2 + 1 < item.rows) {
      const float4 o = *to;
      *to = make_float4(fmaf(w1, acc[0].y, o.x), fmaf(w1, acc[1].y, o.y), fmaf(w1, acc[2].y, o.z), fmaf(w1, acc[3].y, o.w));
    }
  }
  __syncthreads();
  put_out<T, kTile4>(p, part + kWarps4 * p.tokens * kTile4, n0, 0, [&](int t, int n, float4& v) {
#pragma unroll
    for (int w = 0; w < kWarps4; ++w) {
      const float4 y = *reinterpret_cast<const float4*>(part + (w * p.tokens + t) * kTile4 + n);
      v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
    }
  });
}

// ---- launches ----------------------------------------------------------------------------------------------------------
constexpr size_t kDownSmem = 218 * 1024, kHalfSmem = 104 * 1024;      // (227 KB an SM, of which static ones and a KB a CTA take some)

template <class... Params, class... Args>
cudaError_t launch_cluster(void (*kernel)(Params...), dim3 grid, unsigned block, unsigned cluster, size_t smem, cudaStream_t st, Args... args) {
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

// CTAs of a cluster, each with 32 contraction elements at least and an SM of its own: as many as leave room for all clusters at once.  (Of clusters of eight
// 15 fit, of seven as many, of six 22: clusters lie in processing clusters of 14 to 20 SMs.  16 tiles: a cluster that waits for the others took 5 us.)
unsigned cluster_of(int tiles, int J) {
  constexpr int kFit[] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
  unsigned size = 8;
  while (size > 1 && (tiles > kFit[size] || J / static_cast<int>(size) < 32)) --size;
  return size;
}

// Clusters for a tile: several where one leaves half of the SMs or more unused and there is enough to read to pay for another launch.  (us a call, one cluster
// and several: 19 tokens, 3 of 10 experts, 256 x 1792, 38.3 and 28.0; 8 tokens, 4 of 64, 512 x 2048, 41.1 and 37.5; 9 tokens, 2 of 22, 160 x 1760 in float32, 22.6 and 20.7; 4 tokens,
// 2 of 10, 128 x 960, which is less, 14.0 and 14.5.)
int splits_of(int tiles, const LayerParams& p) {
  const int experts = p.tokens * p.k < p.E ? p.tokens * p.k : p.E;
  if (static_cast<long long>(experts) * p.I * p.J < 2 << 20) return 1;
  int best = 1;
  unsigned most = tiles * cluster_of(tiles, p.J);
  for (int n = 2; n <= kMostSplits && most <= 74; ++n) {
    const unsigned ctas = tiles * n * cluster_of(tiles * n, p.J / (2 * n));      // (64 contraction elements a CTA at least)
    if (2 * ctas >= 3 * most) {
      most = ctas;
      best = n;
    }
  }
  return best;
}

template <auto kernel, typename T>
cudaError_t down_launch(LayerParams p, int tile, cudaStream_t st) {
  const int tiles = (p.I + tile - 1) / tile, slots = p.tokens * p.k;
  cudaError_t err = ensure_smem_optin<kernel>(static_cast<int>(kDownSmem));
  if (err != cudaSuccess) return err;
  p.splits = splits_of(tiles, p);
  const unsigned size = p.splits > 1 ? cluster_of(tiles * p.splits, p.J / (2 * p.splits)) : cluster_of(tiles, p.J);
  const size_t ring = static_cast<size_t>(p.ring_words) * 4;
  const size_t part = static_cast<size_t>((slots < 4 * kDownWarps ? 4 * kDownWarps : slots) + (size > 1 ? p.tokens : 0)) * tile * sizeof(float) + 4 * size * sizeof(float);
  size_t act = static_cast<size_t>(slots) * (p.J / (size * p.splits) + 36) * sizeof(float);
  act = (act + 15) & ~static_cast<size_t>(15);
  if (act > kDownSmem - part - ring) act = kDownSmem - part - ring;
  // What other CTAs write of their sums lies behind what this one lists its items with: they may be through before it has begun to.
  const size_t sums = ring + act + static_cast<size_t>(slots < 4 * kDownWarps ? 4 * kDownWarps : slots) * tile * sizeof(float);
  if (size > 1 && sums < sizeof(Scratch)) act += (sizeof(Scratch) - sums + 15) & ~static_cast<size_t>(15);
  p.act_floats = static_cast<int>(act / sizeof(float));
  count_launch(p.splits > 1 ? 2 : 1);
  const size_t smem = ring + act + part;       // (what the items are listed with lies at its begin first)
  err = launch_cluster(kernel, dim3(tiles * size, p.splits), kDownThreads, size, smem > sizeof(Scratch) ? smem : sizeof(Scratch), st, p);
  if (err != cudaSuccess || p.splits == 1) return err;
  return launch_kernel(few_join_kernel<T>, dim3(static_cast<unsigned>((static_cast<long long>(p.tokens) * p.I + 255) / 256)), 256, 0, st, true, p);
}

template <auto kernel>
cudaError_t up_launch(const LayerParams& p, cudaStream_t st) {
  cudaError_t err = ensure_smem_optin<kernel>(static_cast<int>(ring_bytes(kUpThreads, kUpDepth, 8)));
  if (err != cudaSuccess) return err;
  count_launch();
  return launch_kernel(kernel, dim3(kUpGrid), kUpThreads, static_cast<size_t>(p.ring_words) * 4, st, true, p);
}

bool on(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T>
void prepare(LayerParams* p) {
  constexpr int V = 16 / sizeof(T);
  p->x_vectors = p->I % V == 0 && p->x_row % V == 0 && on(p->X, 16) && on(p->router, 16);
  p->by_k = Div(p->k);
}

Layout4 layout4(const void* w, bool cn, long long row, long long far) {
  auto whole = [&](int n) { return row % n == 0 && far % n == 0 && on(w, n); };
  return !cn ? kNC : whole(16) ? kCN16 : whole(4) ? kCN4 : kCN1;
}
template <int LAYOUT>
cudaError_t up4_launch(const LayerParams& p, const Matrix4& t, const Rows4& x, const Rows4& to, cudaStream_t st) {
  cudaError_t err = ensure_smem_optin<few_up4_kernel<LAYOUT>>(static_cast<int>(kRing4));
  if (err != cudaSuccess) return err;
  count_launch();
  return launch_kernel(few_up4_kernel<LAYOUT>, dim3(kUpGrid), kThreads4, kRing4, st, true, p, t, x, to);
}
// CTAs of a cluster: as many as two an SM leave room for (33 clusters of eight, 71 of four, 148 of two), a stage for a warp at least; one an SM where the tokens' sums take
// more shared memory.
template <typename T, int LAYOUT>
cudaError_t down4_launch(LayerParams p, const Matrix4& t, const Rows4& x, cudaStream_t st) {
  const int tiles = (p.I + kTile4 - 1) / kTile4, turns = p.tokens * p.k * stages_of(p.J);
  const size_t smem = kRing4 + static_cast<size_t>(kWarps4 + 1) * p.tokens * kTile4 * sizeof(float) + 128;
  unsigned size = 8;
  if (smem > kHalfSmem) {
    size = cluster_of(tiles, 32 * 8);
  } else {
    while (size > 1 && tiles * size > 256) size /= 2;
  }
  while (size > 1 && turns <= static_cast<int>(size / 2) * kWarps4) size /= 2;
  p.splits = 1;
  cudaError_t err = ensure_smem_optin<few_down4_kernel<T, LAYOUT>>(static_cast<int>(kRing4 + (kWarps4 + 1) * 32 * kTile4 * sizeof(float) + 128));
  if (err != cudaSuccess) return err;
  count_launch();
  return launch_cluster(few_down4_kernel<T, LAYOUT>, dim3(tiles * size), kThreads4, size, smem, st, p, t, x);
}
template <typename T>
cudaError_t layer4_t(LayerParams p, const float* bias, const egs_route& route, bool up_cn, bool down_cn, const Rows4& x, const Rows4& h, cudaStream_t st) {
  prepare<T>(&p);
  const int logits_ctas = (p.E + 7) / 8;
  count_launch();
  cudaError_t err = launch_kernel(few_logits4_kernel<T>, dim3(logits_ctas + (fp4_blocks(p.I) + 31) / 32, (p.tokens + kRows - 1) / kRows), 128, 0, st, true, p, x, logits_ctas);
  if (err != cudaSuccess) return err;
  if ((err = launch_route_tokens(p.logits, bias, p.weights, p.experts, route, p.E, EGS_F32, st)) != cudaSuccess) return err;
  p.by_tiles = Div((p.J + kTile4 - 1) / kTile4);
  p.by_stages = Div(stages_of(p.J));
  auto words = [](const uint8_t* scale, long long row) { return row % 4 == 0 && on(scale, 4); };
  const Matrix4 up{static_cast<const uint8_t*>(p.up), p.up_scale, p.up_far, p.us_row * p.J, static_cast<uint32_t>(p.up_row), static_cast<uint32_t>(p.us_row), p.I, p.J, words(p.up_scale, p.us_row)};
  const Matrix4 down{static_cast<const uint8_t*>(p.down), p.down_scale, p.down_far, p.ds_row * p.I, static_cast<uint32_t>(p.down_row), static_cast<uint32_t>(p.ds_row), p.J, p.I, words(p.down_scale, p.ds_row)};
  switch (layout4(p.up, up_cn, p.up_row, p.up_far)) {
    case kNC: err = up4_launch<kNC>(p, up, x, h, st); break;
    case kCN16: err = up4_launch<kCN16>(p, up, x, h, st); break;
    case kCN4: err = up4_launch<kCN4>(p, up, x, h, st); break;
    default: err = up4_launch<kCN1>(p, up, x, h, st);
  }
  if (err != cudaSuccess) return err;
  switch (layout4(p.down, down_cn, p.down_row, p.down_far)) {
    case kNC: return down4_launch<T, kNC>(p, down, h, st);
    case kCN16: return down4_launch<T, kCN16>(p, down, h, st);
    case kCN4: return down4_launch<T, kCN4>(p, down, h, st);
    default: return down4_launch<T, kCN1>(p, down, h, st);
  }
}

template <typename T>
cudaError_t layer_t(LayerParams p, const float* bias, const egs_route& route, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T), kLanes = 8;
  prepare<T>(&p);
  count_launch();
  cudaError_t err = launch_kernel(few_logits_kernel<T>, dim3((p.E + 7) / 8, (p.tokens + kRows - 1) / kRows), 128, 0, st, true, p);
  if (err != cudaSuccess) return err;
  if ((err = launch_route_tokens(p.logits, bias, p.weights, p.experts, route, p.E, EGS_F32, st)) != cudaSuccess) return err;
  // One width for both products: the parts of `up` are counted by it.  16-byte vectors where rows begin on them.  Rows of whole vectors that do not, as a slice of a larger
  // buffer has them, are shifted together (8 tokens, 4 of 16 experts, 2048 x 512: 45 us, from 16 bytes on 32, and a copy of all experts' weights ahead of it 78).
  // So are rows of other widths in 16 bits from 128 Ki elements of an expert's matrix on; else they come element by element (us a call, shifted and not: 8 tokens, 2047 x 511, 62 and 102; 4 tokens, 500 x 301,
  // 18.8 and 19.5, 330 x 201, 18.0 and 16.9; 4 tokens in float32, 1001 x 500, 34.3 and 34.1).
  const bool whole = p.I % V == 0 && p.J % V == 0;
  const long long elements = static_cast<long long>(p.I) * p.J;
  if (whole || (sizeof(T) == 2 && elements >= 128 << 10)) {
    p.by_tiles = Div((p.J + V * kLanes - 1) / (V * kLanes));
    p.weight_bytes = p.E * elements * static_cast<long long>(sizeof(T));
    auto both = [&](auto up, auto down, int lanes) {
      p.ring_words = static_cast<int>(ring_bytes(kUpThreads, kUpDepth, lanes) / 4);
      if (cudaError_t e = up(); e != cudaSuccess) return e;
      p.ring_words = static_cast<int>(ring_bytes(kDownThreads, kDownDepth, lanes) / 4);
      return down();
    };
    if (!whole || !on(p.up, 16) || !on(p.down, 16)) {
      auto piece = [](const void*& w) {            // the 16 bytes that w lies in
        const uintptr_t behind = reinterpret_cast<uintptr_t>(w) & 15u;
        w = static_cast<const char*>(w) - behind;
        return static_cast<uint32_t>(behind / sizeof(T));
      };
      p.up_first = piece(p.up);
      p.down_first = piece(p.down);
      return both([&] { return up_launch<few_up_kernel<T, V, kLanes, true>>(p, st); }, [&] { return down_launch<few_down_kernel<T, V, kLanes, true>, T>(p, V * kLanes, st); }, kLanes);
    }
    return both([&] { return up_launch<few_up_kernel<T, V, kLanes, false>>(p, st); }, [&] { return down_launch<few_down_kernel<T, V, kLanes, false>, T>(p, V * kLanes, st); }, 0);
  }
  p.by_tiles = Div((p.J + 31) / 32);
  if ((err = up_launch<few_up_kernel<T, 1, 32, false>>(p, st)) != cudaSuccess) return err;
  return down_launch<few_down_kernel<T, 1, 32, false>, T>(p, 32, st);
}

}  // namespace

namespace {
size_t logits_words(const egs_route& r) { return (static_cast<size_t>(r.tokens) * r.E + 3) / 4 * 4; }
size_t rows4_bytes(long long rows, int C) { return static_cast<size_t>(rows) * (fp4_blocks(C) * 64 + stages_of(C) * 16); }
Rows4 rows4_at(void* from, long long rows, int C) {
  return {static_cast<__half*>(from), reinterpret_cast<float*>(static_cast<char*>(from) + static_cast<size_t>(rows) * fp4_blocks(C) * 64), C};
}
}  // namespace

size_t few_layer_workspace(const egs_route& r, int I, int J) {
  const long long slots = static_cast<long long>(r.tokens) * r.top_k;
  const size_t parts = static_cast<size_t>(kMostParts) * slots * J * sizeof(float), fp4 = rows4_bytes(r.tokens, I) + rows4_bytes(slots, J);
  const size_t sums = static_cast<size_t>(kMostSplits) * r.tokens * I * sizeof(float);
  return sizeof(Items) + logits_words(r) * sizeof(float) + (parts + sums > fp4 ? parts + sums : fp4);
}

cudaError_t launch_few_layer(const FewLayer& f, const egs_route& r, int dtype, void* workspace, cudaStream_t st) {
  LayerParams p{};
  p.X = f.X; p.router = f.router; p.up = f.up; p.down = f.down; p.up_scale = f.up_scale; p.down_scale = f.down_scale;
  p.out = f.out; p.weights = f.weights; p.experts = f.experts;
  p.list = static_cast<Items*>(workspace);
  p.logits = reinterpret_cast<float*>(p.list + 1);
  p.h = p.logits + logits_words(r);
  p.x_row = f.x_row;
  p.tokens = static_cast<int>(r.tokens); p.E = r.E; p.k = r.top_k; p.I = f.I; p.J = f.J;
  if (f.up_scale) {
    p.up_row = f.up_row; p.us_row = f.us_row; p.down_row = f.down_row; p.ds_row = f.ds_row;
    p.up_far = f.up_far; p.down_far = f.down_far;
    const Rows4 x = rows4_at(p.h, r.tokens, f.I), h = rows4_at(reinterpret_cast<char*>(p.h) + rows4_bytes(r.tokens, f.I), static_cast<long long>(p.tokens) * p.k, f.J);
    return dtype == EGS_F16 ? layer4_t<__half>(p, f.bias, r, f.up_cn, f.down_cn, x, h, st) : dtype == EGS_BF16 ? layer4_t<__nv_bfloat16>(p, f.bias, r, f.up_cn, f.down_cn, x, h, st) : layer4_t<float>(p, f.bias, r, f.up_cn, f.down_cn, x, h, st);
  }
  p.up_row = p.J;
  p.down_row = p.I;
  p.sums = p.h + static_cast<size_t>(kMostParts) * p.tokens * p.k * p.J;
  return dtype == EGS_F16 ? layer_t<__half>(p, f.bias, r, st) : dtype == EGS_BF16 ? layer_t<__nv_bfloat16>(p, f.bias, r, st) : layer_t<float>(p, f.bias, r, st);
}

}  // namespace egs
