// A whole routed layer for a few tokens: out[t] = sum over j of w[t, j] silu(x[t] up[e]) down[e], e the j-th expert that token t chose.  Its work is
// reading the weights of the experts that were chosen, each of them once, with all SMs.
//
//   choice   where tokens and router are few and small, in `up`: each cluster of CTAs forms the logits, each CTA makes the choice for itself; else two kernels,
//            the logits, in which a warp has two experts' rows of the router and four tokens, and egs_choice.cu's
//   up       units of (an expert's up to four tokens) x (a tile of columns) x (a part of the contraction) go round
//            the CTAs; float32 sums of parts.  The other product's weights are brought to the L2 meanwhile.
//   down     a cluster has a tile of the output's columns, its CTAs the contraction in parts; warps have the experts' tokens in turn.  The parts' sums
//            are joined, activated and weighted on the way into shared memory; a token's products are added in the order of its choices, the
//            CTAs' in theirs: the same bits in every run.
#include "egs_fp4.cuh"

namespace egs {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kMost = EGS_MAX_FEW_SLOTS, kRows = 4;      // slots; tokens that share a read of the weights
constexpr int kUpThreads = 256, kUpWarps = kUpThreads / 32, kUpGrid = 296, kUpPart = 1024;
constexpr int kUpCluster = 4;                // CTAs that form logits together (two SMs: clusters of eight leave SMs of a processing cluster without any)
constexpr int kDownThreads = 512, kDownWarps = kDownThreads / 32;
constexpr int kMostParts = 8;
constexpr int kFixedRows = 128, kFixedRows4 = 512;       // of a unit, in rows of its tile: 16 KB of weights

struct LayerList;
struct LayerParams {
  const void* X;
  const void* router;
  const float* bias;
  const void* up;            // [E, I, J], in 4 bits [E, J, I / 2]
  const void* down;          // [E, J, I], in 4 bits [E, I, J / 2]
  const uint8_t* up_scale;
  const uint8_t* down_scale;
  void* out;
  float* weights;
  int* experts;
  float* logits;
  float* h;                  // [parts][tokens * k][J]
  LayerList* list;    // what `up` has found out
  long long x_row, up_row, us_row, down_row, ds_row;       // elements; in 4 bits bytes
  long long up_far;          // in 4 bits: bytes from one expert of `up` to the next
  int tokens, E, k, I, J;
  int groups, top_groups, group_top, sigmoid, renormalize;
  float scale;
  int own_logits;            // `up` forms them
  int x_vectors;             // rows of X and of the router begin on 16 bytes and are whole 16 bytes
  long long down_far;        // bytes from one expert of `down` to the next
  int down_bytes;            // ... of one, to bring to the L2 ahead; 0: not
  int pieces;                // ... in so many pieces
  int ring_words;            // of weights on their way, in shared memory
  int act_floats;            // down: room for activations
  Div by_pieces, by_tiles, by_k, by_E4;
};

// An expert's tokens, up to four at a time.
struct alignas(16) Item {
  int expert, rows;
  short slot[kRows];
};
struct Items {
  Item item[kMost];
  int ids[kMost];
  unsigned tokens[EGS_MAX_EXPERTS];
  int first[EGS_MAX_EXPERTS];    // an expert's first item
  int count;
};
struct LayerList {
  int count, parts;              // items, parts that sums of `up` are in
  int pad[2];
  Item item[kMost];
};
// From the chosen experts (s->ids); by all threads, which have synchronised behind the ids and s->tokens = 0.
__device__ __forceinline__ void list_items(const LayerParams& p, Items* s) {
  const int tid = threadIdx.x, n = p.tokens * p.k;
  for (int i = tid; i < n; i += blockDim.x) atomicOr(&s->tokens[s->ids[i]], 1u << p.by_k.quotient(i));
  __syncthreads();
  if (tid < 32) {
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + tid, own = e < p.E ? (__popc(s->tokens[e]) + kRows - 1) / kRows : 0;
      int at = before;
#pragma unroll
      for (int bit = 0; bit < 4; ++bit) {        // (eight items at most)
        const unsigned has = __ballot_sync(kAll, own >> bit & 1);
        at += __popc(has & ((1u << tid) - 1u)) << bit;
        before += __popc(has) << bit;
      }
      if (e < p.E) s->first[e] = at;
    }
    if (tid == 0) s->count = before;
  }
  __syncthreads();
  for (int i = tid; i < n; i += blockDim.x) {
    const int e = s->ids[i];
    const unsigned tokens = s->tokens[e];
    const int place = __popc(tokens & ((1u << p.by_k.quotient(i)) - 1u)), rows = min(kRows, __popc(tokens) - place / kRows * kRows);
    Item& x = s->item[s->first[e] + place / kRows];
    x.slot[place % kRows] = static_cast<short>(i);
    if (place % kRows == 0) {
      x.expert = e;
      x.rows = rows;
      for (int r = rows; r < kRows; ++r) x.slot[r] = static_cast<short>(i);
    }
  }
  __syncthreads();
}

// Parts that the contraction of `up` is cut into: the fewest rounds of the CTAs, a unit costing as much as `fixed` rows beside its own.
__device__ __forceinline__ int parts_of(int units, int length, int fixed) {
  int best = 1, least = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = 1 << i, cost = (units * s + kUpGrid - 1) / kUpGrid * (((length + s - 1) >> i) + fixed);
    if (cost < least && (i == 0 || length >> i >= 64)) {
      least = cost;
      best = s;
    }
  }
  return best;
}

// ---- the choice -------------------------------------------------------------------------------------------------------
// Floats as unsigned numbers of the same order; NaN lies below everything and above 0, which stands for "no candidate".
__device__ __forceinline__ uint32_t ordered(float x) {
  x += 0.f;                                    // -0 and 0 are equal
  const uint32_t b = __float_as_uint(x);
  return x != x ? 1u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) { return k <= 1u ? __uint_as_float(0x7fc00000u) : __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// The choice as route_tokens_kernel defines it.  A warp forms a token's keys; logits, keys: shared memory.
struct Softmax {
  float m, total;
};
__device__ __forceinline__ float score_of(const LayerParams& p, const Softmax& soft, float x) {
  return p.sigmoid ? 1.f / (1.f + expf(-x)) : soft.m == -INFINITY ? 0.f : expf(x - soft.m) / soft.total;
}
__device__ __forceinline__ Softmax form_keys(const LayerParams& p, const float* logits, uint32_t* keys, int E4) {
  const int lane = threadIdx.x & 31;
  const bool pairs = p.groups > 1 && p.group_top == 2, scores = p.bias || pairs;
  Softmax soft{0.f, 1.f};
  if (!p.sigmoid && (scores || !p.renormalize)) {
    soft.m = -INFINITY;
    for (int e = lane; e < p.E; e += 32) soft.m = fmaxf(soft.m, logits[e]);
    soft.m = warp_max(soft.m);
    soft.total = 0.f;
    for (int e = lane; e < p.E; e += 32) soft.total += soft.m == -INFINITY ? 0.f : expf(logits[e] - soft.m);
    soft.total = warp_sum(soft.total);
  }
  for (int e = lane; e < E4; e += 32) {
    const float x = e < p.E ? logits[e] : 0.f;
    keys[e] = e >= p.E ? 0u : ordered(!scores ? x : p.bias ? score_of(p, soft, x) + p.bias[e] : score_of(p, soft, x));
  }
  __syncwarp();
  if (p.groups > 1) {
    const int per = p.E / p.groups;
    uint32_t value = 0u;                       // of lane's group
    if (lane < p.groups) {
      uint32_t k1 = 0u, k2 = 0u;
      for (int i = 0; i < per; ++i) {
        const uint32_t v = keys[lane * per + i];
        k2 = max(k2, min(k1, v));
        k1 = max(k1, v);
      }
      value = pairs && k2 ? ordered(unordered(k1) + unordered(k2)) : k1;
    }
    unsigned kept = 0u;
    for (int i = 0; i < p.top_groups; ++i) {
      const int at = __ffs(__ballot_sync(kAll, value == __reduce_max_sync(kAll, value))) - 1;
      kept |= 1u << at;
      if (lane == at) value = 0u;
    }
    __syncwarp();
    for (int e = lane; e < p.E; e += 32) keys[e] = !(kept >> (e / per) & 1u) ? 0u : p.bias ? keys[e] : ordered(logits[e]);
    __syncwarp();
  }
  return soft;
}
// Many experts: the k highest keys one after the other, by a warp.
__device__ __forceinline__ void choose_in_turn(const LayerParams& p, uint32_t* keys, int* ids) {
  const int lane = threadIdx.x & 31;
  uint32_t best = 0u;                          // of this lane's experts
  int who = 0;
  auto look = [&]() {
    best = 0u;
    for (int e = lane; e < p.E; e += 32)
      if (keys[e] > best) {
        best = keys[e];
        who = e;
      }
  };
  look();
  for (int j = 0; j < p.k; ++j) {
    const uint32_t top = __reduce_max_sync(kAll, best);
    const int e = __reduce_min_sync(kAll, best == top && top ? who : 0x7fffffff);
    if (lane == j) ids[j] = e;
    if (best == top && who == e) {
      keys[e] = 0u;
      look();
    }
  }
}
// Few: a thread counts the keys before its expert's (equal ones: those of lower experts).
constexpr int kCounted = 256;
__device__ __forceinline__ void choose_by_count(const LayerParams& p, const uint32_t* keys, int tokens, int E4, int* ids) {
  for (int i = threadIdx.x; i < tokens * E4; i += kUpThreads) {
    const int w = p.by_E4.quotient(i), e = i - w * E4;
    const uint32_t* row = keys + w * E4;
    const uint32_t key = row[e];
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < E4; j += 4) {          // (no key is 2^32 - 1, and there are zeros behind the last one)
      const uint4 other = *reinterpret_cast<const uint4*>(row + j);
      before += other.x + (j < e) > key;
      before += other.y + (j + 1 < e) > key;
      before += other.z + (j + 2 < e) > key;
      before += other.w + (j + 3 < e) > key;
    }
    if (key && before < p.k) ids[w * p.k + before] = e;
  }
}
// A token's weights, lane j < k has the j-th.
__device__ __forceinline__ float weight_of(const LayerParams& p, const Softmax& soft, const float* logits, const int* ids) {
  const int lane = threadIdx.x & 31;
  const bool chosen = lane < p.k;
  const float x = chosen ? logits[ids[lane]] : -INFINITY;
  if (!p.renormalize) return score_of(p, soft, x) * p.scale;
  const float high = p.sigmoid ? 0.f : warp_max(x);
  const float s = !chosen ? 0.f : p.sigmoid ? score_of(p, soft, x) : high == -INFINITY ? 0.f : expf(x - high);
  const float sum = warp_sum(s);
  return (sum == 0.f ? 0.f : s / sum) * p.scale;
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
__device__ __forceinline__ uint32_t in_cta(const void* mine, int rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
  return at;
}
__device__ __forceinline__ float of_cta(const float* mine, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(in_cta(mine, rank)) : "memory");
  return v;
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
// ... by a warp for tokens from t0 to t1, in fours: emit(token, expert, logit)
template <typename T, class Emit>
__device__ __forceinline__ void logits_of(const LayerParams& p, int e0, int e1, int t0, int t1, Emit&& emit) {
  constexpr int V = 16 / sizeof(T);
  for (; t0 < t1; t0 += kRows) {
    if (t1 - t0 == 1) {
      float acc[2][1];
      if (p.x_vectors) dots<T, V, 1, 8>(p, e0, e1, t0, acc);
      else dots<T, 1, 1, 16>(p, e0, e1, t0, acc);
      emit(t0, e0, acc[0][0]);
      if (e1 < p.E) emit(t0, e1, acc[1][0]);
    } else {
      float acc[2][kRows];
      if (p.x_vectors) dots<T, V, kRows, 2>(p, e0, e1, t0, acc);
      else dots<T, 1, kRows, 8>(p, e0, e1, t0, acc);
#pragma unroll
      for (int m = 0; m < kRows; ++m)
        if (t0 + m < t1) {
          emit(t0 + m, e0, acc[0][m]);
          if (e1 < p.E) emit(t0 + m, e1, acc[1][m]);
        }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(128) few_logits_kernel(const __grid_constant__ LayerParams p) {
  pdl_wait();
  pdl_trigger();
  const int e = (blockIdx.x * 4 + (threadIdx.x >> 5)) * 2, lane = threadIdx.x & 31, t0 = blockIdx.y * kRows;
  if (e >= p.E) return;
  logits_of<T>(p, e, e + 1, t0, min(p.tokens, t0 + kRows), [&](int t, int expert, float v) {
    if (lane == 0) p.logits[t * p.E + expert] = v;
  });
}

// The other product's weights to the L2, in pieces that go round the CTAs.
__device__ __forceinline__ void bring_down(const LayerParams& p, const Items& items) {
  constexpr int kPiece = 8192;
  for (int i = blockIdx.x + threadIdx.x * gridDim.x; i < items.count * p.pieces; i += kUpThreads * gridDim.x) {
    const int which = p.by_pieces.quotient(i), from = (i - which * p.pieces) * kPiece;
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(static_cast<const char*>(p.down) + items.item[which].expert * p.down_far + from), "r"(min(kPiece, p.down_bytes - from)) : "memory");
  }
}

// What both `up` kernels begin with: logits and the choice (or that which is there), the items, the parts; the CTAs of a cluster share the logits.
// table: 2 * 8 rows of E4 words, logits and keys.  `tiles`: of columns.
template <typename T>
__device__ __forceinline__ int begin_layer(const LayerParams& p, Items* s, uint32_t* table, int tiles, int fixed) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, E4 = p.by_E4.d;
  float* logits = reinterpret_cast<float*>(table);
  uint32_t* keys = table + kUpWarps * E4;
  if (p.own_logits) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  pdl_trigger();
  for (int e = tid; e < p.E; e += kUpThreads) s->tokens[e] = 0u;
  if (p.own_logits) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");        // all CTAs of the cluster have begun
    constexpr int kAll8 = kUpCluster * kUpWarps;
    for (int e = cluster_rank() * kUpWarps + warp; e < p.E; e += 2 * kAll8)
      logits_of<T>(p, e, e + kAll8, 0, p.tokens, [&](int t, int expert, float v) {
        if (lane < kUpCluster) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(in_cta(logits + t * E4 + expert, lane)), "f"(v) : "memory");
      });
    cluster_sync();
  }
  if (p.own_logits) {
    const int t = warp;
    float* row = logits + warp * E4;
    Softmax soft{};
    if (t < p.tokens) {
      soft = form_keys(p, row, keys + warp * E4, E4);
      if (p.E > kCounted) choose_in_turn(p, keys + warp * E4, s->ids + t * p.k);
    }
    __syncthreads();
    if (p.E <= kCounted) {
      choose_by_count(p, keys, p.tokens, E4, s->ids);
      __syncthreads();
    }
    if (blockIdx.x == 0 && t < p.tokens) {
      const float w = weight_of(p, soft, row, s->ids + t * p.k);
      if (lane < p.k) {
        p.weights[t * p.k + lane] = w;
        p.experts[t * p.k + lane] = s->ids[t * p.k + lane];
      }
    }
  } else {
    for (int i = tid; i < p.tokens * p.k; i += kUpThreads) s->ids[i] = p.experts[i];
    __syncthreads();
  }
  list_items(p, s);
  const int parts = parts_of(s->count * tiles, p.I, fixed);
  if (blockIdx.x == 0) {
    for (int i = tid; i < s->count; i += kUpThreads) p.list->item[i] = s->item[i];
    if (tid == 0) {
      p.list->count = s->count;
      p.list->parts = parts;
    }
  }
  return parts;
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
  __device__ __forceinline__ void set(int v, float a, float b) {          // of v and v + 1
    raw[v / 2] = pair(a, b);
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
// Weights on their way to shared memory, kDepth pieces of 64 bytes a thread, each thread's its own: what it asked for it reads, so that nobody waits for
// others, and the next unit's weights come while this one's sums are joined.  (Into registers, with a wait for all that had been asked for before
// more was, 43 MB came at 3.4 TB/s.)
template <int THREADS, int DEPTH>
struct Ring {
  uint32_t base;
  int slot = 0;
  __device__ __forceinline__ explicit Ring(const void* smem) : base(static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16u) {}
  __device__ __forceinline__ uint32_t at(int r) const { return base + static_cast<uint32_t>(slot * 4 + r) * (THREADS * 16u); }
  __device__ __forceinline__ void ask(int r, const void* from, bool there) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at(r)), "l"(from), "r"(there ? 16 : 0) : "memory");
  }
  __device__ __forceinline__ void asked() {        // (the slot that has been read is the one that is asked for anew)
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++slot == DEPTH) slot = 0;
  }
  __device__ __forceinline__ void wait() const { asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory"); }
  template <class P>
  __device__ __forceinline__ P get(int r) const {
    static_assert(sizeof(P) == 16, "pieces are of 16 bytes");
    union {
      uint4 raw;
      P value;
    } x{};
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.raw.x), "=r"(x.raw.y), "=r"(x.raw.z), "=r"(x.raw.w) : "r"(at(r)) : "memory");
    return x.value;
  }
};
// Four rows of weights times M rows of the other operand at x.
template <typename T, int V, int M, class R>
__device__ __forceinline__ void add_four(Sums<V> (&acc)[M], const R& ring, const float* const (&a)[M], int at) {
  Packed<T, V> w[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) w[r] = ring.template get<Packed<T, V>>(r);
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
__host__ __device__ constexpr int ahead_of(int V) { return V >= 4 ? 2 : 4; }

template <typename T, int V, int LANES>
struct UpShared {
  Items items;
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
        if (c < c1) add_four<T, V, M>(acc, ring, a, c - c0);
        next();
      }
    } else {
      accumulate<T, V, M, ahead_of(V)>(acc, W, static_cast<int>(p.up_row), first, kStep, c1, n < p.J, a, c0, stage);
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
constexpr size_t ring_bytes(int threads, int depth) { return static_cast<size_t>(threads) * depth * 64; }

template <typename T, int V, int LANES>
__global__ void __launch_bounds__(kUpThreads, 2) few_up_kernel(const __grid_constant__ LayerParams p) {
  constexpr int kTile = LANES * V, kStep = kUpThreads / LANES * 4;
  constexpr bool kRing = V == 16 / sizeof(T);
  extern __shared__ __align__(16) uint32_t layer_table[];
  __shared__ UpShared<T, V, LANES> s;
  const int parts = begin_layer<T>(p, &s.items, layer_table + p.ring_words, p.by_tiles.d, kFixedRows), all = s.items.count * p.by_tiles.d, units = all * parts, length = ((p.I + parts - 1) / parts + 3) & ~3;
  Ring<kUpThreads, kUpDepth> ring(layer_table);
  // what is asked for next: rows c .. c + 3 of unit `coming`
  int coming = blockIdx.x, c = 0, end = 0, left = 0;
  bool on = false;
  const T* from = static_cast<const T*>(p.up);
  auto next = [&]() {
    if (left == 0 && coming < units) {
      const UpUnit x = up_unit_of(p, coming, all, length, p.I, kTile);
      const int n = x.n0 + threadIdx.x % LANES * V;
      on = n < p.J;
      c = x.begin + threadIdx.x / LANES * 4;
      end = x.end;
      left = (x.end - x.begin + kStep - 1) / kStep;
      from = static_cast<const T*>(p.up) + s.items.item[x.item].expert * (p.up_row * p.I) + c * p.up_row + n;
      coming += gridDim.x;
    }
    if (left) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool there = on && c + r < end;
        ring.ask(r, there ? from + r * p.up_row : static_cast<const T*>(p.up), there);
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
  bring_down(p, s.items);
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const UpUnit x = up_unit_of(p, u, all, length, p.I, kTile);
    float* to = p.h + static_cast<long long>(x.part) * p.tokens * p.k * p.J;
    const int rows = s.items.item[x.item].rows;
    if (rows == 1) up_unit<T, V, LANES, 1>(p, &s, x, to, ring, next);
    else if (rows == 2) up_unit<T, V, LANES, 2>(p, &s, x, to, ring, next);
    else up_unit<T, V, LANES, kRows>(p, &s, x, to, ring, next);
  }
}

// What `up` has found out, and the weights, in shared memory.
struct DownShared {
  Item item[kMost];
  float weights[kMost];
  int count, parts;
};
__device__ __forceinline__ void begin_down(const LayerParams& p, DownShared* s) {
  const int tid = threadIdx.x, slots = p.tokens * p.k;       // (items are no more than slots)
  if (tid < slots) {
    s->item[tid] = p.list->item[tid];
    s->weights[tid] = p.weights[tid];
  }
  if (tid == 0) {
    s->count = p.list->count;
    s->parts = p.list->parts;
  }
  __syncthreads();
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

// out[t, n0 + n] from the slots' products, part [shares][slots][tile].  Every CTA of a cluster has a share of the outputs, and the others hand it their
// sums: to, room for them, [CTAs][outputs of a share] of shared memory.
template <typename T, int TILE>
__device__ __forceinline__ void put_out(const LayerParams& p, const float* part, float* to, int shares, int n0) {
  const int slots = p.tokens * p.k, rank = cluster_rank(), size = cluster_size(), all = p.tokens * TILE, own = all / size;
  if (size > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // all have begun
  for (int i = threadIdx.x * 4; i < all; i += kDownThreads * 4) {
    const int t = i / TILE, n = i % TILE;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < p.k * shares; ++j) {
      const int choice = shares == 1 ? j : j / shares, s = j - choice * shares;
      const float4 x = *reinterpret_cast<const float4*>(part + (s * slots + t * p.k + choice) * TILE + n);
      v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    }
    if (size == 1) {
      T* out = static_cast<T*>(p.out) + static_cast<long long>(t) * p.I + n0 + n;
      if (n0 + n < p.I) out[0] = from_f32<T>(v.x);
      if (n0 + n + 1 < p.I) out[1] = from_f32<T>(v.y);
      if (n0 + n + 2 < p.I) out[2] = from_f32<T>(v.z);
      if (n0 + n + 3 < p.I) out[3] = from_f32<T>(v.w);
    } else {
      const int owner = i / own;               // (shares are whole fours: a tile has at least 32 columns, a cluster eight CTAs)
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(in_cta(to + rank * own + i - owner * own, owner)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
    }
  }
  if (size == 1) return;
  cluster_sync();
  for (int i = threadIdx.x; i < own; i += kDownThreads) {
    const int x = rank * own + i, t = x / TILE, n = x % TILE;
    float v = to[i];
    for (int r = 1; r < size; ++r) v += to[r * own + i];
    if (n0 + n < p.I) static_cast<T*>(p.out)[static_cast<long long>(t) * p.I + n0 + n] = from_f32<T>(v);
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
      if (c < end) add_four<T, V, M>(acc, ring, a, c - base);
      next();
    }
  } else {
    accumulate<T, V, M, ahead_of(V)>(acc, static_cast<const T*>(p.down) + item.expert * (p.down_row * p.J) + n, static_cast<int>(p.down_row), begin + lane / LANES * 4, kStep, end, n < p.I, a, base, []() {});
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

template <typename T, int V, int LANES>
__global__ void __launch_bounds__(kDownThreads, 1) few_down_kernel(const __grid_constant__ LayerParams p) {
  constexpr int kTile = LANES * V, kStep = 32 / LANES * 4;
  constexpr bool kRing = V == 16 / sizeof(T);
  extern __shared__ __align__(16) float layer_smem[];
  __shared__ DownShared items;
  if (cluster_size() > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  pdl_trigger();
  begin_down(p, &items);
  const int slots = p.tokens * p.k, rank = cluster_rank(), size = cluster_size(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n0 = blockIdx.x / size * kTile;
  float* act = layer_smem + p.ring_words;
  float* part = act + p.act_floats;
  const int parts = items.parts;
  const int length = ((p.J + size - 1) / size + 3) & ~3, begin = min(p.J, rank * length), end = min(p.J, begin + length);
  const int room = min(length, p.act_floats / slots & ~3);
  int shares_log2 = 0;                         // warps that have an item's contraction in turn
  while (items.count << (shares_log2 + 1) <= kDownWarps && length >> shares_log2 >= 64) ++shares_log2;
  const int turns = items.count << shares_log2;
  Ring<kDownThreads, kDownDepth> ring(layer_smem);
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
    auto next = [&]() {
      while (left == 0 && coming < turns) {
        const int b = share_of(coming, &stop);
        c = b + lane / LANES * 4;
        left = (stop - b + kStep - 1) / kStep;
        from = static_cast<const T*>(p.down) + items.item[coming >> shares_log2].expert * (p.down_row * p.J) + c * p.down_row + n0 + lane % LANES * V;
        coming += kDownWarps;
      }
      if (left) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool there = on && c + r < stop;
          ring.ask(r, there ? from + r * p.down_row : static_cast<const T*>(p.down), there);
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
    // activations, four at a time; the first weights are on their way meanwhile
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
  put_out<T, kTile>(p, part, part + max(4 * kDownWarps, slots) * kTile, 1 << shares_log2, n0);
}

// ---- weights in 4 bits -------------------------------------------------------------------------------------------------
// Four columns of an expert times M rows, a block of 32 contraction elements at a time: the weights' bytes lie along the contraction (NC, a lane has 16 of a column) or along
// the columns (CN, a lane has four of each of 16 rows, or one where rows begin anywhere).  Twice the values are integers, so that a block's sum is exact.
constexpr int kTile4 = 64;                     // NC: columns of a tile
__host__ __device__ constexpr int tile4(int layout) { return layout == 0 ? kTile4 : layout == 4 ? 128 : 32; }      // layout: 0 NC, 4 or 1 CN with so many columns a lane
constexpr int kColumns = 4;
struct Weights4 {
  Block4 w[kColumns];
  uint32_t s[kColumns];
};
struct Matrix4 {
  const uint8_t *w, *s;        // of an expert
  uint32_t row, s_row;         // NC: bytes from one column to the next, CN: from one pair of contraction elements to the next; scales: from one column to the next
  int C, N;
};

// acc[j][m] += the block's products; a[m]: twice the rows' 4 bits as bytes, f[m]: a quarter of their scale.
template <int M, int COLUMNS>
__device__ __forceinline__ void add_block(const Weights4& x, const uint8_t* const (&a)[M], const float (&f)[M], float (&acc)[COLUMNS][M]) {
  uint32_t y[M][8];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 z = *reinterpret_cast<const uint4*>(a[m] + h * 16);
      y[m][4 * h] = z.x; y[m][4 * h + 1] = z.y; y[m][4 * h + 2] = z.z; y[m][4 * h + 3] = z.w;
    }
#pragma unroll
  for (int j = 0; j < COLUMNS; ++j) {
    int sum[M];
#pragma unroll
    for (int m = 0; m < M; ++m) sum[m] = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      uint32_t low, high;
      fp4_integers(x.w[j].w[h], low, high);
#pragma unroll
      for (int m = 0; m < M; ++m) sum[m] = __dp4a(static_cast<int>(y[m][2 * h + 1]), static_cast<int>(high), __dp4a(static_cast<int>(y[m][2 * h]), static_cast<int>(low), sum[m]));
    }
    const float power = fp4_power(x.s[j]);
#pragma unroll
    for (int m = 0; m < M; ++m) acc[j][m] = fmaf(static_cast<float>(sum[m]) * f[m], power, acc[j][m]);
  }
}

// CN: a block of four columns from n on; the words of four rows become four columns' words.
template <int V>
__device__ __forceinline__ void load_columns(Weights4& x, const Matrix4& t, int n, int b) {
  const bool there = n < t.N;
  const uint8_t* from = t.w + static_cast<unsigned long long>(b * 16) * t.row + n;
  const int rows = min(16, t.C / 2 - b * 16);
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if constexpr (V == 4) r[i] = there && i < rows ? *reinterpret_cast<const uint32_t*>(from + static_cast<unsigned long long>(i) * t.row) : 0u;
    else r[i] = there && i < rows ? from[static_cast<unsigned long long>(i) * t.row] : 0u;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) x.s[j] = n + j < t.N ? t.s[static_cast<unsigned long long>(n + j) * t.s_row + b] : 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t p0 = __byte_perm(r[4 * i], r[4 * i + 1], 0x5140), p1 = __byte_perm(r[4 * i + 2], r[4 * i + 3], 0x5140);
    x.w[0].w[i] = __byte_perm(p0, p1, 0x5410);
    if constexpr (V == 4) {
      const uint32_t p2 = __byte_perm(r[4 * i], r[4 * i + 1], 0x7362), p3 = __byte_perm(r[4 * i + 2], r[4 * i + 3], 0x7362);
      x.w[1].w[i] = __byte_perm(p0, p1, 0x7632);
      x.w[2].w[i] = __byte_perm(p2, p3, 0x5410);
      x.w[3].w[i] = __byte_perm(p2, p3, 0x7632);
    }
  }
}
// Columns n .. n + V - 1 of a lane over the blocks begin, begin + step, .. below end.  `ready` is called when the first weights have been asked for.
template <int V, int M, class Ready>
__device__ __forceinline__ void along_columns(const Matrix4& t, int n, int begin, int step, int end, const uint8_t* const (&a)[M], const float* const (&f)[M], int base, float (&acc)[V][M], Ready&& ready) {
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[j][m] = 0.f;
  Weights4 next;
  if (begin < end) load_columns<V>(next, t, n, begin);
  ready();
  for (int b = begin; b < end; b += step) {
    const Weights4 now = next;
    if (b + step < end) load_columns<V>(next, t, n, b + step);
    const uint8_t* at[M];
    float g[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      at[m] = a[m] + (b - base) * 32;
      g[m] = f[m][b - base];
    }
    add_block<M, V>(now, at, g, acc);
  }
}

// NC: columns [n0, n0 + columns), blocks [begin, end).  Lanes go along the blocks, 4 to 32 of them; those that are left have other columns, four at a time.
// emit(column, row, sum) by the lanes that have the sums.
template <int M, class Ready, class Emit>
__device__ __forceinline__ void along_rows(const Matrix4& t, int n0, int columns, int begin, int end, const uint8_t* const (&a)[M], const float* const (&f)[M], int base, Ready&& ready, Emit&& emit) {
  int log2 = 2;
  while (log2 < 5 && (1 << log2) < end - begin) ++log2;
  const int lane = threadIdx.x & 31, along = lane & ((1 << log2) - 1), group = lane >> log2, groups = 32 >> log2;
  Weights4 next;
  auto load = [&](int first, int b) {
#pragma unroll
    for (int j = 0; j < kColumns; ++j) {
      const int n = n0 + first + j * groups + group;
      const bool there = first + j * groups < columns && n < t.N && b < end;
      next.w[j] = there ? load_block(t.w + static_cast<unsigned long long>(n) * t.row, b, t.C) : Block4{};
      next.s[j] = there ? t.s[static_cast<unsigned long long>(n) * t.s_row + b] : 0u;
    }
  };
  int first = 0, b = begin + along;            // of the weights that come next
  load(first, b);
  ready();
  while (first < columns) {
    float acc[kColumns][M];
#pragma unroll
    for (int j = 0; j < kColumns; ++j)
#pragma unroll
      for (int m = 0; m < M; ++m) acc[j][m] = 0.f;
    const int now_first = first;
    for (int steps = max(1, (end - begin + (1 << log2) - 1) >> log2); steps; --steps) {
      const Weights4 now = next;
      const int at_block = max(min(b, end - 1) - base, 0);
      const bool on = b < end;
      b += 1 << log2;
      if (steps == 1) {
        first += kColumns * groups;
        b = begin + along;
      }
      if (first < columns) load(first, b);
      const uint8_t* at[M];
      float g[M];
#pragma unroll
      for (int m = 0; m < M; ++m) {
        at[m] = a[m] + at_block * 32;
        g[m] = on ? f[m][at_block] : 0.f;
      }
      add_block<M, kColumns>(now, at, g, acc);
    }
    for (int o = 1; o < 1 << log2; o <<= 1)
#pragma unroll
      for (int j = 0; j < kColumns; ++j)
#pragma unroll
        for (int m = 0; m < M; ++m) acc[j][m] += __shfl_xor_sync(kAll, acc[j][m], o);
#pragma unroll
    for (int j = 0; j < kColumns; ++j) {
      const int c = now_first + j * groups;
      if (along == 0 && c < columns && n0 + c + group < t.N) {
#pragma unroll
        for (int m = 0; m < M; ++m) emit(n0 + c + group, m, acc[j][m]);
      }
    }
  }
}

// Eight of a block's 32 values by each of four neighbouring lanes, in 4 bits, as twice their values in bytes; a quarter of the block's scale.
__device__ __forceinline__ float block4(const float (&v)[8], uint8_t* to) {
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
  if (to) {
    uint2 w;
    fp4_integers(fp4_pack8(x), w.x, w.y);
    *reinterpret_cast<uint2*>(to) = w;
  }
  return 0.25f * fp4_power(byte);
}

constexpr int kUpBlocks = 2 * kUpPart / kFp4Block;       // blocks in shared memory at a time
template <int LAYOUT>
struct Up4Shared {
  Items items;
  alignas(16) uint8_t x[kRows][2 * kUpPart];
  float f[kRows][kUpBlocks];
  float sums[LAYOUT ? kUpWarps : 1][kRows][LAYOUT ? tile4(LAYOUT) : 1];
};

// An item's rows of X, blocks [b0, b0 + n), into shared memory; by all threads.
template <typename T>
__device__ __noinline__ void stage_rows4(const LayerParams& p, const Item& item, int rows, int b0, int n, uint8_t* x, float* f) {
  constexpr int kVec = 16 / sizeof(T);
  __syncthreads();                             // what was in shared memory has been read
  for (int m = 0; m < rows; ++m) {
    const T* from = static_cast<const T*>(p.X) + p.by_k.quotient(item.slot[m]) * p.x_row;
    for (int i0 = 0; i0 < n * 4; i0 += kUpThreads) {       // (whole warps)
      const int i = i0 + threadIdx.x, c = b0 * 32 + i * 8;
      const bool there = i < n * 4;
      float v[8];
      if (p.x_vectors && there && c + 8 <= p.I) {
#pragma unroll
        for (int h = 0; h < 8 / kVec; ++h) {
          const Packed<T, kVec> y = reinterpret_cast<const Packed<T, kVec>*>(from + c)[h];
#pragma unroll
          for (int j = 0; j < kVec; ++j) v[h * kVec + j] = y.get(j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = there && c + j < p.I ? to_f32<T>(from[c + j]) : 0.f;
      }
      const float g = block4(v, there ? x + m * (2 * kUpPart) + i * 8 : nullptr);
      if (there && i % 4 == 0) f[m * kUpBlocks + i / 4] = g;
    }
  }
  __syncthreads();
}

template <typename T, int LAYOUT, int M>
__device__ __forceinline__ void up4_unit(const LayerParams& p, Up4Shared<LAYOUT>* s, const Item& item, int n0, int begin, int end, float* to) {
  const int tid = threadIdx.x, warp = tid >> 5;
  const Matrix4 t{static_cast<const uint8_t*>(p.up) + item.expert * p.up_far, p.up_scale + item.expert * (p.us_row * p.J), static_cast<uint32_t>(p.up_row), static_cast<uint32_t>(p.us_row), (p.I + 1) / 2 * 2, p.J};
  const uint8_t* a[M];
  const float* f[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    a[m] = s->x[m];
    f[m] = s->f[m];
  }
  for (int b0 = begin; b0 < end; b0 += kUpBlocks) {
    const int b1 = min(end, b0 + kUpBlocks);
    const bool first = b0 == begin;
    auto stage = [&]() { stage_rows4<T>(p, item, M, b0, b1 - b0, s->x[0], s->f[0]); };
    auto put = [&](int col, int m, float v) {
      if (m >= item.rows || col >= p.J) return;
      float* o = to + static_cast<long long>(item.slot[m]) * p.J + col;
      *o = first ? v : *o + v;
    };
    if constexpr (LAYOUT == 0) {
      along_rows<M>(t, n0 + warp * (kTile4 / kUpWarps), kTile4 / kUpWarps, b0, b1, a, f, b0, stage, put);
    } else {
      constexpr int kTile = tile4(LAYOUT);
      const int n = (tid & 31) * LAYOUT;
      float acc[LAYOUT][M];
      along_columns<LAYOUT, M>(t, n0 + n, b0 + warp, kUpWarps, b1, a, f, b0, acc, stage);
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int j = 0; j < LAYOUT; ++j) s->sums[warp][m][n + j] = acc[j][m];
      __syncthreads();
      for (int i = tid; i < M * kTile; i += kUpThreads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kUpWarps; ++w) v += s->sums[w][i / kTile][i % kTile];
        put(n0 + i % kTile, i / kTile, v);
      }
    }
  }
}

template <typename T, int LAYOUT>
__global__ void __launch_bounds__(kUpThreads, 2) few_up4_kernel(const __grid_constant__ LayerParams p) {
  constexpr int kTile = tile4(LAYOUT);
  extern __shared__ uint32_t layer_table[];
  __shared__ Up4Shared<LAYOUT> s;
  const int tiles = p.by_tiles.d, parts = begin_layer<T>(p, &s.items, layer_table, tiles, kFixedRows4 * kTile4 / kTile), all = s.items.count * tiles, blocks = fp4_blocks(p.I), length = (blocks + parts - 1) / parts;
  bring_down(p, s.items);
  for (int u = blockIdx.x; u < all * parts; u += gridDim.x) {
    const int part = u / all, x = u - part * all, i = p.by_tiles.quotient(x), n0 = (x - i * tiles) * kTile, begin = min(blocks, part * length), end = min(blocks, begin + length);
    const Item item = s.items.item[i];
    float* to = p.h + static_cast<long long>(part) * p.tokens * p.k * p.J;
    if (begin == end) {                        // (nothing is left for the last parts of a short contraction)
      for (int c = threadIdx.x; c < item.rows * kTile; c += kUpThreads)
        if (n0 + c % kTile < p.J) to[static_cast<long long>(item.slot[c / kTile]) * p.J + n0 + c % kTile] = 0.f;
    } else if (item.rows == 1) {
      up4_unit<T, LAYOUT, 1>(p, &s, item, n0, begin, end, to);
    } else if (item.rows == 2) {
      up4_unit<T, LAYOUT, 2>(p, &s, item, n0, begin, end, to);
    } else {
      up4_unit<T, LAYOUT, kRows>(p, &s, item, n0, begin, end, to);
    }
  }
}

template <int LAYOUT, int M, class Ready>
__device__ __forceinline__ void down4_item(const LayerParams& p, const Item& item, const uint8_t* act, const float* scale, int pitch, int b0, int b1, int n0, int share, int shares, float* part,
                                           bool first, Ready&& ready) {
  constexpr int kTile = tile4(LAYOUT);
  const Matrix4 t{static_cast<const uint8_t*>(p.down) + item.expert * p.down_far, p.down_scale + item.expert * (p.ds_row * p.I), static_cast<uint32_t>(p.down_row), static_cast<uint32_t>(p.ds_row), (p.J + 1) / 2 * 2, p.I};
  const uint8_t* a[M];
  const float* f[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    a[m] = act + item.slot[m] * pitch * 32;
    f[m] = scale + item.slot[m] * pitch;
  }
  auto put = [&](float* row, int m, float v) {
    if (m >= item.rows) return;
    float* o = row + item.slot[m] * kTile;
    *o = first ? v : *o + v;
  };
  if constexpr (LAYOUT == 0) {                 // (shares: of the columns)
    const int columns = kTile / shares;
    along_rows<M>(t, n0 + share * columns, columns, b0, b1, a, f, b0, ready, [&](int col, int m, float v) { put(part + col - n0, m, v); });
  } else {                                     // (of the blocks)
    const int n = (threadIdx.x & 31) * LAYOUT;
    float acc[LAYOUT][M];
    along_columns<LAYOUT, M>(t, n0 + n, b0 + share, shares, b1, a, f, b0, acc, ready);
    float* row = part + share * p.tokens * p.k * kTile + n;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < LAYOUT; ++j) put(row + j, m, acc[j][m]);
  }
}

// The activations of all slots, blocks [b0, b0 + n), in 4 bits into shared memory; by all threads.
__device__ __noinline__ void stage_activations4(const LayerParams& p, const DownShared& items, int b0, int n, int room, uint8_t* act, float* scale) {
  const int slots = p.tokens * p.k, tid = threadIdx.x, all = slots * n * 4;
  __syncthreads();
  for (int i0 = 0; i0 < all; i0 += kDownThreads) {       // (whole warps)
    const int i = min(i0 + tid, all - 1), slot = i / (n * 4), b = i / 4 - slot * n, c = (b0 + b) * 32 + i % 4 * 8;
    float v[8];
    activation<8>(p, items.parts, static_cast<long long>(slot) * p.J + c, p.J - c, v);
    const bool there = i0 + tid < all;
    const float f = items.weights[slot] * block4(v, there ? act + (slot * room + b) * 32 + i % 4 * 8 : nullptr);
    if (there && i % 4 == 0) scale[slot * room + b] = f;
  }
  __syncthreads();
}

template <typename T, int LAYOUT>
__global__ void __launch_bounds__(kDownThreads, 1) few_down4_kernel(const __grid_constant__ LayerParams p) {
  constexpr int kTile = tile4(LAYOUT);
  extern __shared__ __align__(16) float layer_smem[];
  __shared__ DownShared items;
  if (cluster_size() > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  pdl_trigger();
  begin_down(p, &items);
  const int slots = p.tokens * p.k, rank = cluster_rank(), size = cluster_size(), tid = threadIdx.x, warp = tid >> 5;
  const int n0 = blockIdx.x / size * kTile;
  float* part = layer_smem + p.act_floats;
  const int blocks = fp4_blocks(p.J);
  const int length = (blocks + size - 1) / size, begin = min(blocks, rank * length), end = min(blocks, begin + length);
  const int room = min(length, p.act_floats / (9 * slots));            // blocks: eight words of bytes and a scale
  uint8_t* act = reinterpret_cast<uint8_t*>(layer_smem);
  float* scale = layer_smem + static_cast<long long>(slots) * room * 8;
  int shares = 1;                              // warps that have an item's columns or blocks apart
  while (items.count * shares * 2 <= kDownWarps && shares < (LAYOUT ? length : 8)) shares *= 2;
  for (int b0 = begin; b0 == begin || b0 < end; b0 += room) {
    const int b1 = min(end, b0 + room);
    bool staged = false;
    auto stage = [&]() {
      if (staged) return;
      staged = true;
      stage_activations4(p, items, b0, b1 - b0, room, act, scale);
    };
    for (int x = warp; x < items.count * shares; x += kDownWarps) {
      const Item item = items.item[x / shares];
      const int share = x % shares;
      if (item.rows == 1) down4_item<LAYOUT, 1>(p, item, act, scale, room, b0, b1, n0, share, shares, part, b0 == begin, stage);
      else if (item.rows == 2) down4_item<LAYOUT, 2>(p, item, act, scale, room, b0, b1, n0, share, shares, part, b0 == begin, stage);
      else down4_item<LAYOUT, kRows>(p, item, act, scale, room, b0, b1, n0, share, shares, part, b0 == begin, stage);
    }
    stage();
  }
  __syncthreads();
  put_out<T, kTile>(p, part, part + max(4 * kDownWarps, slots) * kTile, LAYOUT ? shares : 1, n0);
}

// ---- launches ----------------------------------------------------------------------------------------------------------
constexpr size_t kDownSmem = 220 * 1024;

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

// CTAs of a cluster, each with 32 contraction elements at least and an SM of its own: of the processing clusters, 16 to 20 SMs, clusters of eight and
// of four leave some SMs unused.
unsigned cluster_of(int tiles, int J) {
  unsigned size = 8;
  auto fit = [](unsigned n) { return n == 8 ? 16 : n == 4 ? 32 : 74; };
  while (size > 1 && (tiles > fit(size) || J / static_cast<int>(size) < 32)) size /= 2;
  return size;
}

template <auto kernel, typename T>
cudaError_t down_launch(LayerParams p, int tile, cudaStream_t st) {
  const int tiles = (p.I + tile - 1) / tile, slots = p.tokens * p.k;
  cudaError_t err = ensure_smem_optin<kernel>(static_cast<int>(kDownSmem));
  if (err != cudaSuccess) return err;
  const unsigned size = cluster_of(tiles, p.J);
  const size_t ring = static_cast<size_t>(p.ring_words) * 4;
  const size_t part = static_cast<size_t>((slots < 4 * kDownWarps ? 4 * kDownWarps : slots) + (size > 1 ? p.tokens : 0)) * tile * sizeof(float);
  size_t act = static_cast<size_t>(slots) * (p.J / size + 36) * sizeof(float);
  act = (act + 15) & ~static_cast<size_t>(15);
  if (act > kDownSmem - part - ring) act = kDownSmem - part - ring;
  p.act_floats = static_cast<int>(act / sizeof(float));
  count_launch();
  return launch_cluster(kernel, tiles * size, kDownThreads, size, ring + act + part, st, p);
}

template <auto kernel>
cudaError_t up_launch(const LayerParams& p, cudaStream_t st) {
  constexpr int kMostTable = 2 * kUpWarps * EGS_MAX_EXPERTS * 4 + static_cast<int>(ring_bytes(kUpThreads, kUpDepth));
  cudaError_t err = ensure_smem_optin<kernel>(kMostTable);
  if (err != cudaSuccess) return err;
  count_launch();
  return launch_cluster(kernel, kUpGrid, kUpThreads, kUpCluster, (p.own_logits ? static_cast<size_t>(2 * kUpWarps) * ((p.E + 3) / 4 * 4) * 4 : 0) + static_cast<size_t>(p.ring_words) * 4, st, p);
}

bool on(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// An expert's weights of `down` that are brought to the L2 ahead: all, where those of all experts that can be chosen leave half of it to others.
void ahead(LayerParams* p, long long bytes) {
  const long long most = p->tokens * p->k < p->E ? p->tokens * p->k : p->E;
  p->down_bytes = bytes * most <= (64ll << 20) ? static_cast<int>(bytes) : 0;
  p->pieces = (p->down_bytes + 8191) / 8192;
  p->by_pieces = Div(p->pieces > 0 ? p->pieces : 1);
}

template <typename T>
cudaError_t layer_t(LayerParams p, const egs_route& route, bool fp4, bool up_cn, bool down_cn, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T), kLanes = 8;
  p.x_vectors = p.I % V == 0 && p.x_row % V == 0 && on(p.X, 16) && on(p.router, 16);
  // Logits by every cluster for itself where that is little: 64 KB of the router and 64 Ki products for a CTA.
  const long long router = static_cast<long long>(p.E) * p.I;
  p.by_k = Div(p.k);
  p.by_E4 = Div((p.E + 3) / 4 * 4);
  p.own_logits = p.tokens <= kUpWarps && router * static_cast<long long>(sizeof(T)) <= (256 << 10) && router * p.tokens <= (256 << 10);
  cudaError_t err = cudaSuccess;
  if (!p.own_logits) {
    count_launch();
    err = launch_kernel(few_logits_kernel<T>, dim3((p.E + 7) / 8, (p.tokens + kRows - 1) / kRows), 128, 0, st, true, p);
    if (err != cudaSuccess) return err;
    if ((err = launch_route_tokens(p.logits, p.bias, p.weights, p.experts, route, p.E, EGS_F32, st)) != cudaSuccess) return err;
  }
  if (fp4) {
    // (what lies behind the last row may be nobody's)
    ahead(&p, down_cn ? p.down_row * ((p.J + 1) / 2 - 1) + p.I / 16 * 16 : p.down_row * (p.I - 1) + (p.J + 1) / 2 / 16 * 16);
    if (p.down_far % 16 || !on(p.down, 16)) p.pieces = 0;
    auto fours = [](const void* w, long long row, long long far, int N) { return row % 4 == 0 && far % 4 == 0 && N % 4 == 0 && on(w, 4); };
    const int up = !up_cn ? 0 : fours(p.up, p.up_row, p.up_far, p.J) ? 4 : 1, down = !down_cn ? 0 : fours(p.down, p.down_row, p.down_far, p.I) ? 4 : 1;
    p.by_tiles = Div((p.J + tile4(up) - 1) / tile4(up));
    err = up == 0 ? up_launch<few_up4_kernel<T, 0>>(p, st) : up == 4 ? up_launch<few_up4_kernel<T, 4>>(p, st) : up_launch<few_up4_kernel<T, 1>>(p, st);
    if (err != cudaSuccess) return err;
    return down == 0 ? down_launch<few_down4_kernel<T, 0>, T>(p, tile4(0), st) : down == 4 ? down_launch<few_down4_kernel<T, 4>, T>(p, tile4(4), st) : down_launch<few_down4_kernel<T, 1>, T>(p, tile4(1), st);
  }
  // (one width for both: the parts of `up` are counted by it)
  const bool wide = p.I % V == 0 && p.J % V == 0 && on(p.up, 16) && on(p.down, 16);
  if (wide) {
    const long long bytes = static_cast<long long>(p.I) * p.J * sizeof(T);
    p.down_far = bytes;
    ahead(&p, bytes);
    p.by_tiles = Div((p.J + V * kLanes - 1) / (V * kLanes));
    p.ring_words = static_cast<int>(ring_bytes(kUpThreads, kUpDepth) / 4);
    if ((err = up_launch<few_up_kernel<T, V, kLanes>>(p, st)) != cudaSuccess) return err;
    p.ring_words = static_cast<int>(ring_bytes(kDownThreads, kDownDepth) / 4);
    return down_launch<few_down_kernel<T, V, kLanes>, T>(p, V * kLanes, st);
  }
  p.by_tiles = Div((p.J + 31) / 32);
  if ((err = up_launch<few_up_kernel<T, 1, 32>>(p, st)) != cudaSuccess) return err;
  return down_launch<few_down_kernel<T, 1, 32>, T>(p, 32, st);
}

}  // namespace

size_t few_layer_workspace(const egs_route& r, long long J) {
  const size_t logits = (static_cast<size_t>(r.tokens) * r.E + 3) / 4 * 4;
  return sizeof(LayerList) + (logits + static_cast<size_t>(kMostParts) * r.tokens * r.top_k * J) * sizeof(float);
}

cudaError_t launch_few_layer(const FewLayer& f, const egs_route& r, int dtype, void* workspace, cudaStream_t st) {
  LayerParams p{};
  p.X = f.X; p.router = f.router; p.up = f.up; p.down = f.down; p.up_scale = f.up_scale; p.down_scale = f.down_scale;
  p.out = f.out; p.weights = f.weights; p.experts = f.experts;
  p.list = static_cast<LayerList*>(workspace);
  p.logits = reinterpret_cast<float*>(p.list + 1);
  p.h = p.logits + (static_cast<size_t>(r.tokens) * r.E + 3) / 4 * 4;
  p.x_row = f.x_row;
  p.tokens = static_cast<int>(r.tokens); p.E = r.E; p.k = r.top_k; p.I = f.I; p.J = f.J;
  p.bias = f.bias; p.groups = r.groups; p.top_groups = r.top_groups; p.group_top = r.group_top;
  p.sigmoid = r.score == EGS_SCORE_SIGMOID; p.renormalize = r.renormalize; p.scale = r.scale;
  const bool fp4 = f.up_scale != nullptr;
  p.up_row = fp4 ? f.up_row : p.J; p.us_row = f.us_row; p.down_row = fp4 ? f.down_row : p.I; p.ds_row = f.ds_row;
  p.up_far = f.up_far; p.down_far = f.down_far;
  return dtype == EGS_F16 ? layer_t<__half>(p, r, fp4, f.up_cn, f.down_cn, st) : dtype == EGS_BF16 ? layer_t<__nv_bfloat16>(p, r, fp4, f.up_cn, f.down_cn, st) : layer_t<float>(p, r, fp4, f.up_cn, f.down_cn, st);
}

}  // namespace egs
