// Tokens that choose experts: routing and its gradient, the counting sort of the routed slots by expert, the weighted sum of a
// token's rows and its gradient, rows rounded to 8 bits, copies with another row pitch, and the CUDA-core products over ragged rows.
//
// Vocabulary beside egs_internal.cuh's:
//   slot         one (token, choice) pair; its number is token * k + choice
//   sorted row   place of a slot among all slots sorted by expert (slots of one expert in ascending order); the rows of expert e are
//                offsets[e] .. offsets[e + 1] - 1, those behind offsets[E] belong to slots that chose no expert
#include "egs_internal.cuh"

namespace egs {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// Floats as unsigned numbers of the same order; NaN lies below everything and above 0, which stands for "no candidate".
__device__ __forceinline__ uint32_t ordered(float x) {
  x += 0.f;                                    // -0 and 0 are equal
  const uint32_t b = __float_as_uint(x);
  return x != x ? 1u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// ------------------------------------------------------------------------------------------------
// Routing.  A warp has a token, lane l the NPER experts from l NPER on.  Softmax and no bias: the logits' order is the scores', so the logits
// are the keys, and a row's sum is only formed where something needs it.  Renormalised softmax weights are formed from the chosen logits
// alone.
//
// What bounds it is instructions (32768 tokens of 256 experts in 8 groups, sigmoid and bias: 35 MB, 5 us at the memory's rate), so few keys
// are formed exactly.  All lanes form keys from the fast exponential and reciprocal, within 2^-21 of a score.  The k-th highest of the
// lanes' own maxima is a lower bound of the k-th highest key; the keys that lie at most a margin of twice that error below it (256 random
// ones, k = 8: ten in the mean) go through shared memory to one lane each, where their exact keys are formed and every lane counts the keys
// before its own.  Where more than 32 lie there (many equal ones), every choice is a maximum over the exact keys of all lanes.
// Groups are compared by their fast keys too; where a group that is left out comes within the errors of one that is kept, all keys are formed
// exactly and the groups compared again (the check takes 1.2 us of 32; as a loop around both comparisons it took 3.4).
// ------------------------------------------------------------------------------------------------
constexpr int kRouteWarps = 8;

struct RouteParams {
  const void* logits;
  const float* bias;
  float* weights;
  int* experts;
  long long stride;      // elements from one token's logits to the next's
  int tokens, E, k, groups, top_groups, group_top, per;
  int sigmoid, renormalize;
  float scale;
  Div by_per;            // experts of a group
  int lanes_log2;        // lanes that look at a group together
  int whole_lanes;       // a group is the experts of 2^lanes_log2 lanes
  int vectors;           // rows (and the bias) begin on 16 bytes and have 32 NPER experts
  int warp_words;        // shared memory of a warp
};

__device__ __forceinline__ float unordered(uint32_t k) {         // (the float of ordered(); a NaN for its 1)
  return k <= 1u ? __uint_as_float(0x7fc00000u) : __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// n elements from `p` on (those that exist: left), in 16-byte loads where `wide`
template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, int left, bool wide, float (&v)[N]) {
  constexpr int V = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  if (wide) {
#pragma unroll
    for (int i = 0; i < N / V; ++i) {
      const Packed<T, V> x = reinterpret_cast<const Packed<T, V>*>(p)[i];
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = x.get(j);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < left ? to_f32<T>(p[i]) : 0.f;
  }
}

// CTAs of an SM, as many as the keys of a thread leave registers for.
__host__ __device__ constexpr int route_ctas(int nper) { return nper <= 2 ? 8 : nper == 4 ? 6 : nper == 8 ? 5 : nper == 16 ? 3 : 2; }

template <typename T, int NPER>
__global__ void __launch_bounds__(kRouteWarps * 32, route_ctas(NPER)) route_tokens_kernel(const __grid_constant__ RouteParams p) {
  extern __shared__ __align__(16) uint32_t route_smem[];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * kRouteWarps + warp;
  if (t >= p.tokens) return;
  uint32_t* mem = route_smem + warp * p.warp_words;      // keys (groups that are not whole lanes), then candidates
  const T* row = static_cast<const T*>(p.logits) + t * p.stride;
  const int e0 = lane * NPER, mine_left = p.E - e0;      // this lane's experts: those of index < mine_left
  float x[NPER];
  load_run<T, NPER>(row + e0, mine_left, p.vectors, x);
  const bool pairs = p.groups > 1 && p.group_top == 2;
  const bool sums = !p.sigmoid && (p.bias || pairs || !p.renormalize);
  float m = 0.f, total = 1.f;
  uint32_t key[NPER];
  if (sums) {                                            // scores of a softmax, in x' place
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NPER; ++i)
      if (i < mine_left) m = fmaxf(m, x[i]);
    m = warp_max(m);
    total = 0.f;
    float ex[NPER];
#pragma unroll
    for (int i = 0; i < NPER; ++i) {
      ex[i] = i < mine_left && m != -INFINITY ? expf(x[i] - m) : 0.f;
      total += ex[i];
    }
    total = warp_sum(total);
    if (p.bias || pairs) {
      const float inverse = m == -INFINITY ? 0.f : 1.f / total;
#pragma unroll
      for (int i = 0; i < NPER; ++i) ex[i] *= inverse;
    }
    if (p.bias) {
      float b[NPER];
      load_run<float, NPER>(p.bias + e0, mine_left, p.vectors, b);
#pragma unroll
      for (int i = 0; i < NPER; ++i) key[i] = ordered(ex[i] + b[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NPER; ++i) key[i] = pairs ? ordered(ex[i]) : ordered(x[i]);
    }
  } else if (p.sigmoid && (p.bias || pairs)) {
    float b[NPER];
    if (p.bias) load_run<float, NPER>(p.bias + e0, mine_left, p.vectors, b);
#pragma unroll
    for (int i = 0; i < NPER; ++i) {
      const float s = __fdividef(1.f, 1.f + __expf(-x[i]));
      key[i] = ordered(p.bias ? s + b[i] : s);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NPER; ++i) key[i] = ordered(x[i]);
  }
  // whether the keys above are fast ones, and the exact key of an expert
  const bool fast = p.bias || pairs;
  auto score_of = [&](float v) { return p.sigmoid ? sigmoid(v) : m == -INFINITY ? 0.f : expf(v - m) / total; };
  auto exact = [&](float v, int e) { return ordered(p.bias ? score_of(v) + p.bias[e] : v); };
  if (!p.vectors) {
#pragma unroll
    for (int i = 0; i < NPER; ++i)
      if (i >= mine_left) key[i] = 0u;
  }
  if (p.groups > 1) {
    const int g = lane >> p.lanes_log2;
    const bool first_lane = g < p.groups && !(lane & ((1 << p.lanes_log2) - 1));
    uint32_t kept;                                       // by first lanes
    // The groups of highest value; whether errors of fast keys may have decided that.
    auto choose_groups = [&](bool fast_keys) {
      uint32_t k1 = 0u, k2 = 0u;                         // the two highest keys
      if (p.whole_lanes) {
#pragma unroll
        for (int i = 0; i < NPER; ++i) {
          k2 = max(k2, min(k1, key[i]));
          k1 = max(k1, key[i]);
        }
      } else {
        // through shared memory: the lanes of a group look at every 2^lanes_log2-th of its keys
#pragma unroll
        for (int i = 0; i < NPER; ++i)
          if (i < mine_left) mem[e0 + i] = key[i];
        __syncwarp();
        if (g < p.groups)
          for (int i = lane & ((1 << p.lanes_log2) - 1); i < p.per; i += 1 << p.lanes_log2) {
            const uint32_t v = mem[g * p.per + i];
            k2 = max(k2, min(k1, v));
            k1 = max(k1, v);
          }
        __syncwarp();
      }
      for (int o = 1; o < (1 << p.lanes_log2); o <<= 1) {
        const uint32_t o1 = __shfl_xor_sync(kFull, k1, o), o2 = __shfl_xor_sync(kFull, k2, o);
        k2 = max(min(k1, o1), max(k2, o2));
        k1 = max(k1, o1);
      }
      // (every lane of a group has its value; the first one stands for it)
      const bool both = pairs && k2;
      const float a = unordered(k1), b = both ? unordered(k2) : 0.f, value = a + b;
      uint32_t gk = !first_lane ? 0u : both ? ordered(value) : k1, low = 0u;
      kept = 0u;
      for (int i = 0; i < p.top_groups; ++i) {
        low = __reduce_max_sync(kFull, gk);
        const int at = __ffs(__ballot_sync(kFull, gk == low)) - 1;
        kept |= 1u << at;
        if (lane == at) gk = 0u;
      }
      if (!fast_keys || p.top_groups == p.groups) return false;
      // A value has to be further from the nearest one beyond the cut than twice its error: of a sum of a score and a bias 2^-21 and a unit, of a
      // score alone 126 units (2 + 1.18 * 88 of the exponential, 2 of the reciprocal, the others the exact ones) and, where the fast reciprocal
      // gives 0, 2^-126.  (Infinite values have no error, and of equal ones the difference is a NaN.)
      const float high = unordered(__reduce_max_sync(kFull, gk));
      const float gap = gk ? unordered(low) - value : value - high;
      const float slack = p.bias ? 2e-6f * (1.f + fabsf(a) + fabsf(b)) : fmaf(3e-5f, value, 8e-38f);
      return __any_sync(kFull, first_lane && slack < INFINITY && gap <= slack) != 0;
    };
    if (choose_groups(fast)) {
      // (one after the other: unrolled, they took registers that leave the common way fewer warps, 80 for 48)
#pragma unroll 1
      for (int j = 0; j < min(NPER, mine_left); ++j) {
        const float x_j = to_f32<T>(row[e0 + j]);
        const uint32_t k = p.bias ? exact(x_j, e0 + j) : ordered(score_of(x_j));
#pragma unroll
        for (int i = 0; i < NPER; ++i)
          if (i == j) key[i] = k;
      }
      __syncwarp();
      choose_groups(false);
    }
    if (p.whole_lanes) {
      if (!((kept >> (g << p.lanes_log2)) & 1u)) {
#pragma unroll
        for (int i = 0; i < NPER; ++i) key[i] = 0u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NPER; ++i)
        if (!((kept >> ((p.by_per.quotient(e0 + i) << p.lanes_log2) & 31)) & 1u)) key[i] = 0u;
    }
    if (pairs && !p.bias) {                              // scores have compared the groups; their experts are compared by the logits
#pragma unroll
      for (int i = 0; i < NPER; ++i)
        if (key[i]) key[i] = ordered(x[i]);
    }
  }
  const float margin = fast && p.bias ? 1e-6f : 0.f;
  // lower bound, candidates
  uint32_t top = key[0];
#pragma unroll
  for (int i = 1; i < NPER; ++i) top = max(top, key[i]);
  uint32_t bound = 0u;
  for (int j = 0; j < p.k; ++j) {              // (equal maxima go together: the bound is then lower than it might be)
    const uint32_t best = __reduce_max_sync(kFull, top);
    bound = best;
    if (best == 0u) break;
    if (top == best) top = 0u;
  }
  if (margin > 0.f && bound > 1u) {
    const float b = unordered(bound);
    bound = ordered(b - margin * (1.f + fabsf(b)));      // (infinities stay where they are)
    if (b != b || fabsf(b) == INFINITY) bound = 1u;
  }
  bound = max(bound, 1u);
  int own = 0;
#pragma unroll
  for (int i = 0; i < NPER; ++i) own += key[i] >= bound ? 1 : 0;
  int at = own;                                // candidates up to this lane's last: in the order of the experts
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, at, o);
    if (lane >= o) at += v;
  }
  const int found = __shfl_sync(kFull, at, 31);
  int mine = 0, place = p.k;                   // this lane's chosen expert and its place among them
  float xc = -INFINITY;                        // ... and its logit
  if (found <= 32) {
    at -= own;
    if (own) {
#pragma unroll
      for (int i = 0; i < NPER; ++i)
        if (key[i] >= bound) mem[at++] = e0 + i;
    }
    __syncwarp();
    mine = lane < found ? static_cast<int>(mem[lane]) : 0;
    xc = lane < found ? to_f32<T>(row[mine]) : -INFINITY;
    const uint32_t k = lane < found ? exact(xc, mine) : 0u;
    mem[32 + lane] = k;
    __syncwarp();
    int before = 0;
    for (int j = 0; j < found; j += 4) {       // (no key is 2^32 - 1, and there are zeros behind the last one)
      const uint4 other = *reinterpret_cast<const uint4*>(mem + 32 + j);
      before += other.x + (j < lane) > k;
      before += other.y + (j + 1 < lane) > k;
      before += other.z + (j + 2 < lane) > k;
      before += other.w + (j + 3 < lane) > k;
    }
    if (lane < found) place = before;
  } else {
    if (fast) {
#pragma unroll
      for (int i = 0; i < NPER; ++i)
        if (key[i]) key[i] = exact(x[i], e0 + i);
    }
    for (int j = 0; j < p.k; ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int i = 1; i < NPER; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(kFull, best);
      uint32_t who = kFull;
#pragma unroll
      for (int i = NPER - 1; i >= 0; --i)
        if (key[i] == best) who = e0 + i;
      who = __reduce_min_sync(kFull, who);
#pragma unroll
      for (int i = 0; i < NPER; ++i)
        if (who == e0 + i) key[i] = 0u;
      if (lane == j) {
        mine = static_cast<int>(who);
        place = j;
      }
    }
    if (place < p.k) xc = to_f32<T>(row[mine]);
  }
  const bool chosen = place < p.k;
  if (!chosen) xc = -INFINITY;
  float w;
  if (p.renormalize) {
    const float best = p.sigmoid ? 0.f : warp_max(xc);
    const float s = !chosen ? 0.f : p.sigmoid ? sigmoid(xc) : best == -INFINITY ? 0.f : expf(xc - best);
    const float sum = warp_sum(s);
    w = sum == 0.f ? 0.f : s / sum;
  } else {
    w = p.sigmoid ? sigmoid(xc) : m == -INFINITY ? 0.f : expf(xc - m) / total;
  }
  if (chosen) {
    p.weights[static_cast<long long>(t) * p.k + place] = w * p.scale;
    p.experts[static_cast<long long>(t) * p.k + place] = mine;
  }
}

// The gradient: rows of zeros with a value for every chosen expert, except where softmax weights are not renormalised.  Ids outside
// [0, E) (a choice that was taken away) have no part in it.
struct RouteBackwardParams {
  const float* dweights;
  const void* logits;
  const int* experts;
  void* dlogits;
  long long stride;
  int tokens, E, k;
  int sigmoid, renormalize, vectors;     // vectors: rows of whole, aligned 16 bytes
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(kRouteWarps * 32) route_backward_kernel(const __grid_constant__ RouteBackwardParams p) {
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + warp;
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.stride;
  T* out = static_cast<T*>(p.dlogits) + t * p.E;
  int e = lane < p.k ? p.experts[t * p.k + lane] : -1;
  const bool on = e >= 0 && e < p.E;
  const float g = on ? p.dweights[t * p.k + lane] * p.scale : 0.f;
  const float x = on ? to_f32<T>(row[e]) : -INFINITY;
  const bool whole_row = !p.sigmoid && !p.renormalize;
  float d;
  if (whole_row) {
    float m = -INFINITY;
    for (int i = lane; i < p.E; i += 32) m = fmaxf(m, to_f32<T>(row[i]));
    m = warp_max(m);
    float total = 0.f;
    for (int i = lane; i < p.E; i += 32) total += m == -INFINITY ? 0.f : expf(to_f32<T>(row[i]) - m);
    total = warp_sum(total);
    const float s = on && m != -INFINITY ? expf(x - m) / total : 0.f;
    const float back = warp_sum(g * s);
    for (int i = lane; i < p.E; i += 32)
      out[i] = from_f32<T>(m == -INFINITY ? 0.f : -(expf(to_f32<T>(row[i]) - m) / total) * back);
    d = s * (g - back);
  } else {
    if (p.vectors) {
      constexpr int V = 16 / sizeof(T);
      for (int i = lane; i < p.E / V; i += 32) reinterpret_cast<uint4*>(out)[i] = make_uint4(0u, 0u, 0u, 0u);
    } else {
      for (int i = lane; i < p.E; i += 32) out[i] = from_f32<T>(0.f);
    }
    if (p.sigmoid) {
      const float s = on ? sigmoid(x) : 0.f, slope = s / (1.f + expf(x));          // s (1 - s)
      if (p.renormalize) {
        // (the weights, not their sum at the end: one choice has the weight 1 and the gradient 0, exactly)
        const float sum = warp_sum(s), w = sum == 0.f ? 0.f : s / sum, back = warp_sum(g * w);
        d = sum == 0.f ? 0.f : (g - back) / sum * slope;
      } else {
        d = g * slope;
      }
    } else {
      const float top = warp_max(x);
      const float s = on && top != -INFINITY ? expf(x - top) : 0.f;
      const float sum = warp_sum(s), w = sum == 0.f ? 0.f : s / sum;
      d = w * (g - warp_sum(w * g));
    }
  }
  __syncwarp();                                // the row before its chosen experts
  if (on) out[e] = from_f32<T>(d);
}

// ------------------------------------------------------------------------------------------------
// Counting sort of the slots by expert.  Every CTA has a stretch of slots, counts it, learns the counts of the others, finds the start of its
// stretch within every expert and places its slots.  Up to 16 CTAs are a cluster and read one another's counts; beyond, a kernel before this
// one counts the stretches (64 experts, 8000 / 32768 / 65536 / 131072 slots: 5.0 / 5.4 / 7.4 / 13.7 us on a cluster, 8.2 / 8.0 / 8.0 / 9.5 in
// two kernels).  Inside a stretch every warp has a
// part, counted and placed 32 slots at a time, so that slots of one expert stay in order.  Ids outside [0, E) are an expert of their
// own behind the others.
// ------------------------------------------------------------------------------------------------
constexpr int kPlanWarps = 16, kPlanThreads = kPlanWarps * 32;

struct PlanParams {
  const int* experts;
  int* offsets;      // [E + 1]
  int* slots;        // [n]
  int* position;     // [n]
  int* counts;       // [E + 1][stretches], unused with one stretch
  int n, E, part, stretches;      // part: slots of a warp, a multiple of 32; a stretch is kPlanWarps of them
  StatusRef status;
};

// A warp's slots: the first 256 of them (all, up to a million slots) in registers, so that their loads are under way together and
// are made once.
constexpr int kPlanHeld = 8;
constexpr int kPlanCluster = 16;         // CTAs of a cluster at most
struct PlanPart {
  const int* ids;
  long long first;
  int n, lane, held[kPlanHeld];
  __device__ __forceinline__ explicit PlanPart(const PlanParams& p) {
    first = (static_cast<long long>(blockIdx.x) * kPlanWarps + (threadIdx.x >> 5)) * p.part;
    n = static_cast<int>(max(0ll, min(static_cast<long long>(p.part), p.n - first)));
    lane = threadIdx.x & 31;
    ids = p.experts + first;
#pragma unroll
    for (int i = 0; i < kPlanHeld; ++i) held[i] = i * 32 + lane < n ? ids[i * 32 + lane] : -1;
  }
  // f(index of the warp's 32 slots, this lane's id) for all of them
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int i = 0; i < kPlanHeld; ++i)
      if (i * 32 < n) f(i * 32, held[i]);
    for (int i = kPlanHeld * 32; i < n; i += 32) f(i, i + lane < n ? ids[i + lane] : -1);
  }
};

// smem: [kPlanWarps][E + 1] counts of the warps' parts
__device__ __forceinline__ void count_parts(const PlanParams& p, const PlanPart& part, int* table, bool report) {
  const int E1 = p.E + 1;
  for (int i = threadIdx.x; i < kPlanWarps * E1; i += kPlanThreads) table[i] = 0;
  __syncthreads();
  int* mine = table + (threadIdx.x >> 5) * E1;
  part.each([&](int i, int e) {
    if (i + part.lane >= part.n) return;
    if (e < 0 || e >= p.E) {
      if (e != -1 && report) p.status.report(EGS_STATUS_INDEX_OUT_OF_RANGE);
      e = p.E;
    }
    atomicAdd(mine + e, 1);
  });
  __syncthreads();
}

__global__ void __launch_bounds__(kPlanThreads) plan_count_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int table[];
  pdl_wait();
  pdl_trigger();
  const PlanPart part(p);
  count_parts(p, part, table, true);
  const int E1 = p.E + 1;
  for (int e = threadIdx.x; e < E1; e += kPlanThreads) {
    int sum = 0;
    for (int w = 0; w < kPlanWarps; ++w) sum += table[w * E1 + e];
    p.counts[static_cast<long long>(e) * p.stretches + blockIdx.x] = sum;
  }
}

// What the CTA `rank` of the cluster has at the address of `mine`.
__device__ __forceinline__ int of_cta(const int* mine, int rank) {
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// S: CTAs of the cluster, which is the grid;  1: any number of stretches, counted before (one: not)
template <int S>
__global__ void __cluster_dims__(S, 1, 1) __launch_bounds__(kPlanThreads) plan_place_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int table[];
  __shared__ int sums[kPlanWarps];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E1 = p.E + 1;
  const bool one = S > 1 || p.stretches == 1;
  const PlanPart part(p);
  // slots of an expert in the stretches before this one, in all of them: a warp has an expert, a lane a stretch (one thread that went
  // through 64 stretches of an expert took 6 us of the kernel's 12)
  int* before = table + kPlanWarps * E1;
  int* all = before + E1;
  if (!one) {
#pragma unroll 4
    for (int e = warp; e < E1; e += kPlanWarps) {
      int b = 0, a = 0;
      for (int s = lane; s < p.stretches; s += 32) {
        const int c = p.counts[static_cast<long long>(e) * p.stretches + s];
        a += c;
        if (s < static_cast<int>(blockIdx.x)) b += c;
      }
      a = __reduce_add_sync(kFull, a);
      b = __reduce_add_sync(kFull, b);
      if (lane == 0) {
        before[e] = b;
        all[e] = a;
      }
    }
  }
  count_parts(p, part, table, one);
  if (one) {
    for (int e = threadIdx.x; e < E1; e += kPlanThreads) {
      int sum = 0;
      for (int w = 0; w < kPlanWarps; ++w) sum += table[w * E1 + e];
      before[e] = 0;
      all[e] = sum;
    }
  }
  if constexpr (S > 1) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    constexpr int kEach = (EGS_MAX_EXPERTS + kPlanThreads) / kPlanThreads;     // experts of a thread
    int a[kEach] = {};
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int e = threadIdx.x + i * kPlanThreads;
      if (e >= E1) break;
      int c[S], b = 0;
#pragma unroll
      for (int r = 0; r < S; ++r) c[r] = of_cta(all + e, r);
#pragma unroll
      for (int r = 0; r < S; ++r) {
        a[i] += c[r];
        if (r < static_cast<int>(blockIdx.x)) b += c[r];
      }
      before[e] = b;
    }
    __syncwarp();
    cluster_arrive();                          // (nobody's counts are written over, and no CTA ends, before all have been read)
    cluster_wait();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (threadIdx.x + i * kPlanThreads < E1) all[threadIdx.x + i * kPlanThreads] = a[i];
  }
  __syncthreads();
  // offsets of the experts, and from them where each warp's slots begin
  int carry = 0;
  for (int e0 = 0; e0 < E1; e0 += kPlanThreads) {
    const int e = e0 + threadIdx.x, own = e < E1 ? all[e] : 0;
    int incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int base = carry;
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) {
      const int v = sums[w];
      if (w < warp) base += v;
      carry += v;
    }
    const int offset = base + incl - own;
    if (e < E1) {
      if (blockIdx.x == 0) p.offsets[e] = offset;
      int c[kPlanWarps], at = offset + before[e];
#pragma unroll
      for (int w = 0; w < kPlanWarps; ++w) c[w] = table[w * E1 + e];
#pragma unroll
      for (int w = 0; w < kPlanWarps; ++w) {
        table[w * E1 + e] = at;
        at += c[w];
      }
    }
    __syncthreads();
  }
  int* mine = table + warp * E1;
  part.each([&](int i0, int e) {
    const bool on = i0 + lane < part.n;
    const bool real = e >= 0 && e < p.E;
    if (!real) e = p.E;
    const unsigned same = __match_any_sync(kFull, on ? e : -1);
    const int rank = __popc(same & ((1u << lane) - 1u));
    const int at = on ? mine[e] + rank : 0;
    __syncwarp();
    if (on && rank == 0) mine[e] += __popc(same);
    __syncwarp();
    if (on) {
      const long long slot = part.first + i0 + lane;
      p.slots[at] = static_cast<int>(slot);
      p.position[slot] = real ? at : ~at;
    }
  });
}

// ------------------------------------------------------------------------------------------------
// Weighted sum of a token's rows, float32 in the order of its choices, rounded once.
// ------------------------------------------------------------------------------------------------
// V elements in one store
template <typename T, int V> struct Vec {
  static __device__ __forceinline__ void store(T* p, const float (&v)[V]) {
    Packed<T, V> x;
    T* h = reinterpret_cast<T*>(x.raw);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = from_f32<T>(v[i]);
    *reinterpret_cast<Packed<T, V>*>(p) = x;
  }
};

struct CombineParams {
  const void* Y;           // sorted rows
  const void* weights;     // [tokens, k] or NULL (ones)
  const int* position;
  void* out;               // token rows;  backward: dY, sorted rows
  const void* dOut;        // backward: token rows
  void* dweights;          // backward: [tokens, k]
  int tokens, k, N, vecs;  // vecs: vectors of a row
  int w_f32;               // weights (and their gradient) in float32, else in the output's type
  Div by_blocks;           // forward: blocks of 32 vectors of a row
  Div by_k;                // backward
  int work;                // forward: tokens * blocks
};
template <typename T>
__device__ __forceinline__ float weight_of(const CombineParams& p, long long slot) {
  return !p.weights ? 1.f : p.w_f32 ? static_cast<const float*>(p.weights)[slot] : to_f32<T>(static_cast<const T*>(p.weights)[slot]);
}

// The rows lie anywhere, and what a thread may have in registers is not enough to keep the memory busy (eight loads a thread, 24 warps an
// SM: 200 us for 131072 rows of 2048 bf16, 3.4 TB/s).  So vectors go to shared memory by cp.async, each to the thread that sums it: a warp
// has 512 bytes of a token's columns at a time, four choices are a step, three steps are on their way, and positions are asked for a
// step before that.
constexpr int kCombineStages = 4, kCombineAhead = kCombineStages - 1, kCombineWarps = 4, kCombineCtas = 148 * 6;

// T: the rows' type, O: the output's (and the weights', where those are not float32)
template <typename T, typename O, int V>
__global__ void __launch_bounds__(kCombineWarps * 32) combine_kernel(const __grid_constant__ CombineParams p) {
  using P = Packed<T, V>;
  static_assert(sizeof(P) == 16 || sizeof(P) == 8 || sizeof(P) == 4, "what cp.async copies");
  constexpr int U = 16 / sizeof(P);            // vectors of a lane, 32 V columns apart
  __shared__ P ring[kCombineStages][4][U][kCombineWarps * 32];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int first = blockIdx.x * kCombineWarps + (threadIdx.x >> 5), stride = gridDim.x * kCombineWarps;
  const int items = p.work > first ? static_cast<int>((p.work - 1 - first) / stride) + 1 : 0;
  const int groups = (p.k + 3) / 4;            // steps of an item
  const T* Y = static_cast<const T*>(p.Y);
  // a step further along: the token, its block of columns, the first of the four choices
  struct Step {
    int item, group;
  };
  auto next = [&](Step& s) {
    if (++s.group == groups) {
      s.group = 0;
      ++s.item;
    }
  };
  auto place = [&](const Step& s, int* block) {
    int i = first + s.item * stride;
    *block = p.by_blocks.remainder(i);
    return i;
  };
  Step ask{0, 0}, copy{0, 0}, use{0, 0};
  auto position = [&]() {                      // of choice `lane` of the step asked for
    int block, pos = -1;
    if (ask.item < items && lane < 4 && ask.group * 4 + lane < p.k) pos = p.position[static_cast<long long>(place(ask, &block)) * p.k + ask.group * 4 + lane];
    next(ask);
    return pos;
  };
  auto weight = [&](const Step& s) {
    int block;
    if (s.item >= items || lane >= 4 || s.group * 4 + lane >= p.k) return 0.f;
    return weight_of<O>(p, static_cast<long long>(place(s, &block)) * p.k + s.group * 4 + lane);
  };
  unsigned present[kCombineStages];            // choices of a stage that have a row
  int pos = position();
  auto fetch = [&](int stage) {
    unsigned have = 0u;
    if (copy.item < items) {
      int block;
      place(copy, &block);
      const int c = (block * 32 * U + lane) * V;
      have = __ballot_sync(kFull, pos >= 0) & 15u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = __shfl_sync(kFull, pos, j);
        if (at < 0) continue;
        const T* src = Y + static_cast<long long>(at) * p.N + c;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (c + u * 32 * V >= p.N) break;
          const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(&ring[stage][j][u][threadIdx.x]));
          if constexpr (sizeof(P) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src + u * 32 * V) : "memory");
          else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src + u * 32 * V), "n"(sizeof(P)) : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    next(copy);
    pos = position();
    return have;
  };
#pragma unroll
  for (int i = 0; i < kCombineAhead; ++i) present[i] = fetch(i);
  float w = weight(use), sum[U][V];
  while (use.item < items) {
#pragma unroll
    for (int stage = 0; stage < kCombineStages; ++stage) {
      if (use.item >= items) break;
      present[(stage + kCombineAhead) % kCombineStages] = fetch((stage + kCombineAhead) % kCombineStages);
      Step after = use;
      next(after);
      const float w_next = weight(after);
      asm volatile("cp.async.wait_group %0;" ::"n"(kCombineAhead) : "memory");
      if (use.group == 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int v = 0; v < V; ++v) sum[u][v] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float wj = __shfl_sync(kFull, w, j);
        if ((present[stage] >> j) & 1u) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const P y = ring[stage][j][u][threadIdx.x];
#pragma unroll
            for (int v = 0; v < V; ++v) sum[u][v] = fmaf(wj, y.get(v), sum[u][v]);
          }
        }
      }
      if (use.group == groups - 1) {
        int block;
        const long long t = place(use, &block);
        const int c = (block * 32 * U + lane) * V;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c + u * 32 * V < p.N) Vec<O, V>::store(static_cast<O*>(p.out) + t * p.N + c + u * 32 * V, sum[u]);
      }
      use = after;
      w = w_next;
    }
  }
}

// Rows that do not even begin on 4 bytes: 64 threads have a token, each every 64th column.
template <typename T, typename O>
__global__ void __launch_bounds__(256) combine_columns_kernel(const __grid_constant__ CombineParams p) {
  pdl_wait();
  pdl_trigger();
  const long long t = static_cast<long long>(blockIdx.x) * 4 + threadIdx.x / 64;
  if (t >= p.tokens) return;
  const int* pos = p.position + t * p.k;
  O* out = static_cast<O*>(p.out) + t * p.N;
  for (int c0 = threadIdx.x & 63; c0 < p.N; c0 += 256) {
    float sum[4] = {};
    for (int j = 0; j < p.k; ++j) {
      const int at = pos[j];
      if (at < 0) continue;
      const float w = weight_of<O>(p, t * p.k + j);
      const T* y = static_cast<const T*>(p.Y) + static_cast<long long>(at) * p.N;
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = c0 + 64 * i < p.N ? to_f32<T>(y[c0 + 64 * i]) : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = fmaf(w, v[i], sum[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c0 + 64 * i < p.N) out[c0 + 64 * i] = from_f32<O>(sum[i]);
  }
}

// Rows of at most 32 vectors: 2^lanes_log2 threads have a token, one vector each; four rows are on their way, and the next four places.  bf16,
// this and the kernel above, which leaves lanes without work: 32768 tokens of eight rows of 64 16 and 33 us, of one row 10 and 18; 21419 of eight
// rows of 152 25 and 27; from 64 vectors on no faster (32768 of four rows of 512: 43 and 42).
template <typename T, typename O, int V>
__global__ void __launch_bounds__(256) combine_narrow_kernel(const __grid_constant__ CombineParams p, int lanes_log2) {
  using P = Packed<T, V>;
  pdl_wait();
  pdl_trigger();
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, t = i >> lanes_log2;
  const int c = static_cast<int>(i) & ((1 << lanes_log2) - 1);
  if (t >= p.tokens || c >= p.vecs) return;
  const long long slot = t * p.k;
  const P* Y = static_cast<const P*>(p.Y) + c;
  int at[4], coming[4];
  auto places = [&](int j0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) coming[j] = j0 + j < p.k ? p.position[slot + j0 + j] : -1;
  };
  places(0);
  float sum[V] = {};
  for (int j0 = 0; j0 < p.k; j0 += 4) {
    P y[4];
    float w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      at[j] = coming[j];
      if (at[j] < 0) continue;
      y[j] = Y[static_cast<long long>(at[j]) * p.vecs];
      w[j] = weight_of<O>(p, slot + j0 + j);
    }
    places(j0 + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (at[j] < 0) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) sum[v] = fmaf(w[j], y[j].get(v), sum[v]);
    }
  }
  Vec<O, V>::store(static_cast<O*>(p.out) + (t * p.vecs + c) * V, sum);
}

// A warp has a slot: dY = weight * dOut of its token, dweight = the product of the two rows.  Slots without an expert have a row of
// zeros and a gradient of zero.  (A warp for every token, ten loads of four choices under way together: no faster for 512 bf16, 22 us
// instead of 20 for 65536 slots of 256, 17 instead of 11 for 32768 of 64 float32.)
template <typename T, int V>
__global__ void __launch_bounds__(256) combine_backward_kernel(const __grid_constant__ CombineParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long slot = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (slot >= static_cast<long long>(p.tokens) * p.k) return;
  const long long t = slot / p.k;
  const int at = p.position[slot];
  float dot = 0.f;
  if (at >= 0) {
    const float w = weight_of<T>(p, slot);
    const T* g = static_cast<const T*>(p.dOut) + t * p.N;
    const T* y = static_cast<const T*>(p.Y) + static_cast<long long>(at) * p.N;
    T* d = static_cast<T*>(p.out) + static_cast<long long>(at) * p.N;
    for (int c = lane; c < p.vecs; c += 32) {
      const Packed<T, V> gp = *reinterpret_cast<const Packed<T, V>*>(g + c * V);
      Packed<T, V> yp;
      if (p.dweights) yp = *reinterpret_cast<const Packed<T, V>*>(y + c * V);
      float x[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = gp.get(v);
        if (p.dweights) dot = fmaf(x[v], yp.get(v), dot);
        x[v] *= w;
      }
      Vec<T, V>::store(d + c * V, x);
    }
  }
  if (at < 0) {
    T* d = static_cast<T*>(p.out) + static_cast<long long>(~at) * p.N;
    const float zeros[V] = {};
    for (int c = lane; c < p.vecs; c += 32) Vec<T, V>::store(d + c * V, zeros);
  }
  if (!p.dweights) return;
  dot = warp_sum(dot);
  if (lane == 0) {
    if (p.w_f32) static_cast<float*>(p.dweights)[slot] = dot;
    else static_cast<T*>(p.dweights)[slot] = from_f32<T>(dot);
  }
}

// ... of rows of at most 16 vectors: 2^lanes_log2 lanes have a slot, one vector each, and slot after slot; the two rows of the next one are on
// their way and its successor's place is asked for.  bf16, this and a warp for every slot: 240000 slots of 32 16 and 64 us, 32768 of 64 10 and
// 14 to 16, 24000 of 128 11 and 12; with all 32 lanes 65536 of 256 27 and 27, 171352 of 152 56 and 53.
constexpr int kNarrowCtas = 148 * 5;
template <typename T, int V>
__global__ void __launch_bounds__(256, 5) combine_backward_narrow_kernel(const __grid_constant__ CombineParams p, int lanes_log2) {
  using P = Packed<T, V>;
  pdl_wait();
  const int lane = threadIdx.x & 31, lanes = 1 << lanes_log2, c = lane & (lanes - 1), each = 32 >> lanes_log2;
  const long long total = static_cast<long long>(p.tokens) * p.k, stride = static_cast<long long>(gridDim.x) * 8 * each;
  const P* G = static_cast<const P*>(p.dOut) + c;
  const P* Y = static_cast<const P*>(p.Y) + c;
  auto place = [&](long long slot) { return slot < total ? p.position[slot] : -1; };
  struct Held {
    P g, y;
    float w;
  };
  auto fetch = [&](Held& h, long long slot, int at) {
    if (at < 0) return;
    h.w = weight_of<T>(p, slot);
    if (c >= p.vecs) return;
    h.g = G[static_cast<long long>(p.by_k.quotient(static_cast<int>(slot))) * p.vecs];
    if (p.dweights) h.y = Y[static_cast<long long>(at) * p.vecs];
  };
  long long slot = (static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * each + (lane >> lanes_log2);
  int at = place(slot), at_next = place(slot + stride);
  Held now, next;
  fetch(now, slot, at);
  for (long long first = slot - (lane >> lanes_log2); first < total; first += stride, slot += stride) {
    fetch(next, slot + stride, at_next);
    const int at_after = place(slot + 2 * stride);
    float dot = 0.f;
    if (slot < total && c < p.vecs) {
      float x[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = at >= 0 ? now.g.get(v) : 0.f;
        if (p.dweights && at >= 0) dot = fmaf(x[v], now.y.get(v), dot);
        x[v] = at >= 0 ? x[v] * now.w : 0.f;
      }
      Vec<T, V>::store(static_cast<T*>(p.out) + (static_cast<long long>(at >= 0 ? at : ~at) * p.vecs + c) * V, x);
    }
    if (p.dweights) {
      for (int o = lanes >> 1; o; o >>= 1) dot += __shfl_xor_sync(kFull, dot, o);
      if (c == 0 && slot < total) {
        if (p.w_f32) static_cast<float*>(p.dweights)[slot] = dot;
        else static_cast<T*>(p.dweights)[slot] = from_f32<T>(dot);
      }
    }
    at = at_next;
    at_next = at_after;
    now = next;
  }
}

// ------------------------------------------------------------------------------------------------
// Rows in 8 bits: scale = largest magnitude / 127, q = x / scale to the nearest integer, ties to even.  A row with an infinity or a
// NaN in it has the scale NaN and zeros, so that its products are NaN.  The elements a thread has seen for the maximum stay in
// registers as far as they fit.
// ------------------------------------------------------------------------------------------------
struct QuantizeParams {
  const void* X;
  int8_t* q;
  float* scale;
  long long x_stride, q_stride;
  int rows, C;
};

// The largest magnitude so far, as a bit pattern: those have the magnitudes' order, and a NaN lies above infinity; 16-bit ones are compared
// in pairs (top_of makes one float32 pattern of them).
template <typename T, int V>
__device__ __forceinline__ void look(uint32_t& top, const Packed<T, V>& y) {
  if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
    for (int v = 0; v < V / 2; ++v) top = __vmaxu2(top, reinterpret_cast<const uint32_t*>(&y)[v] & 0x7fff7fffu);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) top = max(top, __float_as_uint(y.get(v)) & 0x7fffffffu);
  }
}
template <typename T, int V>
__device__ __forceinline__ uint32_t top_of(uint32_t top) {
  if constexpr (sizeof(T) == 2 && V > 1) {
    const unsigned short h = static_cast<unsigned short>(max(top & 0xffffu, top >> 16));
    top = __float_as_uint(to_f32<T>(*reinterpret_cast<const T*>(&h)));
  }
  return __reduce_max_sync(kFull, top);
}

// The nearest integers of x times a little less and a little more than 1 / scale: where they are one it is that of x / scale, else the
// division decides (one vector in 500; with a division for each of 33 million elements the kernel took 44 us).  kRound: a float32 whose
// unit is 1, so that adding it rounds to nearest even and leaves the integer in the low bits.  Scales below 2^-126 have no reciprocal to
// work with.
struct RowScale {
  bool finite, divide;
  float scale, less, more;
  __device__ __forceinline__ explicit RowScale(uint32_t top) {
    finite = top < 0x7f800000u;
    scale = finite ? __uint_as_float(top) / 127.f : __uint_as_float(0x7fc00000u);
    const bool zeros = !finite || scale == 0.f;
    const float inverse = zeros ? 0.f : 1.f / scale;
    less = inverse * (1.f - 0x1p-20f);
    more = inverse * (1.f + 0x1p-20f);
    divide = !zeros && !(inverse < 1e38f);
  }
  template <typename T, int V>
  __device__ __forceinline__ void put(int8_t* q, const Packed<T, V>& y) const {
    constexpr float kRound = 12582912.f;
    uint32_t b[V], apart = divide;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float z = y.get(v);
      b[v] = __float_as_uint(fmaf(z, less, kRound));
      apart |= b[v] ^ __float_as_uint(fmaf(z, more, kRound));
    }
    if (apart) {
#pragma unroll
      for (int v = 0; v < V; ++v) b[v] = static_cast<uint32_t>(max(-127, min(127, __float2int_rn(y.get(v) / scale))));
    }
    if (!finite) {
#pragma unroll
      for (int v = 0; v < V; ++v) b[v] = 0u;
    }
    if constexpr (V == 2) {
      *reinterpret_cast<unsigned short*>(q) = static_cast<unsigned short>(__byte_perm(b[0], b[1], 0x0040));
    } else if constexpr (V >= 4) {
      uint32_t w[V / 4];
#pragma unroll
      for (int v = 0; v < V / 4; ++v) w[v] = __byte_perm(__byte_perm(b[4 * v], b[4 * v + 1], 0x0040), __byte_perm(b[4 * v + 2], b[4 * v + 3], 0x0040), 0x5410);
      if constexpr (V == 8) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(q) = w[0];
    } else {
      q[0] = static_cast<int8_t>(b[0]);
    }
  }
};

template <typename T, int V, int WARPS>
__global__ void __launch_bounds__(128, 7) quantize_rows_kernel(const __grid_constant__ QuantizeParams p) {
  using P = Packed<T, V>;
  constexpr int kKeep = V <= 2 ? 16 : 8;
  __shared__ uint32_t found[4];
  pdl_wait();
  pdl_trigger();
  constexpr int kRowThreads = WARPS * 32;
  const int r = threadIdx.x / kRowThreads, i0 = threadIdx.x % kRowThreads;
  const long long row = static_cast<long long>(blockIdx.x) * (128 / kRowThreads) + r;
  const bool on = row < p.rows;
  const P* x = reinterpret_cast<const P*>(static_cast<const T*>(p.X) + row * p.x_stride);
  const int n = on ? p.C / V : 0;
  P kept[kKeep];
  uint32_t top = 0u;
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if (i0 + j * kRowThreads < n) kept[j] = x[i0 + j * kRowThreads];
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if (i0 + j * kRowThreads < n) look(top, kept[j]);
  for (int i = i0 + kKeep * kRowThreads; i < n; i += kRowThreads) look(top, x[i]);
  top = top_of<T, V>(top);
  if (WARPS > 1) {
    if ((threadIdx.x & 31) == 0) found[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = max(top, found[w]);
  }
  const RowScale scale(top);
  if (on && i0 == 0) p.scale[row] = scale.scale;
  int8_t* q = p.q + row * p.q_stride;
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if (i0 + j * kRowThreads < n) scale.put(q + (i0 + j * kRowThreads) * V, kept[j]);
  for (int i = i0 + kKeep * kRowThreads; i < n; i += kRowThreads) scale.put(q + static_cast<long long>(i) * V, x[i]);
}

// Many short rows: a warp has one after the other, with the next one on its way to shared memory (each vector to the thread that reads it)
// while it looks through this one.  bf16, this and the kernel above: 60000 rows of 128 23 and 31 us, 65536 of 512 35 and 41, 12000 of 128 8 and
// 10; but 16384 of 2048 29 and 27, 8192 of 4096 37 and 31: longer rows leave too few warps on an SM.
constexpr int kStreamWarps = 4, kStreamCtas = 148 * 12, kStreamSmem = kStreamWarps * 2 * 2048;
template <typename T>
__global__ void __launch_bounds__(kStreamWarps * 32) quantize_stream_kernel(const __grid_constant__ QuantizeParams p) {
  constexpr int V = 16 / sizeof(T);
  using P = Packed<T, V>;
  extern __shared__ __align__(16) unsigned char stream_smem[];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = p.C / V;
  P* ring = reinterpret_cast<P*>(stream_smem) + warp * 2 * n;
  const int stride = gridDim.x * kStreamWarps;
  auto ask = [&](long long row, int half) {
    if (row < p.rows) {
      const P* x = reinterpret_cast<const P*>(static_cast<const T*>(p.X) + row * p.x_stride);
      for (int i = lane; i < n; i += 32)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(ring + half * n + i))), "l"(x + i) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  long long row = blockIdx.x * kStreamWarps + warp;
  ask(row, 0);
  for (int half = 0; row < p.rows; row += stride, half ^= 1) {
    ask(row + stride, half ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const P* x = ring + half * n;
    uint32_t top = 0u;
#pragma unroll 4
    for (int i = lane; i < n; i += 32) look(top, x[i]);
    const RowScale scale(top_of<T, V>(top));
    if (lane == 0) p.scale[row] = scale.scale;
    int8_t* q = p.q + row * p.q_stride;
#pragma unroll 2
    for (int i = lane; i < n; i += 32) scale.put(q + i * V, x[i]);
  }
}

// ------------------------------------------------------------------------------------------------
// Products over ragged rows on the CUDA cores, any width and alignment: rows of 16 and 8 bits, weight gradients of 16 bits and of few float32
// features (the other float32 products are below).  Tiles of 64 x 64, a step of 16 contraction elements,
// 4 x 4 products a thread; float32 (8-bit operands: int32) sums.
// ------------------------------------------------------------------------------------------------
constexpr int kGTile = 64, kGStep = 16;

// The tile-th block of `rows` rows of an expert: its expert, its first sorted row and the expert's end; expert -1 behind the last block.  By all
// threads, with a barrier at the end: the offsets come to shared memory together (warp by warp they were four dependent loads for 111
// experts, more time than the eight steps of a tile behind them).
struct Block {
  int expert, first, end;
  int offsets[EGS_MAX_EXPERTS + 1];
};
__device__ __forceinline__ void locate_block(const int* offsets, int E, int rows, int tile, Block* b) {
  for (int e = threadIdx.x; e <= E; e += blockDim.x) b->offsets[e] = offsets[e];
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int seen = 0, e_found = -1, first_found = 0, end_found = 0;
    for (int e0 = 0; e0 < E && e_found < 0; e0 += 32) {
      const int e = e0 + lane;
      const int a = e < E ? b->offsets[e] : 0, end = e < E ? b->offsets[e + 1] : 0;
      const int blocks = static_cast<int>((static_cast<unsigned>(end - a) + rows - 1) / rows);     // (`rows` may be nearly all)
      int incl = blocks;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned hit = __ballot_sync(kFull, seen + incl > tile);
      if (hit) {
        const int src = __ffs(hit) - 1;
        const int f = a + (tile - seen - (incl - blocks)) * rows;
        e_found = e0 + src;
        first_found = __shfl_sync(kFull, f, src);
        end_found = __shfl_sync(kFull, end, src);
      }
      seen += __shfl_sync(kFull, incl, 31);
    }
    if (lane == 0) {
      b->expert = e_found;
      b->first = first_found;
      b->end = end_found;
    }
  }
  __syncthreads();
}

template <typename T> struct Acc { using type = float; };
template <> struct Acc<int8_t> { using type = int; };
template <typename T> __device__ __forceinline__ typename Acc<T>::type widen(T v) { return to_f32<T>(v); }
template <> __device__ __forceinline__ int widen<int8_t>(int8_t v) { return v; }
__device__ __forceinline__ float mac(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ int mac(int a, int b, int c) { return a * b + c; }

template <typename T> __device__ __forceinline__ float four(const Packed<T, 4>& x, int i) { return x.get(i); }
__device__ __forceinline__ int four(const Packed<int8_t, 4>& x, int i) { return x.raw[i]; }

// Four elements of a row from `p` on, `left` of which exist (p is not looked at where that is none); `wide`: they may be loaded together.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int left, bool wide, typename Acc<T>::type (&v)[4]) {
  if (wide && left >= 4) {
    const Packed<T, 4> x = *reinterpret_cast<const Packed<T, 4>*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = four(x, i);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? widen<T>(p[i]) : 0;
  }
}

// Rows behind the last expert's: zeros.
template <typename T>
__device__ __forceinline__ void zero_unrouted(const RaggedParams& p, int routed) {
  T* out = static_cast<T*>(p.Out);
  if (routed < p.rows) zero_by_grid(out + static_cast<long long>(routed) * p.N, out + static_cast<long long>(p.rows) * p.N);
}

// A step in shared memory, contraction by contraction; two of them, so that the next one is written while this one is read.
template <typename A>
struct alignas(16) GenericTile {
  A a[2][kGStep][kGTile + 4], b[2][kGStep][kGTile + 4];
};
template <typename A>
__device__ __forceinline__ void multiply(const GenericTile<A>& s, int buf, int tx, int ty, A (&acc)[4][4]) {
#pragma unroll
  for (int c = 0; c < kGStep; ++c) {
    const Packed<A, 4> a = *reinterpret_cast<const Packed<A, 4>*>(&s.a[buf][c][ty * 4]), b = *reinterpret_cast<const Packed<A, 4>*>(&s.b[buf][c][tx * 4]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mac(a.raw[i], b.raw[j], acc[i][j]);
  }
}

template <typename T, typename OutT>
__global__ void __launch_bounds__(256) ragged_rows_kernel(const __grid_constant__ RaggedParams p) {
  using A = typename Acc<T>::type;
  __shared__ GenericTile<A> s;
  __shared__ Block block;
  __shared__ int src[kGTile];
  pdl_wait();
  const int tid = threadIdx.x;
  int e = 0, first = blockIdx.x * kGTile, end = p.rows;
  if (p.offsets) {
    locate_block(p.offsets, p.E, kGTile, blockIdx.x, &block);
    e = block.expert;
    first = block.first;
    end = block.end;
    zero_unrouted<OutT>(p, block.offsets[p.E]);
  }
  if (e < 0) return;
  if (tid < kGTile) src[tid] = first + tid >= end ? -1 : p.slots ? p.by_k.quotient(p.slots[first + tid]) : first + tid;
  __syncthreads();
  const T* W = static_cast<const T*>(p.W) + e * p.w_expert;
  const int n0 = column_tile() * kGTile, tx = tid & 15, ty = tid >> 4;
  // of A (and of weights [E, N, C]): row tid / 4, elements 4 (tid mod 4) ..;  of weights [E, C, N]: row tid / 16
  const int lr = tid >> 2, lc = (tid & 3) * 4, row = src[lr];
  const T* a_row = static_cast<const T*>(p.A) + (row < 0 ? 0 : row) * p.a_row;
  const bool a_wide = p.a_row % 4 == 0 && (reinterpret_cast<uintptr_t>(p.A) % sizeof(Packed<T, 4>)) == 0;
  const bool w_wide = p.w_row % 4 == 0 && p.w_expert % 4 == 0 && (reinterpret_cast<uintptr_t>(p.W) % sizeof(Packed<T, 4>)) == 0;
  A va[4], vb[4];
  auto fetch = [&](int c0) {
    load4<T>(a_row + c0 + lc, row < 0 ? 0 : p.C - c0 - lc, a_wide, va);
    if (p.nc) load4<T>(W + (n0 + lr) * p.w_row + c0 + lc, n0 + lr < p.N ? p.C - c0 - lc : 0, w_wide, vb);
    else load4<T>(W + (c0 + ty) * p.w_row + n0 + tx * 4, c0 + ty < p.C ? p.N - n0 - tx * 4 : 0, w_wide, vb);
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s.a[buf][lc + i][lr] = va[i];
    if (p.nc) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s.b[buf][lc + i][lr] = vb[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) s.b[buf][ty][tx * 4 + i] = vb[i];
    }
  };
  A acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0;
  if (p.C > 0) {
    fetch(0);
    put(0);
  }
  __syncthreads();
  for (int c0 = 0, buf = 0; c0 < p.C; c0 += kGStep, buf ^= 1) {
    const bool more = c0 + kGStep < p.C;
    if (more) fetch(c0 + kGStep);
    multiply(s, buf, tx, ty, acc);
    if (more) put(buf ^ 1);
    __syncthreads();
  }
  OutT* out = static_cast<OutT*>(p.Out);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = ty * 4 + i;
    if (src[m] < 0) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n >= p.N) continue;
      float v = static_cast<float>(acc[i][j]);
      if (p.a_scale) v *= p.a_scale[src[m]] * p.w_scale[static_cast<long long>(e) * p.N + n];
      out[static_cast<long long>(first + m) * p.N + n] = from_f32<OutT>(v);
    }
  }
}

// dW[e, c, n] = sum over the rows of e of X[row, c] dY[row, n].  Where `length` is not 0 a CTA has that many rows of an expert at most; the sums of
// all those ranges go to the workspace [range, C, N] and are added in their order by a second kernel.  (Equal numbers of ranges for all
// experts left the CTAs of the largest ones at work alone: 44 us for 32 experts of 128 x 64 float32.)
struct DweightRange {
  int expert, first, end;
};
__device__ __forceinline__ DweightRange range_of(const RaggedParams& p, int length, Block* block) {
  if (length == 0) return {static_cast<int>(blockIdx.z), p.offsets[blockIdx.z], p.offsets[blockIdx.z + 1]};
  locate_block(p.offsets, p.E, length, blockIdx.z, block);
  return {block->expert, block->first, block->end - block->first > length ? block->first + length : block->end};
}
template <typename T>
__global__ void __launch_bounds__(256) ragged_dweight_kernel(const __grid_constant__ RaggedParams p, int length, float* partial) {
  __shared__ Block block;
  __shared__ GenericTile<float> s;
  pdl_wait();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const DweightRange range = range_of(p, length, &block);
  if (range.expert < 0) return;
  const int e = range.expert, first = range.first, end = range.end;
  const int tiles_n = (p.N + kGTile - 1) / kGTile;
  const int c0 = blockIdx.x / tiles_n * kGTile, n0 = blockIdx.x % tiles_n * kGTile;
  const T* X = static_cast<const T*>(p.A);
  const T* Y = static_cast<const T*>(p.W);
  const bool a_wide = p.a_row % 4 == 0 && (reinterpret_cast<uintptr_t>(p.A) % sizeof(Packed<T, 4>)) == 0;
  const bool w_wide = p.w_row % 4 == 0 && (reinterpret_cast<uintptr_t>(p.W) % sizeof(Packed<T, 4>)) == 0;
  float va[4], vb[4];
  int source = -1;                             // row of X in the step to come
  auto look = [&](int r0) {
    const int r = r0 + ty;
    source = r >= end ? -1 : p.slots ? p.slots[r] : r;
  };
  auto fetch = [&](int r0) {
    const long long row = source < 0 ? -1 : p.slots ? p.by_k.quotient(source) : source;
    load4<T>(X + (row < 0 ? 0 : row) * p.a_row + c0 + tx * 4, row < 0 ? 0 : p.C - c0 - tx * 4, a_wide, va);
    load4<T>(Y + (r0 + ty < end ? r0 + ty : 0) * p.w_row + n0 + tx * 4, r0 + ty < end ? p.N - n0 - tx * 4 : 0, w_wide, vb);
    look(r0 + kGStep);
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s.a[buf][ty][tx * 4 + i] = va[i];
      s.b[buf][ty][tx * 4 + i] = vb[i];
    }
  };
  float acc[4][4] = {};
  if (first < end) {
    look(first);
    fetch(first);
    put(0);
  }
  __syncthreads();
  for (int r0 = first, buf = 0; r0 < end; r0 += kGStep, buf ^= 1) {
    const bool more = r0 + kGStep < end;
    if (more) fetch(r0 + kGStep);
    multiply(s, buf, tx, ty, acc);
    if (more) put(buf ^ 1);
    __syncthreads();
  }
  const long long size = static_cast<long long>(p.C) * p.N;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (c >= p.C || n >= p.N) continue;
      const long long at = static_cast<long long>(c) * p.N + n;
      if (length) partial[blockIdx.z * size + at] = acc[i][j];
      else static_cast<T*>(p.Out)[e * size + at] = from_f32<T>(acc[i][j]);
    }
}

// ------------------------------------------------------------------------------------------------
// float32, where experts have rows enough: tiles of 128 x 64, 8 x 8 products a thread, two of them an instruction (fma.rn.f32x2, pairs of
// rows).  What bounds it is reads of shared memory, which cost by the bytes a lane asks for, equal addresses or not: 16 floats for 64
// products are as long as the products (8 x 4 products a thread: 36 TFLOP/s, the load unit at 85 %).
// ------------------------------------------------------------------------------------------------
constexpr int kWide = 128, kWideThreads = 128;

struct alignas(16) WideTile {
  float a[2][kGStep][kWide + 4], b[2][kGStep][kGTile + 4];
};
__device__ __forceinline__ unsigned long long pack(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void fma2(unsigned long long& c, unsigned long long a, unsigned long long b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}
// acc[i][j]: rows 8 ty + 2 i and the next one; columns 4 tx + j and 32 + 4 tx + j - 4
template <int STEP = kGStep>
__device__ __forceinline__ void multiply_wide(const WideTile& s, int buf, int tx, int ty, unsigned long long (&acc)[4][8]) {
#pragma unroll
  for (int c = 0; c < STEP; ++c) {
    const ulonglong2 a0 = *reinterpret_cast<const ulonglong2*>(&s.a[buf][c][ty * 8]), a1 = *reinterpret_cast<const ulonglong2*>(&s.a[buf][c][ty * 8 + 4]);
    const float4 b0 = *reinterpret_cast<const float4*>(&s.b[buf][c][tx * 4]), b1 = *reinterpret_cast<const float4*>(&s.b[buf][c][32 + tx * 4]);
    const float b[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
    const unsigned long long aa[4] = {a0.x, a0.y, a1.x, a1.y};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned long long bb = pack(b[j], b[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) fma2(acc[i][j], aa[i], bb);
    }
  }
}
__device__ __forceinline__ float half_of(unsigned long long v, int high) { return __uint_as_float(static_cast<uint32_t>(high ? v >> 32 : v)); }
// f(row of the tile, first of four columns, the four values)
template <class F>
__device__ __forceinline__ void each_of(const unsigned long long (&acc)[4][8], int tx, int ty, F&& f) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = half_of(acc[i / 2][h * 4 + j], i & 1);
      f(ty * 8 + i, h * 32 + tx * 4, v);
    }
}
__device__ __forceinline__ void store_up_to4(float* to, int left, bool wide, const float (&v)[4]) {
  if (wide && left >= 4) {
    *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) to[j] = v[j];
  }
}

__global__ void __launch_bounds__(kWideThreads, 3) ragged_rows_f32_kernel(const __grid_constant__ RaggedParams p) {
  __shared__ WideTile s;
  __shared__ Block block;
  __shared__ int src[kWide];
  pdl_wait();
  const int tid = threadIdx.x;
  locate_block(p.offsets, p.E, kWide, blockIdx.x, &block);
  const int e = block.expert, first = block.first, end = block.end;
  zero_unrouted<float>(p, block.offsets[p.E]);
  if (e < 0) return;
  src[tid] = first + tid >= end ? -1 : p.slots ? p.by_k.quotient(p.slots[first + tid]) : first + tid;
  const float* W = static_cast<const float*>(p.W) + e * p.w_expert;
  const int n0 = column_tile() * kGTile, tx = tid & 7, ty = tid >> 3;
  // X (and weights [E, N, C]): rows tid / 4 and every 32nd from there, elements 4 (tid mod 4) ..;  weights [E, C, N]: rows tid / 16 and 8 more
  const int lr = tid >> 2, lc = (tid & 3) * 4, wr = tid >> 4, wc = (tid & 15) * 4;
  const bool a_wide = p.a_row % 4 == 0 && (reinterpret_cast<uintptr_t>(p.A) & 15u) == 0;
  const bool w_wide = p.w_row % 4 == 0 && p.w_expert % 4 == 0 && (reinterpret_cast<uintptr_t>(p.W) & 15u) == 0;
  float va[4][4], vb[2][4];
  auto fetch_w = [&](int c0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (p.nc) load4<float>(W + (n0 + lr + 32 * h) * p.w_row + c0 + lc, n0 + lr + 32 * h < p.N ? p.C - c0 - lc : 0, w_wide, vb[h]);
      else load4<float>(W + (c0 + wr + 8 * h) * p.w_row + n0 + wc, c0 + wr + 8 * h < p.C ? p.N - n0 - wc : 0, w_wide, vb[h]);
    }
  };
  fetch_w(0);
  __syncthreads();
  int row[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) row[h] = src[lr + 32 * h];
  auto fetch_x = [&](int c0) {
#pragma unroll
    for (int h = 0; h < 4; ++h)
      load4<float>(static_cast<const float*>(p.A) + (row[h] < 0 ? 0 : row[h]) * p.a_row + c0 + lc, row[h] < 0 ? 0 : p.C - c0 - lc, a_wide, va[h]);
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) s.a[buf][lc + i][lr + 32 * h] = va[h][i];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (p.nc) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s.b[buf][lc + i][lr + 32 * h] = vb[h][i];
      } else {
        *reinterpret_cast<float4*>(&s.b[buf][wr + 8 * h][wc]) = make_float4(vb[h][0], vb[h][1], vb[h][2], vb[h][3]);
      }
    }
  };
  unsigned long long acc[4][8] = {};
  fetch_x(0);
  put(0);
  __syncthreads();
  for (int c0 = 0, buf = 0; c0 < p.C; c0 += kGStep, buf ^= 1) {
    const bool more = c0 + kGStep < p.C;
    if (more) {
      fetch_x(c0 + kGStep);
      fetch_w(c0 + kGStep);
    }
    multiply_wide(s, buf, tx, ty, acc);
    if (more) put(buf ^ 1);
    __syncthreads();
  }
  float* out = static_cast<float*>(p.Out) + static_cast<long long>(first) * p.N + n0;
  const bool wide = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.Out) & 15u) == 0;
  each_of(acc, tx, ty, [&](int m, int n, const float (&v)[4]) {
    if (src[m] >= 0) store_up_to4(out + static_cast<long long>(m) * p.N + n, p.N - n0 - n, wide, v);
  });
}

// ------------------------------------------------------------------------------------------------
// float32, where experts have a few rows or tens: tiles of 32 x 64, whose work is reading weights.  Three steps of 32 contraction elements are on
// their way by cp.async.  G groups of 64 threads have a part of each step; their sums are joined, in order, at the end (one group alone, five
// CTAs on an SM, left the load unit waiting: 64 experts of 32 rows, 1024 x 512, 114 us, two groups 82; 16 of 2048 x 1024, of which an SM has
// fewer than two CTAs: 158, two 121, four 88 - but four 88 in the first case, where there are CTAs enough).  Threads have rows ty, ty + 4, ..
// and as many of them as the block has.  Weights [E, N, C]: the two halves of a fma.rn.f32x2 are even and odd contraction elements, both operands
// lie in pairs; [E, C, N]: neighbouring columns.  12 floats of shared memory for 32 products hold it to 36 TFLOP/s.
// ------------------------------------------------------------------------------------------------
constexpr int kMidRows = 32, kMidCols = 64, kMidStep = 32, kMidStages = 3;
constexpr int kMidPitch = kMidStep + 4;      // floats: eight rows are in different banks
constexpr int kMidStage = kMidRows * kMidPitch + (kMidCols * kMidPitch > kMidStep * (kMidCols + 4) ? kMidCols * kMidPitch : kMidStep * (kMidCols + 4));
constexpr int kMidSmem = kMidStages * kMidStage * 4;

// Four floats to shared memory, `left` of which exist; zeros for the others.
__device__ __forceinline__ void copy4(float* dst, const float* src, int left, bool wide) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if (wide) {
    const int bytes = left >= 4 ? 16 : left > 0 ? left * 4 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(bytes) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + i * 4), "l"(i < left ? src + i : src), "r"(i < left ? 4 : 0) : "memory");
  }
}

template <bool NC, int G, int R>
__device__ __forceinline__ void mid_tile(const RaggedParams& p, float* ring, const int* src, int e, int first, int rows) {
  constexpr int kThreads = 64 * G;
  constexpr int kX = (R * 32 + kThreads - 1) / kThreads, kWn = kMidCols * 8 / kThreads, kWc = kMidStep * 16 / kThreads;
  const int tid = threadIdx.x, tx = tid & 15, ty = (tid >> 4) & 3, group = tid >> 6, n0 = column_tile() * kMidCols;
  const float* A = static_cast<const float*>(p.A);
  const float* W = static_cast<const float*>(p.W) + e * p.w_expert;
  const bool a_wide = p.a_row % 4 == 0 && (reinterpret_cast<uintptr_t>(p.A) & 15u) == 0;
  const bool w_wide = p.w_row % 4 == 0 && p.w_expert % 4 == 0 && (reinterpret_cast<uintptr_t>(p.W) & 15u) == 0;
  const int lr = tid >> 3, lc = (tid & 7) * 4;
  const float* x[kX];
#pragma unroll
  for (int i = 0; i < kX; ++i) x[i] = lr + kThreads / 8 * i < rows ? A + src[lr + kThreads / 8 * i] * p.a_row : nullptr;
  auto issue = [&](int step) {
    const int c0 = step * kMidStep;
    if (c0 < p.C) {
      float* a = ring + step % kMidStages * kMidStage;
      float* b = a + kMidRows * kMidPitch;
#pragma unroll
      for (int i = 0; i < kX; ++i)
        if (x[i]) copy4(a + (lr + kThreads / 8 * i) * kMidPitch + lc, c0 + lc < p.C ? x[i] + c0 + lc : x[i], p.C - c0 - lc, a_wide);
#pragma unroll
      for (int i = 0; i < (NC ? kWn : kWc); ++i) {
        if (NC) {
          const int at = lr + kThreads / 8 * i;
          const float* w = W + (n0 + at) * p.w_row;
          if (n0 + at < p.N) copy4(b + at * kMidPitch + lc, c0 + lc < p.C ? w + c0 + lc : w, p.C - c0 - lc, w_wide);
        } else {
          const int at = (tid >> 4) + kThreads / 16 * i, c = c0 + at, n = n0 + tx * 4;
          if (n < p.N) copy4(b + at * (kMidCols + 4) + tx * 4, c < p.C ? W + c * p.w_row + n : W, c < p.C ? p.N - n : 0, w_wide);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  unsigned long long acc[R][NC ? 4 : 2] = {};
#pragma unroll
  for (int s = 0; s < kMidStages - 1; ++s) issue(s);
  for (int step = 0; step * kMidStep < p.C; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kMidStages - 2) : "memory");
    __syncthreads();
    issue(step + kMidStages - 1);
    const int part = group * (kMidStep / G);
    const float* a = ring + step % kMidStages * kMidStage + part;
    const float* b = ring + step % kMidStages * kMidStage + kMidRows * kMidPitch + (NC ? part : part * (kMidCols + 4));
#pragma unroll
    for (int c = 0; c < kMidStep / G; c += 4) {
      if (NC) {
        ulonglong2 bv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) bv[j] = *reinterpret_cast<const ulonglong2*>(b + (tx + 16 * j) * kMidPitch + c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const ulonglong2 av = *reinterpret_cast<const ulonglong2*>(a + (ty + 4 * i) * kMidPitch + c);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            fma2(acc[i][j], av.x, bv[j].x);
            fma2(acc[i][j], av.y, bv[j].y);
          }
        }
      } else {
        float4 av[R];
#pragma unroll
        for (int i = 0; i < R; ++i) av[i] = *reinterpret_cast<const float4*>(a + (ty + 4 * i) * kMidPitch + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(b + (c + k) * (kMidCols + 4) + tx * 4);
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const float v = k == 0 ? av[i].x : k == 1 ? av[i].y : k == 2 ? av[i].z : av[i].w;
            fma2(acc[i][0], pack(v, v), bv.x);
            fma2(acc[i][1], pack(v, v), bv.y);
          }
        }
      }
    }
  }
  float v[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[i][j] = NC ? half_of(acc[i][NC ? j : 0], 0) + half_of(acc[i][NC ? j : 0], 1) : half_of(acc[i][NC ? 0 : j / 2], j & 1);
  __syncthreads();                             // (the ring has been read: the other groups' sums take its place)
  float4* sums = reinterpret_cast<float4*>(ring) + (tid & 63);
  if (group > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) sums[((group - 1) * R + i) * 64] = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
  }
  __syncthreads();
  if (group > 0) return;
  float* out = static_cast<float*>(p.Out) + static_cast<long long>(first) * p.N + n0;
  const bool wide = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.Out) & 15u) == 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int m = ty + 4 * i;
    if (m >= rows) break;
#pragma unroll
    for (int g = 1; g < G; ++g) {
      const float4 x = sums[((g - 1) * R + i) * 64];
      v[i][0] += x.x;
      v[i][1] += x.y;
      v[i][2] += x.z;
      v[i][3] += x.w;
    }
    float* o = out + static_cast<long long>(m) * p.N;
    if (NC) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + tx + 16 * j < p.N) o[tx + 16 * j] = v[i][j];
    } else {
      store_up_to4(o + tx * 4, p.N - n0 - tx * 4, wide, v[i]);
    }
  }
}

template <bool NC, int G>
__global__ void __launch_bounds__(64 * G, G == 4 ? 2 : 4) ragged_rows_mid_kernel(const __grid_constant__ RaggedParams p) {
  extern __shared__ __align__(16) float mid_ring[];
  static_assert(sizeof(Block) <= kMidSmem, "the offsets, which give way to the ring");
  __shared__ int src[kMidRows];
  pdl_wait();
  const int tid = threadIdx.x;
  Block* block = reinterpret_cast<Block*>(mid_ring);
  locate_block(p.offsets, p.E, kMidRows, blockIdx.x, block);
  const int e = block->expert, first = block->first, rows = min(kMidRows, block->end - first), routed = block->offsets[p.E];
  zero_unrouted<float>(p, routed);
  if (e < 0) return;
  if (tid < rows) src[tid] = p.slots ? p.by_k.quotient(p.slots[first + tid]) : first + tid;
  __syncthreads();
  if (rows <= 8) mid_tile<NC, G, 2>(p, mid_ring, src, e, first, rows);
  else if (rows <= 16) mid_tile<NC, G, 4>(p, mid_ring, src, e, first, rows);
  else if (rows <= 24) mid_tile<NC, G, 6>(p, mid_ring, src, e, first, rows);
  else mid_tile<NC, G, 8>(p, mid_ring, src, e, first, rows);
}

// See ragged_dweight_kernel, whose ranges these are.
__global__ void __launch_bounds__(kWideThreads, 3) ragged_dweight_f32_kernel(const __grid_constant__ RaggedParams p, int length, float* partial) {
  __shared__ WideTile s;
  __shared__ Block block;
  pdl_wait();
  const int tid = threadIdx.x, tx = tid & 7, ty = tid >> 3;
  const DweightRange range = range_of(p, length, &block);
  if (range.expert < 0) return;
  const int e = range.expert, first = range.first, end = range.end;
  const int tiles_n = (p.N + kGTile - 1) / kGTile;
  const int c0 = blockIdx.x / tiles_n * kWide, n0 = blockIdx.x % tiles_n * kGTile;
  const float* X = static_cast<const float*>(p.A) + c0;
  const float* Y = static_cast<const float*>(p.W) + n0;
  const bool a_wide = p.a_row % 4 == 0 && (reinterpret_cast<uintptr_t>(p.A) & 15u) == 0;
  const bool w_wide = p.w_row % 4 == 0 && (reinterpret_cast<uintptr_t>(p.W) & 15u) == 0;
  // X: rows tid / 32 and every fourth from there, 4 (tid mod 32) ..;  dY: rows tid / 16 and 8 more, 4 (tid mod 16) ..
  const int xr = tid >> 5, xc = (tid & 31) * 4, yr = tid >> 4, yc = (tid & 15) * 4;
  float va[4][4], vb[2][4];
  int source[4];                               // slots (rows) of the step to come
  auto look = [&](int r0) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int r = r0 + xr + 4 * h;
      source[h] = r >= end ? -1 : p.slots ? p.slots[r] : r;
    }
  };
  auto fetch = [&](int r0) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const long long row = source[h] < 0 ? -1 : p.slots ? p.by_k.quotient(source[h]) : source[h];
      load4<float>(X + (row < 0 ? 0 : row) * p.a_row + xc, row < 0 ? 0 : p.C - c0 - xc, a_wide, va[h]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + yr + 8 * h;
      load4<float>(Y + (r < end ? r : 0) * p.w_row + yc, r < end ? p.N - n0 - yc : 0, w_wide, vb[h]);
    }
    look(r0 + kGStep);
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int h = 0; h < 4; ++h) *reinterpret_cast<float4*>(&s.a[buf][xr + 4 * h][xc]) = make_float4(va[h][0], va[h][1], va[h][2], va[h][3]);
#pragma unroll
    for (int h = 0; h < 2; ++h) *reinterpret_cast<float4*>(&s.b[buf][yr + 8 * h][yc]) = make_float4(vb[h][0], vb[h][1], vb[h][2], vb[h][3]);
  };
  unsigned long long acc[4][8] = {};
  if (first < end) {
    look(first);
    fetch(first);
    put(0);
  }
  __syncthreads();
  for (int r0 = first, buf = 0; r0 < end; r0 += kGStep, buf ^= 1) {
    const bool more = r0 + kGStep < end;
    if (more) fetch(r0 + kGStep);
    if (end - r0 > kGStep / 2) multiply_wide(s, buf, tx, ty, acc);
    else multiply_wide<kGStep / 2>(s, buf, tx, ty, acc);       // (an expert of 17 rows)
    if (more) put(buf ^ 1);
    __syncthreads();
  }
  const long long size = static_cast<long long>(p.C) * p.N;
  float* out = length ? partial + blockIdx.z * size : static_cast<float*>(p.Out) + e * size;
  const bool wide = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  each_of(acc, tx, ty, [&](int m, int n, const float (&v)[4]) {
    if (c0 + m < p.C) store_up_to4(out + static_cast<long long>(c0 + m) * p.N + n0 + n, p.N - n0 - n, wide, v);
  });
}

template <typename T>
__global__ void __launch_bounds__(256) dweight_join_kernel(const int* offsets, const float* partial, T* out, long long size, int length) {
  __shared__ int s_base, s_count;
  pdl_wait();
  const int expert = blockIdx.y, lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    int base = 0;
    auto ranges = [&](int e) { return static_cast<int>((static_cast<unsigned>(offsets[e + 1] - offsets[e]) + length - 1) / length); };
    for (int e = lane; e < expert; e += 32) base += ranges(e);
    base = __reduce_add_sync(kFull, base);
    if (lane == 0) {
      s_base = base;
      s_count = ranges(expert);
    }
  }
  __syncthreads();
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= size) return;
  const float* p = partial + s_base * size + i;
  const int n = s_count;
  float sum = 0.f;
#pragma unroll 8
  for (int r = 0; r < n; ++r) sum += p[r * size];
  out[expert * size + i] = from_f32<T>(sum);
}

// Rows of 16-bit elements with another pitch; a thread writes eight elements.  Two matrices with one launch.
struct PadMatrix {
  const unsigned short* src;
  uint4* dst;
  long long vectors;
  int width, per_row;
};
__global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ PadMatrix a, const __grid_constant__ PadMatrix b) {
  pdl_wait();
  long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const bool second = i >= a.vectors;
  if (second) i -= a.vectors;
  if (second && i >= b.vectors) return;
  const int width = second ? b.width : a.width, per_row = second ? b.per_row : a.per_row;
  const long long row = i / per_row;
  const int c = static_cast<int>(i - row * per_row) * 8;
  const unsigned short* s = (second ? b.src : a.src) + row * width + c;
  unsigned short v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < width ? s[j] : 0;
  (second ? b.dst : a.dst)[i] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, int NPER>
cudaError_t route_n(RouteParams& p, cudaStream_t st) {
  const int lanes = p.per / NPER;
  p.whole_lanes = p.per % NPER == 0 && (lanes & (lanes - 1)) == 0;
  if (p.whole_lanes) {
    p.lanes_log2 = 0;
    while ((1 << p.lanes_log2) < lanes) ++p.lanes_log2;
  }
  p.vectors = p.E == 32 * NPER && (p.stride * sizeof(T)) % 16 == 0 && aligned(p.logits) && (!p.bias || aligned(p.bias));
  p.warp_words = p.groups > 1 && !p.whole_lanes && p.E > 64 ? (p.E + 3) / 4 * 4 : 64;      // (read 16 bytes at a time)
  const size_t smem = sizeof(uint32_t) * kRouteWarps * p.warp_words;
  return launch_kernel(route_tokens_kernel<T, NPER>, (p.tokens + kRouteWarps - 1) / kRouteWarps, kRouteWarps * 32, smem, st, true, p);
}
template <typename T>
cudaError_t route_t(RouteParams& p, cudaStream_t st) {
  if (p.E <= 32) return route_n<T, 1>(p, st);
  if (p.E <= 64) return route_n<T, 2>(p, st);
  if (p.E <= 128) return route_n<T, 4>(p, st);
  if (p.E <= 256) return route_n<T, 8>(p, st);
  if (p.E <= 512) return route_n<T, 16>(p, st);
  return route_n<T, 32>(p, st);
}

template <class F16, class BF16, class F32>
cudaError_t by_type(int dtype, F16&& f16, BF16&& bf16, F32&& f32) {
  return dtype == EGS_F16 ? f16() : dtype == EGS_BF16 ? bf16() : f32();
}

template <typename T, typename O, int V>
cudaError_t combine_v(CombineParams& p, bool backward, cudaStream_t st) {
  p.vecs = p.N / V;
  if (backward) {
    const long long slots = static_cast<long long>(p.tokens) * p.k;
    if (p.vecs <= 16) {
      int lanes_log2 = 2;
      while ((1 << lanes_log2) < p.vecs) ++lanes_log2;
      const long long ctas = ((slots << lanes_log2) + 255) / 256;
      p.by_k = Div(p.k);
      return launch_kernel(combine_backward_narrow_kernel<T, V>, static_cast<unsigned>(ctas < kNarrowCtas ? ctas : kNarrowCtas), 256, 0, st, true, p, lanes_log2);
    }
    return launch_kernel(combine_backward_kernel<T, V>, static_cast<unsigned>((slots + 7) / 8), 256, 0, st, true, p);
  }
  if constexpr (sizeof(T) * V < 4) {
    return launch_kernel(combine_columns_kernel<T, O>, (p.tokens + 3) / 4, 256, 0, st, true, p);
  } else {
    if (p.vecs <= 32) {
      int lanes_log2 = 2;
      while ((1 << lanes_log2) < p.vecs) ++lanes_log2;
      return launch_kernel(combine_narrow_kernel<T, O, V>, static_cast<unsigned>(((static_cast<long long>(p.tokens) << lanes_log2) + 255) / 256), 256, 0, st, true, p, lanes_log2);
    }
    const int blocks = (p.vecs * static_cast<int>(sizeof(T) * V) + 511) / 512;
    p.by_blocks = Div(blocks);
    p.work = p.tokens * blocks;
    const int ctas = (p.work + kCombineWarps - 1) / kCombineWarps;
    return launch_kernel(combine_kernel<T, O, V>, ctas < kCombineCtas ? ctas : kCombineCtas, kCombineWarps * 32, 0, st, true, p);
  }
}
// The widest vectors that rows of N elements are whole numbers of and begin on.
template <typename T, typename O = T>
cudaError_t combine_t(CombineParams& p, bool backward, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](int v) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.Y) | reinterpret_cast<uintptr_t>(p.dOut);
    return p.N % v == 0 && all % (v * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p.out) % (v * sizeof(O)) == 0;
  };
  if (fits(V)) return combine_v<T, O, V>(p, backward, st);
  if (fits(V / 2)) return combine_v<T, O, V / 2>(p, backward, st);
  if constexpr (V > 4) {
    if (fits(V / 4)) return combine_v<T, O, V / 4>(p, backward, st);
  }
  return combine_v<T, O, 1>(p, backward, st);
}

template <typename T, int V>
cudaError_t quantize_v(const QuantizeParams& p, cudaStream_t st) {
  if (p.C <= 32 * V * (V <= 2 ? 16 : 8)) return launch_kernel(quantize_rows_kernel<T, V, 1>, (p.rows + 3) / 4, 128, 0, st, true, p);
  return launch_kernel(quantize_rows_kernel<T, V, 4>, p.rows, 128, 0, st, true, p);
}
template <typename T>
cudaError_t quantize_t(const QuantizeParams& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](int v) {
    return p.C % v == 0 && p.x_stride % v == 0 && reinterpret_cast<uintptr_t>(p.X) % (v * sizeof(T)) == 0 && p.q_stride % v == 0 &&
           reinterpret_cast<uintptr_t>(p.q) % v == 0;
  };
  if (fits(V)) {
    const size_t smem = static_cast<size_t>(kStreamWarps) * 2 * p.C * sizeof(T);
    if (smem <= kStreamSmem && p.rows > kStreamCtas * kStreamWarps) return launch_kernel(quantize_stream_kernel<T>, kStreamCtas, kStreamWarps * 32, smem, st, true, p);
    return quantize_v<T, V>(p, st);
  }
  if (fits(2)) return quantize_v<T, 2>(p, st);
  return quantize_v<T, 1>(p, st);
}

}  // namespace

cudaError_t launch_route_tokens(const void* logits, const float* bias, float* weights, int* experts, const egs_route& r, long long stride,
                                int dtype, cudaStream_t st) {
  RouteParams p{};
  p.logits = logits; p.bias = bias; p.weights = weights; p.experts = experts; p.stride = stride;
  p.tokens = static_cast<int>(r.tokens); p.E = r.E; p.k = r.top_k; p.groups = r.groups; p.top_groups = r.top_groups;
  p.group_top = r.group_top; p.per = r.E / r.groups; p.by_per = Div(p.per);
  p.sigmoid = r.score == EGS_SCORE_SIGMOID; p.renormalize = r.renormalize; p.scale = r.scale;
  while ((32 >> p.lanes_log2) > 1 && (32 >> (p.lanes_log2 + 1)) >= r.groups) ++p.lanes_log2;
  count_launch();
  return by_type(dtype, [&] { return route_t<__half>(p, st); }, [&] { return route_t<__nv_bfloat16>(p, st); }, [&] { return route_t<float>(p, st); });
}

cudaError_t launch_route_backward(const float* dweights, const void* logits, const int* experts, void* dlogits, const egs_route& r,
                                  long long stride, int dtype, cudaStream_t st) {
  RouteBackwardParams p{};
  p.dweights = dweights; p.logits = logits; p.experts = experts; p.dlogits = dlogits; p.stride = stride;
  p.tokens = static_cast<int>(r.tokens); p.E = r.E; p.k = r.top_k;
  p.sigmoid = r.score == EGS_SCORE_SIGMOID; p.renormalize = r.renormalize; p.scale = r.scale;
  p.vectors = (r.E * (dtype == EGS_F32 ? 4 : 2)) % 16 == 0 && aligned(dlogits);
  const int grid = (p.tokens + kRouteWarps - 1) / kRouteWarps;
  count_launch();
  auto go = [&](auto kernel) { return launch_kernel(kernel, grid, kRouteWarps * 32, 0, st, true, p); };
  return by_type(dtype, [&] { return go(route_backward_kernel<__half>); }, [&] { return go(route_backward_kernel<__nv_bfloat16>); },
                 [&] { return go(route_backward_kernel<float>); });
}

// Slots of a warp: 128, 256 where a cluster then is enough, more where there would be more than 256 stretches of them.
static long long plan_part(long long n) {
  if (n > 128ll * kPlanWarps * kPlanCluster && n <= 256ll * kPlanWarps * kPlanCluster) return 256;
  const long long part = (n + 256ll * kPlanWarps - 1) / (256ll * kPlanWarps);
  return part < 128 ? 128 : (part + 31) / 32 * 32;
}
static long long plan_stretches(long long n) {
  const long long stretch = plan_part(n) * kPlanWarps;
  return n ? (n + stretch - 1) / stretch : 1;
}
size_t plan_workspace_ints(long long n, int E) { return plan_stretches(n) <= kPlanCluster ? 0 : static_cast<size_t>(plan_stretches(n)) * (E + 1); }

template <int S>
static cudaError_t launch_plan_place(const PlanParams& p, size_t smem, cudaStream_t st) {
  cudaError_t err = ensure_smem_optin<plan_place_kernel<S>>(sizeof(int) * (kPlanWarps + 2) * (EGS_MAX_EXPERTS + 1));
  if (err != cudaSuccess) return err;
  if constexpr (S > 8) {
    static thread_local int done_device = -1;
    int dev = 0;
    if ((err = cudaGetDevice(&dev)) != cudaSuccess) return err;
    if (done_device != dev && (err = cudaFuncSetAttribute(plan_place_kernel<S>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return err;
    done_device = dev;
  }
  count_launch();
  return launch_kernel(plan_place_kernel<S>, S > 1 ? S : p.stretches, kPlanThreads, smem, st, true, p);
}

cudaError_t launch_plan_experts(const int* experts, long long n, int E, int* offsets, int* slots, int* position, int* workspace,
                                StatusRef status, cudaStream_t st) {
  const PlanParams p{experts, offsets, slots, position, workspace, static_cast<int>(n), E, static_cast<int>(plan_part(n)), static_cast<int>(plan_stretches(n)), status};
  const size_t smem = sizeof(int) * (kPlanWarps + 2) * (E + 1);
  if (p.stretches > 1 && p.stretches <= kPlanCluster) {
    if (p.stretches <= 2) return launch_plan_place<2>(p, smem, st);
    if (p.stretches <= 4) return launch_plan_place<4>(p, smem, st);
    if (p.stretches <= 8) return launch_plan_place<8>(p, smem, st);
    return launch_plan_place<16>(p, smem, st);
  }
  if (p.stretches > 1) {
    cudaError_t err = ensure_smem_optin<plan_count_kernel>(sizeof(int) * (kPlanWarps + 2) * (EGS_MAX_EXPERTS + 1));
    if (err != cudaSuccess) return err;
    err = launch_kernel(plan_count_kernel, p.stretches, kPlanThreads, smem, st, true, p);
    count_launch();
    if (err != cudaSuccess) return err;
  }
  return launch_plan_place<1>(p, smem, st);
}

cudaError_t launch_combine(const void* Y, const void* weights, const int* position, void* out, long long tokens, int k, int N, int dtype,
                           int w_f32, int out_dtype, cudaStream_t st) {
  CombineParams p{};
  p.Y = Y; p.weights = weights; p.position = position; p.out = out; p.tokens = static_cast<int>(tokens); p.k = k; p.N = N; p.w_f32 = w_f32;
  count_launch();
  if (dtype == EGS_F32 && out_dtype != EGS_F32)
    return out_dtype == EGS_F16 ? combine_t<float, __half>(p, false, st) : combine_t<float, __nv_bfloat16>(p, false, st);
  return by_type(dtype, [&] { return combine_t<__half>(p, false, st); }, [&] { return combine_t<__nv_bfloat16>(p, false, st); },
                 [&] { return combine_t<float>(p, false, st); });
}

cudaError_t launch_combine_backward(const void* dOut, const void* Y, const void* weights, const int* position, void* dY, void* dweights,
                                    long long tokens, int k, int N, int dtype, int w_f32, cudaStream_t st) {
  CombineParams p{};
  p.Y = Y; p.weights = weights; p.position = position; p.out = dY; p.dOut = dOut; p.dweights = dweights;
  p.tokens = static_cast<int>(tokens); p.k = k; p.N = N; p.w_f32 = w_f32;
  count_launch();
  return by_type(dtype, [&] { return combine_t<__half>(p, true, st); }, [&] { return combine_t<__nv_bfloat16>(p, true, st); },
                 [&] { return combine_t<float>(p, true, st); });
}

cudaError_t launch_quantize_rows(const void* X, int8_t* q, float* scale, long long rows, int C, long long x_stride, long long q_stride, int dtype,
                                 cudaStream_t st) {
  const QuantizeParams p{X, q, scale, x_stride, q_stride, static_cast<int>(rows), C};
  count_launch();
  return by_type(dtype, [&] { return quantize_t<__half>(p, st); }, [&] { return quantize_t<__nv_bfloat16>(p, st); },
                 [&] { return quantize_t<float>(p, st); });
}

cudaError_t launch_pad_rows(const PadRows (&m)[2], cudaStream_t st) {
  PadMatrix p[2]{};
  for (int i = 0; i < 2; ++i)
    if (m[i].dst) p[i] = {static_cast<const unsigned short*>(m[i].src), static_cast<uint4*>(m[i].dst), m[i].rows * (m[i].pitch / 8), m[i].width, m[i].pitch / 8};
  const long long vectors = p[0].vectors + p[1].vectors;
  if (vectors == 0) return cudaSuccess;
  count_launch();
  return launch_kernel(pad_rows_kernel, static_cast<unsigned>((vectors + 255) / 256), 256, 0, st, true, p[0], p[1]);
}

// Row blocks there can be: every expert with rows may have one that is not full.
static long long blocks_bound(const RaggedParams& p, int rows) {
  return p.offsets ? p.rows / rows + (p.rows < p.E ? p.rows : p.E) : (p.rows + rows - 1) / rows;
}

// float32 products in wide tiles: where the mean expert fills most of one, and there are as many as the SMs hold (short contractions, which begin and
// end most of their time: one for every SM).  128 rows for each of 64 experts, 1024 x 512, 512 wide tiles: 205 us, smaller ones 250;  of 16,
// 2048 x 1024, 256 tiles: 301 and 254;  1024 rows of 32, 128 x 64, 256 tiles: 20 and 27;  384 of 8, 256 x 128, 48 tiles: 25 and 18.
static bool wide_rows(const RaggedParams& p) {
  return p.rows >= 96ll * p.E && p.rows / kWide * ((p.N + kGTile - 1) / kGTile) >= (p.C <= 256 ? 148 : 3 * 148);
}
// ... of a weight gradient: where the features of X fill most of its rows
static bool wide_dweight(const RaggedParams& p) { return p.C > 64; }

cudaError_t launch_ragged_rows(const RaggedParams& p, int dtype, int out_dtype, cudaStream_t st) {
  if (dtype == EGS_F32 && wide_rows(p)) {
    const dim3 grid = rows_by_columns(blocks_bound(p, kWide), (p.N + kGTile - 1) / kGTile);
    count_launch();
    return launch_kernel(ragged_rows_f32_kernel, grid, kWideThreads, 0, st, true, p);
  }
  if (dtype == EGS_F32) {
    const dim3 grid = rows_by_columns(blocks_bound(p, kMidRows), (p.N + kMidCols - 1) / kMidCols);
    count_launch();
    auto go = [&](auto kernel, int threads) { return launch_kernel(kernel, grid, threads, kMidSmem, st, true, p); };
    const long long mean = p.rows / kMidRows + p.E / 2, blocks = mean > p.E ? mean : p.rows < p.E ? p.rows : p.E;
    if (blocks * grid.y * grid.z < 3 * 148) return p.nc ? go(ragged_rows_mid_kernel<true, 4>, 256) : go(ragged_rows_mid_kernel<false, 4>, 256);
    return p.nc ? go(ragged_rows_mid_kernel<true, 2>, 128) : go(ragged_rows_mid_kernel<false, 2>, 128);
  }
  long long blocks = blocks_bound(p, kGTile);
  if (blocks < 1) blocks = 1;
  const dim3 grid = rows_by_columns(blocks, (p.N + kGTile - 1) / kGTile);
  count_launch();
  auto go = [&](auto kernel) { return launch_kernel(kernel, grid, 256, 0, st, true, p); };
  if (dtype == EGS_I8)
    return by_type(out_dtype, [&] { return go(ragged_rows_kernel<int8_t, __half>); }, [&] { return go(ragged_rows_kernel<int8_t, __nv_bfloat16>); },
                   [&] { return go(ragged_rows_kernel<int8_t, float>); });
  if (out_dtype == EGS_F32) return dtype == EGS_F16 ? go(ragged_rows_kernel<__half, float>) : go(ragged_rows_kernel<__nv_bfloat16, float>);
  return dtype == EGS_F16 ? go(ragged_rows_kernel<__half, __half>) : go(ragged_rows_kernel<__nv_bfloat16, __nv_bfloat16>);
}

// Rows of a range, so that there are as many CTAs for an SM as it holds (three with wide tiles, four); 0: whole experts.
struct DweightCut {
  bool wide;
  long long tiles, ranges;
  int length;
};
static DweightCut dweight_cut(const RaggedParams& p, int dtype) {
  DweightCut c{};
  c.wide = dtype == EGS_F32 && wide_dweight(p);
  const int tile = c.wide ? kWide : kGTile;
  c.tiles = static_cast<long long>((p.C + tile - 1) / tile) * ((p.N + kGTile - 1) / kGTile);
  const long long length = p.rows * c.tiles / (c.wide ? 3 * 148 : 4 * 148);
  c.length = static_cast<int>(length < 4 * kGStep ? 4 * kGStep : (length + kGStep - 1) / kGStep * kGStep);
  if (c.length >= p.rows || c.tiles * p.E >= 4 * 148) c.length = 0;
  c.ranges = c.length ? p.rows / c.length + p.E : p.E;
  return c;
}
size_t generic_dweight_workspace(const RaggedParams& p, int dtype) {
  const DweightCut c = dweight_cut(p, dtype);
  return c.length ? static_cast<size_t>(c.ranges) * p.C * p.N * sizeof(float) : 0;
}

cudaError_t launch_ragged_dweight(const RaggedParams& p, int dtype, void* workspace, cudaStream_t st) {
  const DweightCut c = dweight_cut(p, dtype);
  float* partial = static_cast<float*>(workspace);
  const dim3 grid(static_cast<unsigned>(c.tiles), 1, static_cast<unsigned>(c.ranges));
  const long long size = static_cast<long long>(p.C) * p.N;
  auto go = [&](auto kernel, auto join, auto* out) {
    count_launch();
    cudaError_t err = launch_kernel(kernel, grid, c.wide ? kWideThreads : 256, 0, st, true, p, c.length, partial);
    if (err != cudaSuccess || c.length == 0) return err;
    count_launch();
    return launch_kernel(join, dim3(static_cast<unsigned>((size + 255) / 256), p.E), 256, 0, st, true, p.offsets, partial, out, size, c.length);
  };
  return by_type(dtype, [&] { return go(ragged_dweight_kernel<__half>, dweight_join_kernel<__half>, static_cast<__half*>(p.Out)); },
                 [&] { return go(ragged_dweight_kernel<__nv_bfloat16>, dweight_join_kernel<__nv_bfloat16>, static_cast<__nv_bfloat16*>(p.Out)); },
                 [&] { return go(c.wide ? ragged_dweight_f32_kernel : ragged_dweight_kernel<float>, dweight_join_kernel<float>, static_cast<float*>(p.Out)); });
}

}  // namespace egs
