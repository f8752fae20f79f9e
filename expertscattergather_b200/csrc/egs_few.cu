// Products over ragged rows where experts have few of them: a decoding step, whose work is reading the weights of the experts that were
// chosen.  No tiles: every weight is read once for every four rows of its expert, 16 bytes a thread, and the grid is made large enough
// that all SMs read.
//
// Weights [E, N, C] (8-bit integers always): a warp has four channels, its lanes go along C and their sums are joined by shuffles.
// Weights [E, C, N]: LANES lanes have that many vectors of columns, and the groups of LANES lanes of a CTA have the rows of C in turn; their
// sums are joined by shuffles and then, in the warps' order, through shared memory.  LANES is as large as leaves a CTA for every SM (rows
// of the weights are then read in longer pieces).  One token of eight experts, 2048 x 512 bf16: clusters of eight CTAs with parts of C
// and 32 lanes to a row took 45 us.
#include "egs_internal.cuh"

namespace egs {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kFewWarps = 8, kFewThreads = kFewWarps * 32;
constexpr int kFewRows = 4;            // rows that share a read of the weights
constexpr int kFewChannels = 4;        // [E, N, C]: channels of a warp
constexpr int kFewCnThreads = 512;     // [E, C, N]
__host__ __device__ constexpr int few_part(int lanes) { return lanes == 16 ? 512 : 1024; }     // ... contraction elements of the rows in shared memory at a time
constexpr int kFewAhead = 8;           // ... vectors a thread asks for at a time

template <typename T> struct Sum { using type = float; };
template <> struct Sum<int8_t> { using type = int; };

struct Segment {
  int expert, first, end;
};
// Of this CTA (blockIdx.y); shared by its first warp.
__device__ __forceinline__ Segment segment_of(const RaggedParams& p, Segment* shared) {
  if (threadIdx.x < 32) {
    Segment s{0, 0, p.rows};
    if (p.offsets) s.expert = nth_expert(p.offsets, p.E, blockIdx.y, &s.first, &s.end);
    if (threadIdx.x == 0) *shared = s;
  }
  __syncthreads();
  return *shared;
}
template <typename OutT>
__device__ __forceinline__ void few_zero(const RaggedParams& p) {
  if (!p.offsets) return;
  OutT* out = static_cast<OutT*>(p.Out);
  if (const int routed = p.offsets[p.E]; routed < p.rows) zero_by_grid(out + static_cast<long long>(routed) * p.N, out + static_cast<long long>(p.rows) * p.N);
}

template <typename T, int V>
__device__ __forceinline__ void dot(float& acc, const Packed<T, V>& a, const Packed<T, V>& b) {
#pragma unroll
  for (int v = 0; v < V; ++v) acc = fmaf(a.get(v), b.get(v), acc);
}
__device__ __forceinline__ void dot(int& acc, const Packed<int8_t, 16>& a, const Packed<int8_t, 16>& b) {
#pragma unroll
  for (int v = 0; v < 4; ++v) acc = __dp4a(reinterpret_cast<const int*>(&a)[v], reinterpret_cast<const int*>(&b)[v], acc);
}
__device__ __forceinline__ void dot(int& acc, const Packed<int8_t, 1>& a, const Packed<int8_t, 1>& b) { acc += a.raw[0] * b.raw[0]; }
template <typename T> __device__ __forceinline__ float product(T a, T b) { return to_f32<T>(a) * to_f32<T>(b); }
__device__ __forceinline__ int product(int8_t a, int8_t b) { return a * b; }

// Rows first .. first + M - 1 (at least one, those from `end` on stand for the first) times four channels.
template <typename T, typename OutT, int V, int M>
__device__ __forceinline__ void few_nc(const RaggedParams& p, const Segment& s, int first, int n0) {
  using A = typename Sum<T>::type;
  using P = Packed<T, V>;
  const int lane = threadIdx.x & 31;
  const T* w[kFewChannels];
  const T* x[M];
  int src[M];
#pragma unroll
  for (int j = 0; j < kFewChannels; ++j) w[j] = static_cast<const T*>(p.W) + s.expert * p.w_expert + min(n0 + j, p.N - 1) * p.w_row;
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const int r = first + m < s.end ? first + m : first;
    src[m] = p.slots ? p.by_k.quotient(p.slots[r]) : r;
    x[m] = static_cast<const T*>(p.A) + src[m] * p.a_row;
  }
  A acc[M][kFewChannels];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int j = 0; j < kFewChannels; ++j) acc[m][j] = 0;
  const int full = p.C / V;
#pragma unroll 2
  for (int c = lane; c < full; c += 32) {
    P wv[kFewChannels], xv[M];
#pragma unroll
    for (int j = 0; j < kFewChannels; ++j) wv[j] = reinterpret_cast<const P*>(w[j])[c];
#pragma unroll
    for (int m = 0; m < M; ++m) xv[m] = reinterpret_cast<const P*>(x[m])[c];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < kFewChannels; ++j) dot(acc[m][j], xv[m], wv[j]);
  }
  for (int c = full * V + lane; c < p.C; c += 32) {        // what is less than a vector
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < kFewChannels; ++j) acc[m][j] += product(x[m][c], w[j][c]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < kFewChannels; ++j) acc[m][j] += __shfl_xor_sync(kAll, acc[m][j], o);
  OutT* out = static_cast<OutT*>(p.Out);
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int j = 0; j < kFewChannels; ++j)
      if (lane == m * kFewChannels + j && first + m < s.end && n0 + j < p.N) {
        float v = static_cast<float>(acc[m][j]);
        if (p.a_scale) v *= p.a_scale[src[m]] * p.w_scale[static_cast<long long>(s.expert) * p.N + n0 + j];
        out[static_cast<long long>(first + m) * p.N + n0 + j] = from_f32<OutT>(v);
      }
}

template <typename T, typename OutT, int V>
__global__ void __launch_bounds__(kFewThreads) few_rows_nc_kernel(const __grid_constant__ RaggedParams p) {
  __shared__ Segment shared;
  pdl_wait();
  pdl_trigger();
  few_zero<OutT>(p);
  const Segment s = segment_of(p, &shared);
  if (s.expert < 0) return;
  const int n0 = (blockIdx.x * kFewWarps + (threadIdx.x >> 5)) * kFewChannels;
  if (n0 >= p.N) return;
  int r = s.first;
  for (; r + 1 < s.end; r += kFewRows) few_nc<T, OutT, V, kFewRows>(p, s, r, n0);
  if (r < s.end) few_nc<T, OutT, V, 1>(p, s, r, n0);
}

template <int LANES>
struct CnShared {
  float x[kFewRows][few_part(LANES)];
  Segment segment;
  int src[kFewRows];
};

// Rows first .. first + M - 1 (as in few_nc) times LANES * V columns from n0 on.  sums: [warps][M][LANES * V]
template <typename T, typename OutT, int V, int LANES, int M>
__device__ __forceinline__ void few_cn(const RaggedParams& p, const Segment& s, CnShared<LANES>* sh, float* sums, int first, int n0) {
  using P = Packed<T, V>;
  constexpr int kFewPart = few_part(LANES), kGroups = kFewCnThreads / LANES, kWidth = LANES * V, kWarps = kFewCnThreads / 32;
  const int tid = threadIdx.x, group = tid / LANES, l = tid % LANES, n = n0 + l * V;
  const T* W = static_cast<const T*>(p.W) + s.expert * p.w_expert + n;
  const bool on = n < p.N;
  float acc[M][V];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[m][v] = 0.f;
  for (int c0 = 0; c0 < p.C; c0 += kFewPart) {
    const int part = min(kFewPart, p.C - c0);
    P w[kFewAhead];
    int c = group;
    auto load = [&]() {                        // the weights first, the rows (and the barriers) while they come
#pragma unroll
      for (int i = 0; i < kFewAhead; ++i)
        if (on && c + i * kGroups < part) w[i] = *reinterpret_cast<const P*>(W + (c0 + c + i * kGroups) * p.w_row);
    };
    load();
    __syncthreads();                           // the rows of the part before have been read
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const T* x = static_cast<const T*>(p.A) + sh->src[m] * p.a_row + c0;
      for (int i = tid; i < part; i += kFewCnThreads) sh->x[m][i] = to_f32<T>(x[i]);
    }
    __syncthreads();
    while (c < part) {
#pragma unroll
      for (int i = 0; i < kFewAhead; ++i)
        if (on && c + i * kGroups < part) {
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const float xm = sh->x[m][c + i * kGroups];
#pragma unroll
            for (int v = 0; v < V; ++v) acc[m][v] = fmaf(xm, w[i].get(v), acc[m][v]);
          }
        }
      c += kFewAhead * kGroups;
      if (c < part) load();
    }
  }
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[m][v] += __shfl_xor_sync(kAll, acc[m][v], o);
  if ((tid & 31) < LANES) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int v = 0; v < V; ++v) sums[((tid >> 5) * M + m) * kWidth + l * V + v] = acc[m][v];
  }
  __syncthreads();
  OutT* out = static_cast<OutT*>(p.Out);
  for (int i = tid; i < M * kWidth; i += kFewCnThreads) {
    const int m = i / kWidth, col = n0 + i % kWidth;
    if (first + m >= s.end || col >= p.N) continue;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += sums[w * M * kWidth + i];
    out[static_cast<long long>(first + m) * p.N + col] = from_f32<OutT>(t);
  }
}

template <typename T, typename OutT, int V, int LANES>
__global__ void __launch_bounds__(kFewCnThreads, 1) few_rows_cn_kernel(const __grid_constant__ RaggedParams p) {
  __shared__ CnShared<LANES> sh;
  __shared__ float sums[kFewCnThreads / 32 * kFewRows * LANES * V];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x;
  few_zero<OutT>(p);
  const Segment s = segment_of(p, &sh.segment);
  if (s.expert < 0) return;
  for (int r = s.first; r < s.end; r += kFewRows) {
    __syncthreads();                           // the rows before these have been read, and their sums
    if (tid < kFewRows) {
      const int row = r + tid < s.end ? r + tid : r;
      sh.src[tid] = p.slots ? p.by_k.quotient(p.slots[row]) : row;
    }
    __syncthreads();
    if (r + 1 < s.end) few_cn<T, OutT, V, LANES, kFewRows>(p, s, &sh, sums, r, blockIdx.x * LANES * V);
    else few_cn<T, OutT, V, LANES, 1>(p, s, &sh, sums, r, blockIdx.x * LANES * V);
  }
}

template <typename T, typename OutT, int V>
cudaError_t few_nc_launch(const RaggedParams& p, int segments, cudaStream_t st) {
  const int per_cta = kFewWarps * kFewChannels;
  return launch_kernel(few_rows_nc_kernel<T, OutT, V>, dim3((p.N + per_cta - 1) / per_cta, segments), kFewThreads, 0, st, true, p);
}

template <typename T, typename OutT, int V, int LANES>
cudaError_t few_cn_lanes(const RaggedParams& p, int segments, cudaStream_t st) {
  return launch_kernel(few_rows_cn_kernel<T, OutT, V, LANES>, dim3((p.N + LANES * V - 1) / (LANES * V), segments), kFewCnThreads, 0, st, true, p);
}
template <typename T, typename OutT, int V>
cudaError_t few_cn_launch(const RaggedParams& p, int segments, cudaStream_t st) {
  if constexpr (V == 1) {
    return few_cn_lanes<T, OutT, 1, 32>(p, segments, st);
  } else {
    auto enough = [&](int lanes) { return (p.N + lanes * V - 1) / (lanes * V) * segments >= 148; };
    if (enough(16)) return few_cn_lanes<T, OutT, V, 16>(p, segments, st);
    if (enough(8)) return few_cn_lanes<T, OutT, V, 8>(p, segments, st);
    return few_cn_lanes<T, OutT, V, 4>(p, segments, st);
  }
}

bool on(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T, typename OutT>
cudaError_t few_launch(const RaggedParams& p, int segments, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool rows_on = p.w_row % V == 0 && p.w_expert % V == 0 && on(p.W, 16);
  if (p.nc) return rows_on && p.a_row % V == 0 && on(p.A, 16) ? few_nc_launch<T, OutT, V>(p, segments, st) : few_nc_launch<T, OutT, 1>(p, segments, st);
  if constexpr (sizeof(T) > 1) return rows_on && p.N % V == 0 ? few_cn_launch<T, OutT, V>(p, segments, st) : few_cn_launch<T, OutT, 1>(p, segments, st);
  return cudaErrorInvalidValue;
}

}  // namespace

// Up to how many rows this is faster than tiles, measured with 1 to 81 experts of 352 x 384 to 2048 x 2048 (whole calls, other kernels in brackets):
// 16 bits, 64 experts of 1024 x 256: 32 rows 14 us (18), 128 rows 27 (20); of 2048 x 512: 8 rows 19 (24), 32 rows 29 (27), 64 rows 45 (32)
// 8 bits, 2048 x 512: 32 rows 19 (21), 64 rows 25 (23);  one matrix of 2048 x 2048: 8 rows 16 (17), 16 rows 27 (17)
// float32, 64 experts of 1024 x 512: 128 rows 50 (45), 256 rows 55 (45);  16 of 2048 x 1024: 32 rows 47 (57), 64 rows 50 (57);  8 of 256 x 128:
// 16 rows 10 (12), 64 rows 14 (12)
bool few_rows_fit(const RaggedParams& p, int dtype) {
  if (dtype == EGS_F32) return p.rows <= 3ll * p.E || p.rows <= 8;
  if (dtype == EGS_I8) return 4ll * p.rows <= 3 * p.E || p.rows <= 8;
  return 8ll * p.rows <= 3 * p.E || p.rows <= 4;
}

cudaError_t launch_few_rows(const RaggedParams& p, int dtype, int out_dtype, cudaStream_t st) {
  const int segments = p.offsets ? (p.rows < p.E ? p.rows : p.E) : 1;
  count_launch();
  if (dtype == EGS_I8) {
    if (out_dtype == EGS_F16) return few_launch<int8_t, __half>(p, segments, st);
    if (out_dtype == EGS_BF16) return few_launch<int8_t, __nv_bfloat16>(p, segments, st);
    return few_launch<int8_t, float>(p, segments, st);
  }
  const bool wide = out_dtype == EGS_F32;
  if (dtype == EGS_F16) return wide ? few_launch<__half, float>(p, segments, st) : few_launch<__half, __half>(p, segments, st);
  if (dtype == EGS_BF16) return wide ? few_launch<__nv_bfloat16, float>(p, segments, st) : few_launch<__nv_bfloat16, __nv_bfloat16>(p, segments, st);
  return few_launch<float, float>(p, segments, st);
}

}  // namespace egs
