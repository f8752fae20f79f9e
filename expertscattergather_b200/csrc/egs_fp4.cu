// Rows in 4 bits and back, and products of few such rows on the CUDA cores.
#include "egs_fp4.cuh"

namespace egs {

namespace {

constexpr unsigned kAll = 0xffffffffu;

// ------------------------------------------------------------------------------------------------
// Rows into 4 bits.  A lane has eight neighbours, four lanes a block, 2^lanes_log2 lanes a row's stretch (short rows share a warp), up to four such
// stretches at a time, whose loads go out together.  Bound by memory, nearly: 16384 x 2048 bf16, 85 MB, 15.3 us (5.6 TB/s), with one stretch at a time 20.
// ------------------------------------------------------------------------------------------------
constexpr int kToWarps = 8, kToAhead = 4;

struct ToFp4 {
  const void* X;
  uint8_t* q;
  uint8_t* scale;
  long long x_stride, q_stride, s_stride, rows;
  int C, chunks, lanes_log2;      // chunks: of eight elements, whole blocks
};

// The largest magnitude of eight 16-bit elements in pairs, as float32's bits (a NaN where there is one).
template <typename T>
__device__ __forceinline__ uint32_t most_of(const uint32_t (&w)[4]) {
  using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const P* x = reinterpret_cast<const P*>(w);
  const P most = __hmax2_nan(__hmax2_nan(__habs2(x[0]), __habs2(x[1])), __hmax2_nan(__habs2(x[2]), __habs2(x[3])));
  return __float_as_uint(to_f32<T>(__hmax_nan(most.x, most.y)));
}
// V: elements that are loaded together; AHEAD: stretches whose loads go out together; WIDE: of 32 lanes, which makes their distances known (74
// instructions for eight elements, 101 with addresses and bounds of each: 33.5 million elements 17.0 us and 17.6, 1 million 2.9 and 4.4).
template <typename T, int V, bool SILU, int AHEAD, bool WIDE>
__global__ void __launch_bounds__(kToWarps * 32) to_fp4_kernel(const __grid_constant__ ToFp4 p) {
  using P = Packed<T, V>;
  union Eight {
    P packs[8 / V];
    T each[8];
    uint32_t words[2 * sizeof(T)];
    __device__ Eight() {}
  };
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lanes_log2 = WIDE ? 5 : p.lanes_log2, lanes = 1 << lanes_log2;
  const long long row = (static_cast<long long>(blockIdx.x) * kToWarps + warp) * (32 >> lanes_log2) + (lane >> lanes_log2);
  const int first = blockIdx.y * lanes * AHEAD + (lane & (lanes - 1));
  const bool on = row < p.rows;
  const T* x = static_cast<const T*>(p.X) + row * p.x_stride + first * 8ll;
  uint32_t* q = reinterpret_cast<uint32_t*>(p.q + row * p.q_stride) + first;
  uint8_t* scale = p.scale + row * p.s_stride;
  auto pass = [&](auto whole) {                // whole: all of it is there
    constexpr bool kWhole = decltype(whole)::value;
    Eight y[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int c = (first + u * lanes) * 8;
      if (kWhole || (on && c + 8 <= p.C)) {
#pragma unroll
        for (int i = 0; i < 8 / V; ++i) y[u].packs[i] = reinterpret_cast<const P*>(x + u * lanes * 8)[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[u].each[i] = on && c + i < p.C ? x[u * lanes * 8 + i] : from_f32<T>(0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int chunk = first + u * lanes;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = to_f32<T>(y[u].each[i]);
        if constexpr (SILU) v[i] = silu_exact(v[i]);
      }
      uint32_t top = 0u;
      if constexpr (!SILU && sizeof(T) == 2) {
        top = most_of<T>(y[u].words);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(kAll, top, 1));
      top = max(top, __shfl_xor_sync(kAll, top, 2));
      if (!kWhole && (!on || chunk >= p.chunks)) continue;
      const uint32_t byte = fp4_scale(top);
      const float inverse = fp4_inverse(byte);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= inverse;
      const uint32_t w = fp4_pack8(v);
      q[u * lanes] = inverse == 0.f ? 0u : w;
      if (!(lane & 3)) scale[chunk >> 2] = static_cast<uint8_t>(byte);
    }
  };
  if (WIDE && __all_sync(kAll, on && (first + (AHEAD - 1) * lanes + 1) * 8 <= p.C)) pass(std::true_type{});
  else pass(std::false_type{});
}

template <typename T, int V>
cudaError_t to_fp4_v(const ToFp4& p, int act, cudaStream_t st) {
  const long long per_cta = kToWarps * (32 >> p.lanes_log2), ctas = (p.rows + per_cta - 1) / per_cta;
  auto go = [&](auto kernel, int ahead) {
    const int stretch = ahead << p.lanes_log2;
    return launch_kernel(kernel, dim3(static_cast<unsigned>(ctas), (p.chunks + stretch - 1) / stretch), kToWarps * 32, 0, st, true, p);
  };
  // Few rows: a stretch a CTA, so that all SMs have some (1003 x 1030 with SiLU, and back: 8.8 us, with four of them 13.7; now 5.8).
  const bool spread = ctas * ((p.chunks >> p.lanes_log2) + 3) / 4 < 148 * 4;
  auto by_width = [&](auto silu) {
    constexpr bool kSilu = decltype(silu)::value;
    if (spread) return p.lanes_log2 == 5 ? go(to_fp4_kernel<T, V, kSilu, 1, true>, 1) : go(to_fp4_kernel<T, V, kSilu, 1, false>, 1);
    return p.lanes_log2 == 5 ? go(to_fp4_kernel<T, V, kSilu, kToAhead, true>, kToAhead) : go(to_fp4_kernel<T, V, kSilu, kToAhead, false>, kToAhead);
  };
  return act == EGS_ACT_SILU ? by_width(std::true_type{}) : by_width(std::false_type{});
}
template <typename T>
cudaError_t to_fp4_t(const ToFp4& p, int act, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](int v) { return p.x_stride % v == 0 && reinterpret_cast<uintptr_t>(p.X) % (v * sizeof(T)) == 0; };
  if (fits(V)) return to_fp4_v<T, V>(p, act, st);
  if (fits(2)) return to_fp4_v<T, 2>(p, act, st);
  return to_fp4_v<T, 1>(p, act, st);
}

// ------------------------------------------------------------------------------------------------
// What 4 bits stand for.  A lane has V neighbours, as many as rows of the output begin on, so that a warp's stores are of whole lines; lanes and stretches as above.
// 16384 x 2048 to bf16: 13.2 us (6.5 TB/s); through integers, with a 64-bit division for each eight, 27.5.
// ------------------------------------------------------------------------------------------------
struct FromFp4 {
  const uint8_t* q;
  const uint8_t* scale;
  void* X;
  long long q_stride, s_stride, rows;
  int C, chunks, lanes_log2;      // chunks: of V elements
};
// V / 2 pairs to where V elements begin on (16 bytes at most).
template <typename T, int V>
__device__ __forceinline__ void store_pairs(T* to, const float2 (&f)[V / 2]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V == 2) *reinterpret_cast<float2*>(to) = f[0];
    else
#pragma unroll
      for (int i = 0; i < V / 2; i += 2) reinterpret_cast<float4*>(to)[i / 2] = make_float4(f[i].x, f[i].y, f[i + 1].x, f[i + 1].y);
  } else {
    uint32_t o[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(f[i].x, f[i].y);
        o[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[i].x, f[i].y);
        o[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (V == 2) *reinterpret_cast<uint32_t*>(to) = o[0];
    else *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}
__host__ __device__ constexpr int from_ahead(int V) { return V == 8 ? 4 : 8; }

template <typename T, int V, bool WIDE>
__global__ void __launch_bounds__(kToWarps * 32) from_fp4_kernel(const __grid_constant__ FromFp4 p) {
  using Q = typename std::conditional<V == 8, uint32_t, uint8_t>::type;
  constexpr int kAhead = from_ahead(V);
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lanes_log2 = WIDE ? 5 : p.lanes_log2, lanes = 1 << lanes_log2;
  const long long row = (static_cast<long long>(blockIdx.x) * kToWarps + warp) * (32 >> lanes_log2) + (lane >> lanes_log2);
  if (row >= p.rows) return;
  const uint8_t *q = p.q + row * p.q_stride, *scale = p.scale + row * p.s_stride;
  T* x = static_cast<T*>(p.X) + row * p.C;
  for (int first = blockIdx.y * lanes * kAhead + (lane & (lanes - 1)); first < p.chunks; first += gridDim.y * lanes * kAhead) {
    const Q* q1 = reinterpret_cast<const Q*>(q + first * V / 2);         // (V = 1: of an even element and of the one behind it the same)
    const uint8_t* scale1 = scale + first * V / kFp4Block;
    T* x1 = x + first * V;
    auto pass = [&](auto whole) {
      constexpr bool kWhole = decltype(whole)::value;      // all of it is there, and lanes * V are whole blocks
      uint32_t w[kAhead], s[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int c = (first + u * lanes) * V;
        w[u] = kWhole ? q1[u * 32 * V / 2 / sizeof(Q)] : c < p.C ? *reinterpret_cast<const Q*>(q + c / 2) : 0u;
        s[u] = kWhole ? scale1[u * 32 * V / kFp4Block] : c < p.C ? scale[c / kFp4Block] : 0u;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int c = (first + u * lanes) * V;
        if (!kWhole && c >= p.C) break;
        T* to = kWhole ? x1 + u * 32 * V : x + c;
        const float power = fp4_power(s[u]);
        if constexpr (V == 8) {
          uint32_t h[4];
          fp4_halves(w[u], h);
          float2 f[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[i] = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
            f[i].x *= power;
            f[i].y *= power;
          }
          store_pairs<T, 8>(to, f);
        } else {
          const float even = fp4_value(w[u]) * power, odd = fp4_value(w[u] >> 4) * power;
          if constexpr (V == 1) {
            *to = from_f32<T>(c & 1 ? odd : even);
          } else {
            const float2 f[1] = {make_float2(even, odd)};
            store_pairs<T, 2>(to, f);
          }
        }
      }
    };
    if (WIDE && (first + (kAhead - 1) * lanes + 1) * V <= p.C) pass(std::true_type{});
    else pass(std::false_type{});
  }
}
template <typename T>
cudaError_t from_fp4_t(FromFp4 p, cudaStream_t st) {
  auto go = [&](auto kernel, int v) {
    p.chunks = (p.C + v - 1) / v;
    p.lanes_log2 = 0;
    while (p.lanes_log2 < 5 && (1 << p.lanes_log2) < p.chunks) ++p.lanes_log2;
    const long long per_cta = kToWarps * (32 >> p.lanes_log2);
    const int stretch = from_ahead(v) << p.lanes_log2, stretches = (p.chunks + stretch - 1) / stretch;
    return launch_kernel(kernel, dim3(static_cast<unsigned>((p.rows + per_cta - 1) / per_cta), stretches < 65535 ? stretches : 65535), kToWarps * 32, 0, st, true, p);
  };
  auto by_width = [&](auto vector) {
    constexpr int V = decltype(vector)::value;
    return p.C > 16 * V ? go(from_fp4_kernel<T, V, true>, V) : go(from_fp4_kernel<T, V, false>, V);      // (more than 16 of them: 32 lanes)
  };
  if (p.C % 8 == 0 && (reinterpret_cast<uintptr_t>(p.X) & 15u) == 0) return by_width(std::integral_constant<int, 8>{});
  if (p.C % 2 == 0 && reinterpret_cast<uintptr_t>(p.X) % (2 * sizeof(T)) == 0) return by_width(std::integral_constant<int, 2>{});
  return by_width(std::integral_constant<int, 1>{});
}

// ------------------------------------------------------------------------------------------------
// Products of few rows: a warp has four channels, its lanes have the blocks of the contraction in turn, up to four rows share a read of the weights.
// Twice the values are integers, so a block's 32 products are eight dp4a and their sum is exact; it is scaled and added in float32.  Bound by the
// latency of one pass where experts have one row (8 of 64 experts, 2048 x 512: 4.8 us for 4.5 MB), beyond by instructions.  (16 channels x 8 rows on mma.sync, a
// quarter of the contraction a warp: 14.3 us for 12.7 at 24 slots, four bytes of a channel at a time; tiles of 128 rows 9.5.)
// ------------------------------------------------------------------------------------------------
constexpr int kFewWarps = 8, kFewRows = 4, kFewChannels = 4;

template <typename OutT, int M>
__device__ __forceinline__ void few_fp4(const Fp4Params& p, int expert, int first, int end, int n0) {
  const int lane = threadIdx.x & 31;
  const uint8_t *w[kFewChannels], *ws[kFewChannels], *x[M], *xs[M];
#pragma unroll
  for (int j = 0; j < kFewChannels; ++j) {
    const int n = min(n0 + j, p.N - 1);
    w[j] = p.W + expert * p.w_expert + n * p.w_row;
    ws[j] = p.Ws + expert * p.ws_expert + n * p.ws_row;
  }
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const int r = first + m < end ? first + m : first, src = p.slots ? p.by_k.quotient(p.slots[r]) : r;
    x[m] = p.A + src * p.a_row;
    xs[m] = p.As + src * p.as_row;
  }
  float acc[M][kFewChannels];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int j = 0; j < kFewChannels; ++j) acc[m][j] = 0.f;
  const int blocks = fp4_blocks(p.C);
#pragma unroll 2
  for (int c = lane; c < blocks; c += 32) {
    Block4 wv[kFewChannels], xv[M];
    uint32_t sw[kFewChannels], sx[M];
#pragma unroll
    for (int j = 0; j < kFewChannels; ++j) {
      wv[j] = load_block(w[j], c, p.C);
      sw[j] = ws[j][c];
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      xv[m] = load_block(x[m], c, p.C);
      sx[m] = xs[m][c];
    }
    int sum[M][kFewChannels];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < kFewChannels; ++j) sum[m][j] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t xl[M], xh[M];
#pragma unroll
      for (int m = 0; m < M; ++m) fp4_integers(xv[m].w[i], xl[m], xh[m]);
#pragma unroll
      for (int j = 0; j < kFewChannels; ++j) {
        uint32_t wl, wh;
        fp4_integers(wv[j].w[i], wl, wh);
#pragma unroll
        for (int m = 0; m < M; ++m) sum[m][j] = __dp4a(static_cast<int>(xh[m]), static_cast<int>(wh), __dp4a(static_cast<int>(xl[m]), static_cast<int>(wl), sum[m][j]));
      }
    }
    float low[M], high[M];
#pragma unroll
    for (int m = 0; m < M; ++m) fp4_factors(fp4_power(sx[m]), low[m], high[m]);
#pragma unroll
    for (int j = 0; j < kFewChannels; ++j) {
      const float f = fp4_power(sw[j]);
#pragma unroll
      for (int m = 0; m < M; ++m) acc[m][j] = fmaf(static_cast<float>(sum[m][j]) * (0.25f * low[m]) * f, high[m], acc[m][j]);
    }
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
      if (lane == m * kFewChannels + j && first + m < end && n0 + j < p.N) out[(first + m) * p.y_row + n0 + j] = from_f32<OutT>(acc[m][j]);
}

template <typename OutT>
__global__ void __launch_bounds__(kFewWarps * 32) few_fp4_kernel(const __grid_constant__ Fp4Params p) {
  __shared__ int segment[3];
  pdl_wait();
  pdl_trigger();
  if (p.offsets) {
    if (const int routed = p.offsets[p.E]; routed < p.rows) {
      OutT* out = static_cast<OutT*>(p.Out);
      zero_by_grid(out + routed * p.y_row, out + p.rows * p.y_row);
    }
  }
  if (threadIdx.x < 32) {                            // the expert with rows that is this CTA's
    int e = 0, first = 0, end = p.rows;
    if (p.offsets) e = nth_expert(p.offsets, p.E, blockIdx.z, &first, &end);
    if (threadIdx.x == 0) segment[0] = e, segment[1] = first, segment[2] = end;
  }
  __syncthreads();
  const int e = segment[0], end = segment[2];
  const long long tile = static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x;
  const long long n0 = (tile * kFewWarps + (threadIdx.x >> 5)) * kFewChannels;
  if (e < 0 || n0 >= p.N) return;
  int r = segment[1];
  for (; end - r > 1; r += kFewRows) {
    few_fp4<OutT, kFewRows>(p, e, r, end, static_cast<int>(n0));
    if (end - r <= kFewRows) return;
  }
  if (r < end) few_fp4<OutT, 1>(p, e, r, end, static_cast<int>(n0));
}

}  // namespace

cudaError_t launch_quantize_fp4(const void* X, uint8_t* q, uint8_t* scale, long long rows, int C, long long x_stride, long long q_stride,
                                long long s_stride, int act, int dtype, cudaStream_t st) {
  ToFp4 p{X, q, scale, x_stride, q_stride, s_stride, rows, C, fp4_blocks(C) * 4, 2};
  while (p.lanes_log2 < 5 && (1 << p.lanes_log2) < p.chunks) ++p.lanes_log2;
  count_launch();
  return dtype == EGS_F16 ? to_fp4_t<__half>(p, act, st) : dtype == EGS_BF16 ? to_fp4_t<__nv_bfloat16>(p, act, st) : to_fp4_t<float>(p, act, st);
}

cudaError_t launch_dequantize_fp4(const uint8_t* q, const uint8_t* scale, void* X, long long rows, int C, long long q_stride, long long s_stride,
                                  int dtype, cudaStream_t st) {
  const FromFp4 p{q, scale, X, q_stride, s_stride, rows, C, 0, 0};
  count_launch();
  return dtype == EGS_F16 ? from_fp4_t<__half>(p, st) : dtype == EGS_BF16 ? from_fp4_t<__nv_bfloat16>(p, st) : from_fp4_t<float>(p, st);
}

// Where experts have one row each, or nearly all: a token's choices differ.  (us, this kernel and tiles of 128 rows: 1 token, 8 of 64 experts, 2048 x 512, 4.8 and 8.4;
// 1 row, 4096 x 4096, 6.4 and 10.6; 2 tokens, 4 of 64, 1024 x 1024, 5.8 and 8.4; two rows an expert cost as much as four: 3 tokens, 8 of 64, 2048 x 512, 12.7 and 9.5;
// 16 tokens, 2 of 64, 512 x 512, 11.1 and 6.5; 8 rows, 2048 x 512, 11.3 and 7.4.)
bool few_fp4_fit(const Fp4Params& p) { return p.rows <= p.by_k.d || 8ll * p.rows <= p.E; }

cudaError_t launch_few_fp4(const Fp4Params& p, int out_dtype, cudaStream_t st) {
  const int segments = p.offsets ? (p.rows < p.E ? p.rows : p.E) : 1, per_cta = kFewWarps * kFewChannels, tiles = (p.N + per_cta - 1) / per_cta;
  const dim3 grid(tiles, 1, segments);
  count_launch();
  auto go = [&](auto kernel) { return launch_kernel(kernel, grid, kFewWarps * 32, 0, st, true, p); };
  return out_dtype == EGS_F16 ? go(few_fp4_kernel<__half>) : out_dtype == EGS_BF16 ? go(few_fp4_kernel<__nv_bfloat16>) : go(few_fp4_kernel<float>);
}

}  // namespace egs
