// C entries of the operators for tokens that choose experts: checks of arguments, choice of kernels.
#include "egs_internal.cuh"

namespace egs {
namespace {

// Rows are counted in 32 bits, and what lies up to a few tiles behind the last one has to be countable too.
constexpr long long kInt32Max = 2147483647LL, kMaxRows = EGS_MAX_ROWS, kMaxWidth = 1 << 24;

bool valid_dtype(int d) { return d == EGS_F32 || d == EGS_F16 || d == EGS_BF16; }
bool valid_path(int p) { return p == EGS_PATH_AUTO || p == EGS_PATH_GENERIC || p == EGS_PATH_TENSOR; }
bool valid_layout(int l) { return l == EGS_W_CN || l == EGS_W_NC; }
bool valid_rows(int r) { return r == EGS_ROWS_TOKENS || r == EGS_ROWS_SORTED; }
int done(cudaError_t err, const char* where) { return err == cudaSuccess ? EGS_OK : fail_cuda(err, where); }
cudaStream_t stream_of(void* s) { return static_cast<cudaStream_t>(s); }

int check_route(const egs_route* r, int64_t row_stride, int dtype, bool choice) {
  if (!r || !valid_dtype(dtype) || r->tokens < 0 || r->E < 1 || r->top_k < 1 || row_stride < 0 ||
      (r->score != EGS_SCORE_SOFTMAX && r->score != EGS_SCORE_SIGMOID))
    return EGS_ERR_INVALID_ARGUMENT;
  if (choice && (r->groups < 1 || r->E % r->groups || r->top_groups < 1 || r->top_groups > r->groups || (r->group_top != 1 && r->group_top != 2) ||
                 r->top_k > r->E / r->groups * r->top_groups))
    return EGS_ERR_INVALID_ARGUMENT;
  if (r->E > EGS_MAX_EXPERTS || r->top_k > EGS_MAX_CHOICES || (choice && r->groups > EGS_MAX_GROUPS) || r->tokens > kMaxRows) return EGS_ERR_TOO_LARGE;
  return EGS_OK;
}

int check_ragged(const egs_ragged* d) {
  if (!d || d->tokens < 0 || d->k < 0 || d->E < 0 || d->C < 0 || d->N < 0) return EGS_ERR_INVALID_ARGUMENT;
  if (d->E > EGS_MAX_EXPERTS || d->tokens > kMaxRows || d->k > kMaxRows || d->tokens * d->k > kMaxRows || d->C > kMaxWidth || d->N > kMaxWidth)
    return EGS_ERR_TOO_LARGE;
  if (d->E == 0 && d->tokens * d->k > 0) return EGS_ERR_INVALID_ARGUMENT;
  return EGS_OK;
}

RaggedParams ragged(const egs_ragged& d, int rows) {
  RaggedParams p{};
  p.rows = static_cast<int>(d.tokens * d.k);
  p.a_rows = static_cast<int>(rows == EGS_ROWS_TOKENS ? d.tokens : d.tokens * d.k);
  p.E = static_cast<int>(d.E);
  p.C = static_cast<int>(d.C);
  p.N = static_cast<int>(d.N);
  p.by_k = Div(d.k > 0 ? static_cast<int>(d.k) : 1);
  return p;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Tiles have 32-bit numbers.
bool tiles_fit(const RaggedParams& p) {
  const double blocks = p.rows / 128.0 + p.E + 1, wide = p.N / 64.0 + 1, deep = p.C / 128.0 + 1;
  return blocks * wide < 2e9 && (p.E + 1024) * deep * wide < 2e9 && p.rows < kInt32Max - (1 << 22);
}

// The tensor cores read 16-bit rows that begin on 16 bytes.  Others are copied: bytes of such a copy, 0 where none is needed.
long long pitch8(long long width) { return (width + 7) / 8 * 8; }
size_t copy_bytes(long long rows, long long width) {
  return width % 8 ? (static_cast<size_t>(rows) * pitch8(width) * 2 + 255) & ~static_cast<size_t>(255) : 0;
}
// ... of `rows` rows of `width` elements at *src, which becomes the copy and *pitch its pitch; moves `workspace` on
PadRows padded(const void** src, long long* pitch, long long rows, long long width, char** workspace) {
  if (width % 8 == 0) return {};
  const PadRows m{*src, *workspace, rows, static_cast<int>(width), static_cast<int>(pitch8(width))};
  *workspace += copy_bytes(rows, width);
  *pitch = m.pitch;
  *src = m.dst;
  return m;
}
long long a_rows_of(const egs_ragged& d, int rows) { return rows == EGS_ROWS_TOKENS ? d.tokens : d.tokens * d.k; }

}  // namespace
}  // namespace egs

using namespace egs;

extern "C" {

int egs_route_tokens(const void* logits, const float* bias, float* weights, int32_t* experts, const egs_route* route, int64_t row_stride,
                     int dtype, void* cuda_stream) {
  if (int rc = check_route(route, row_stride, dtype, true)) return rc;
  if (route->tokens == 0) return EGS_OK;
  if (!logits || !weights || !experts) return EGS_ERR_INVALID_ARGUMENT;
  return done(launch_route_tokens(logits, bias, weights, experts, *route, row_stride, dtype, stream_of(cuda_stream)), "route_tokens launch");
}

int egs_route_tokens_backward(const float* dweights, const void* logits, const int32_t* experts, void* dlogits, const egs_route* route,
                              int64_t row_stride, int dtype, void* cuda_stream) {
  if (int rc = check_route(route, row_stride, dtype, false)) return rc;
  if (route->tokens == 0) return EGS_OK;
  if (!dweights || !logits || !experts || !dlogits) return EGS_ERR_INVALID_ARGUMENT;
  return done(launch_route_backward(dweights, logits, experts, dlogits, *route, row_stride, dtype, stream_of(cuda_stream)), "route_tokens_backward launch");
}

size_t egs_plan_workspace_bytes(int64_t n, int E) {
  return n <= 0 || n > kMaxRows || E < 0 || E > EGS_MAX_EXPERTS ? 0 : plan_workspace_ints(n, E) * sizeof(int);
}

int egs_plan_experts(const int32_t* experts, int64_t n, int E, int32_t* offsets, int32_t* slots, int32_t* position, void* workspace,
                     size_t workspace_bytes, int32_t* status_word, void* cuda_stream) {
  if (n < 0 || E < 1 || !offsets || (n > 0 && (!experts || !slots || !position))) return EGS_ERR_INVALID_ARGUMENT;
  if (n > kMaxRows || E > EGS_MAX_EXPERTS) return EGS_ERR_TOO_LARGE;
  const size_t need = egs_plan_workspace_bytes(n, E);
  if (need && (!workspace || workspace_bytes < need)) return EGS_ERR_WORKSPACE;
  return done(launch_plan_experts(experts, n, E, offsets, slots, position, static_cast<int*>(workspace), status_ref(status_word), stream_of(cuda_stream)),
              "plan_experts launch");
}

size_t egs_expert_matmul_workspace_bytes(const egs_ragged* dims, int rows, int w_layout, int dtype) {
  if (dtype == EGS_F32 || check_ragged(dims) != EGS_OK || !valid_rows(rows) || !valid_layout(w_layout)) return 0;
  return copy_bytes(a_rows_of(*dims, rows), dims->C) +
         (w_layout == EGS_W_NC ? copy_bytes(dims->E * dims->N, dims->C) : copy_bytes(dims->E * dims->C, dims->N));
}

int egs_expert_matmul_out(const void* X, const void* W, const int32_t* offsets, const int32_t* slots, void* Y, const egs_ragged* dims, int rows,
                          int w_layout, int dtype, int out_dtype, int path, void* workspace, size_t workspace_bytes, int32_t* status_word, void* cuda_stream) {
  if (!valid_dtype(dtype) || (out_dtype != dtype && out_dtype != EGS_F32) || !valid_path(path) || !valid_layout(w_layout) || !valid_rows(rows))
    return EGS_ERR_INVALID_ARGUMENT;
  if (int rc = check_ragged(dims)) return rc;
  RaggedParams p = ragged(*dims, rows);
  if (p.rows == 0 || p.N == 0) return EGS_OK;
  if (!offsets || !slots || !Y || (p.C > 0 && (!X || !W))) return EGS_ERR_INVALID_ARGUMENT;
  p.A = X; p.W = W; p.Out = Y; p.offsets = offsets; p.slots = rows == EGS_ROWS_TOKENS ? slots : nullptr;
  p.status = status_ref(status_word);
  p.nc = w_layout == EGS_W_NC;
  p.a_row = p.C; p.w_row = p.nc ? p.C : p.N; p.w_expert = static_cast<long long>(p.C) * p.N;
  const cudaStream_t st = stream_of(cuda_stream);
  const bool able = device_is_sm100() && dtype != EGS_F32 && p.C > 0 && aligned16(X) && aligned16(W) && tiles_fit(p);
  if (path == EGS_PATH_TENSOR && !able) return EGS_ERR_UNSUPPORTED;
  if (path == EGS_PATH_AUTO && p.C > 0 && few_rows_fit(p, dtype)) return done(launch_few_rows(p, dtype, out_dtype, st), "expert_matmul launch");
  if (!able || path == EGS_PATH_GENERIC) return done(launch_ragged_rows(p, dtype, out_dtype, st), "expert_matmul launch");
  const size_t need = egs_expert_matmul_workspace_bytes(dims, rows, w_layout, dtype);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return EGS_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  const PadRows rows_copy = padded(&p.A, &p.a_row, p.a_rows, p.C, &ws);
  const PadRows copies[2] = {rows_copy, padded(&p.W, &p.w_row, dims->E * (p.nc ? p.N : p.C), p.w_row, &ws)};
  if (cudaError_t err = launch_pad_rows(copies, st); err != cudaSuccess) return fail_cuda(err, "expert_matmul copies");
  p.w_expert = p.w_row * (p.nc ? p.N : p.C);
  return done(launch_ragged_rows_tensor(p, dtype, out_dtype, st), "expert_matmul launch");
}

int egs_expert_matmul(const void* X, const void* W, const int32_t* offsets, const int32_t* slots, void* Y, const egs_ragged* dims, int rows,
                      int w_layout, int dtype, int path, void* workspace, size_t workspace_bytes, int32_t* status_word, void* cuda_stream) {
  return egs_expert_matmul_out(X, W, offsets, slots, Y, dims, rows, w_layout, dtype, dtype, path, workspace, workspace_bytes, status_word, cuda_stream);
}

size_t egs_expert_dweight_workspace_bytes(const egs_ragged* dims, int rows, int dtype) {
  if (!valid_dtype(dtype) || check_ragged(dims) != EGS_OK || !valid_rows(rows)) return 0;
  if (dims->tokens * dims->k == 0 || dims->E * dims->C * dims->N == 0) return 0;
  const RaggedParams p = ragged(*dims, rows);
  const size_t generic = generic_dweight_workspace(p, dtype);
  if (dtype == EGS_F32) return generic;
  const size_t tensor = copy_bytes(a_rows_of(*dims, rows), dims->C) + copy_bytes(p.rows, dims->N) + ragged_dweight_workspace(p);
  return tensor > generic ? tensor : generic;
}

int egs_expert_dweight(const void* X, const void* dY, const int32_t* offsets, const int32_t* slots, void* dW, const egs_ragged* dims, int rows,
                       int dtype, int path, void* workspace, size_t workspace_bytes, int32_t* status_word, void* cuda_stream) {
  if (!valid_dtype(dtype) || !valid_path(path) || !valid_rows(rows)) return EGS_ERR_INVALID_ARGUMENT;
  if (int rc = check_ragged(dims)) return rc;
  RaggedParams p = ragged(*dims, rows);
  const size_t elements = static_cast<size_t>(dims->E) * dims->C * dims->N;
  if (elements == 0) return EGS_OK;
  if (!dW) return EGS_ERR_INVALID_ARGUMENT;
  if (p.rows == 0) return done(launch_fill_zero(dW, elements * (dtype == EGS_F32 ? 4 : 2), stream_of(cuda_stream)), "expert_dweight fill");
  if (!X || !dY || !offsets || !slots) return EGS_ERR_INVALID_ARGUMENT;
  p.A = X; p.W = dY; p.Out = dW; p.offsets = offsets; p.slots = rows == EGS_ROWS_TOKENS ? slots : nullptr;
  p.status = status_ref(status_word);
  p.a_row = p.C; p.w_row = p.N;
  const cudaStream_t st = stream_of(cuda_stream);
  const bool able = device_is_sm100() && dtype != EGS_F32 && aligned16(X) && aligned16(dY) && tiles_fit(p);
  if (path == EGS_PATH_TENSOR && !able) return EGS_ERR_UNSUPPORTED;
  const size_t need = egs_expert_dweight_workspace_bytes(dims, rows, dtype);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return EGS_ERR_WORKSPACE;
  if (!able || path == EGS_PATH_GENERIC) return done(launch_ragged_dweight(p, dtype, workspace, st), "expert_dweight launch");
  char* ws = static_cast<char*>(workspace);
  const PadRows rows_copy = padded(&p.A, &p.a_row, p.a_rows, p.C, &ws);
  const PadRows copies[2] = {rows_copy, padded(&p.W, &p.w_row, p.rows, p.N, &ws)};
  if (cudaError_t err = launch_pad_rows(copies, st); err != cudaSuccess) return fail_cuda(err, "expert_dweight copies");
  return done(launch_ragged_dweight_tensor(p, dtype, ws, st), "expert_dweight launch");
}

int egs_combine_out(const void* Y, const void* weights, const int32_t* position, void* out, int64_t tokens, int64_t k, int64_t N, int dtype,
                    int weights_dtype, int out_dtype, void* cuda_stream) {
  const egs_ragged d{tokens, k, EGS_MAX_EXPERTS, 0, N};
  if (int rc = check_ragged(&d)) return rc;
  if (!valid_dtype(dtype) || !valid_dtype(out_dtype) || (out_dtype != dtype && dtype != EGS_F32) || (weights && weights_dtype != EGS_F32 && weights_dtype != out_dtype))
    return EGS_ERR_INVALID_ARGUMENT;
  if (tokens == 0 || N == 0) return EGS_OK;
  if (tokens * (N / 32 + 1) > kInt32Max) return EGS_ERR_TOO_LARGE;
  if (!out || (k > 0 && (!Y || !position))) return EGS_ERR_INVALID_ARGUMENT;
  // (the kernels go from choice to choice: a token without any is not for them)
  if (k == 0) return done(launch_fill_zero(out, static_cast<size_t>(tokens) * N * (out_dtype == EGS_F32 ? 4 : 2), stream_of(cuda_stream)), "combine fill");
  return done(launch_combine(Y, weights, position, out, tokens, static_cast<int>(k), static_cast<int>(N), dtype, weights_dtype == EGS_F32, out_dtype,
                             stream_of(cuda_stream)),
              "combine launch");
}

int egs_combine(const void* Y, const void* weights, const int32_t* position, void* out, int64_t tokens, int64_t k, int64_t N, int dtype,
                int weights_dtype, void* cuda_stream) {
  return egs_combine_out(Y, weights, position, out, tokens, k, N, dtype, weights_dtype, dtype, cuda_stream);
}

int egs_combine_backward(const void* dOut, const void* Y, const void* weights, const int32_t* position, void* dY, void* dweights,
                         int64_t tokens, int64_t k, int64_t N, int dtype, int weights_dtype, void* cuda_stream) {
  const egs_ragged d{tokens, k, EGS_MAX_EXPERTS, 0, N};
  if (int rc = check_ragged(&d)) return rc;
  if (!valid_dtype(dtype) || ((weights || dweights) && weights_dtype != EGS_F32 && weights_dtype != dtype)) return EGS_ERR_INVALID_ARGUMENT;
  if (tokens * k == 0) return EGS_OK;
  if (!position || (N > 0 && (!dOut || !dY || (dweights && !Y)))) return EGS_ERR_INVALID_ARGUMENT;
  return done(launch_combine_backward(dOut, Y, weights, position, dY, dweights, tokens, static_cast<int>(k), static_cast<int>(N), dtype,
                                      weights_dtype == EGS_F32, stream_of(cuda_stream)),
              "combine_backward launch");
}

int egs_quantize_rows(const void* X, int8_t* q, float* scale, int64_t rows, int64_t C, int64_t x_stride, int64_t q_stride, int dtype,
                      void* cuda_stream) {
  if (!valid_dtype(dtype) || rows < 0 || C < 0 || x_stride < 0 || q_stride < C) return EGS_ERR_INVALID_ARGUMENT;
  if (rows > kMaxRows || C > kMaxWidth) return EGS_ERR_TOO_LARGE;
  if (rows == 0) return EGS_OK;
  if (!scale || (C > 0 && (!X || !q))) return EGS_ERR_INVALID_ARGUMENT;
  return done(launch_quantize_rows(X, q, scale, rows, static_cast<int>(C), x_stride, q_stride, dtype, stream_of(cuda_stream)), "quantize_rows launch");
}

int egs_expert_matmul_int8(const int8_t* q, const float* q_scale, int64_t q_stride, const int8_t* Wq, const float* w_scale, int64_t w_stride,
                           const int32_t* offsets, const int32_t* slots, void* Y, const egs_ragged* dims, int rows, int out_dtype, int path,
                           int32_t* status_word, void* cuda_stream) {
  if (!valid_dtype(out_dtype) || !valid_path(path) || !valid_rows(rows)) return EGS_ERR_INVALID_ARGUMENT;
  if (int rc = check_ragged(dims)) return rc;
  if (dims->C >= 131072) return EGS_ERR_TOO_LARGE;             // 2^17 products of magnitude 2^14 no longer fit in an int32 sum
  if (q_stride < dims->C || w_stride < dims->C || (!offsets && (dims->E != 1 || dims->k != 1))) return EGS_ERR_INVALID_ARGUMENT;
  RaggedParams p = ragged(*dims, rows);
  if (p.rows == 0 || p.N == 0) return EGS_OK;
  if (!Y || !q_scale || !w_scale || (offsets && !slots) || (p.C > 0 && (!q || !Wq))) return EGS_ERR_INVALID_ARGUMENT;
  p.A = q; p.W = Wq; p.Out = Y; p.offsets = offsets; p.slots = offsets && rows == EGS_ROWS_TOKENS ? slots : nullptr;
  p.a_scale = q_scale; p.w_scale = w_scale;
  p.status = status_ref(status_word);
  p.nc = 1;
  p.a_row = q_stride; p.w_row = w_stride; p.w_expert = w_stride * p.N;
  const bool able = device_is_sm100() && p.C > 0 && p.a_row % 16 == 0 && p.w_row % 16 == 0 && aligned16(q) && aligned16(Wq) && tiles_fit(p);
  if (path == EGS_PATH_TENSOR && !able) return EGS_ERR_UNSUPPORTED;
  if (path == EGS_PATH_AUTO && p.C > 0 && few_rows_fit(p, EGS_I8))
    return done(launch_few_rows(p, EGS_I8, out_dtype, stream_of(cuda_stream)), "expert_matmul_int8 launch");
  if (!able || path == EGS_PATH_GENERIC) return done(launch_ragged_rows(p, EGS_I8, out_dtype, stream_of(cuda_stream)), "expert_matmul_int8 launch");
  return done(launch_ragged_rows_tensor(p, EGS_I8, out_dtype, stream_of(cuda_stream)), "expert_matmul_int8 launch");
}

}  // extern "C"
