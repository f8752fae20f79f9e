// C entries of the operators in 4 bits and of the whole layer for a few tokens: checks of arguments, choice of kernels.
#include "egs_fp4.cuh"

namespace egs {
namespace {

constexpr long long kMaxRows = EGS_MAX_ROWS, kMaxWidth = 1 << 24;

bool valid_dtype(int d) { return d == EGS_F32 || d == EGS_F16 || d == EGS_BF16; }
bool valid_act(int a) { return a == EGS_ACT_NONE || a == EGS_ACT_SILU; }
bool valid_path(int p) { return p == EGS_PATH_AUTO || p == EGS_PATH_GENERIC || p == EGS_PATH_TENSOR; }
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int done(cudaError_t err, const char* where) { return err == cudaSuccess ? EGS_OK : fail_cuda(err, where); }
cudaStream_t stream_of(void* s) { return static_cast<cudaStream_t>(s); }
// Strides of rows of C elements and of their scales
bool strides_hold(long long q_stride, long long s_stride, long long C, bool whole_blocks) {
  return q_stride >= (whole_blocks ? 16 * ((C + 31) / 32) : (C + 1) / 2) && s_stride >= (C + 31) / 32 && q_stride % 16 == 0 && s_stride % 16 == 0;
}

int check_dims(const egs_ragged* d) {
  if (!d || d->tokens < 0 || d->k < 0 || d->E < 0 || d->C < 0 || d->N < 0 || d->C % 2) return EGS_ERR_INVALID_ARGUMENT;
  if (d->E > EGS_MAX_EXPERTS || d->tokens > kMaxRows || d->k > kMaxRows || d->tokens * d->k > kMaxRows || d->C > kMaxWidth || d->N > kMaxWidth)
    return EGS_ERR_TOO_LARGE;
  if (d->E == 0 && d->tokens * d->k > 0) return EGS_ERR_INVALID_ARGUMENT;
  return EGS_OK;
}
// Tiles of the tensor cores have 32-bit numbers.
bool tiles_fit(const egs_ragged& d) { return (static_cast<double>(d.tokens) * d.k / 128 + d.E + 1) * (d.N / 32.0 + 1) < 2e9; }

struct Operands {
  const uint8_t *q, *q_scale;
  int64_t q_stride, qs_stride;
  const uint8_t *Wq, *w_scale;
  int64_t w_stride, ws_stride;
  const int32_t *offsets, *slots;
};
// Everything but the output; `p` is only made where there is something to do.
int product(const Operands& o, const egs_ragged* dims, int rows, int path, int32_t* status_word, bool* nothing, Fp4Params* p) {
  *nothing = false;
  if (!valid_path(path) || (rows != EGS_ROWS_TOKENS && rows != EGS_ROWS_SORTED)) return EGS_ERR_INVALID_ARGUMENT;
  if (int rc = check_dims(dims)) return rc;
  if (!strides_hold(o.q_stride, o.qs_stride, dims->C, false) || !strides_hold(o.w_stride, o.ws_stride, dims->C, false) ||
      (!o.offsets && (dims->E != 1 || dims->k != 1)))
    return EGS_ERR_INVALID_ARGUMENT;
  if (dims->tokens * dims->k == 0 || dims->N == 0) {
    *nothing = true;
    return EGS_OK;
  }
  if ((o.offsets && !o.slots) || (dims->C > 0 && (!o.q || !o.q_scale || !o.Wq || !o.w_scale))) return EGS_ERR_INVALID_ARGUMENT;
  if (!on16(o.q) || !on16(o.q_scale) || !on16(o.Wq) || !on16(o.w_scale)) return EGS_ERR_INVALID_ARGUMENT;
  p->A = o.q; p->As = o.q_scale; p->W = o.Wq; p->Ws = o.w_scale;
  p->offsets = o.offsets;
  p->slots = o.offsets && rows == EGS_ROWS_TOKENS ? o.slots : nullptr;
  p->status = status_ref(status_word);
  p->a_row = o.q_stride; p->as_row = o.qs_stride; p->w_row = o.w_stride; p->ws_row = o.ws_stride;
  p->w_expert = o.w_stride * dims->N; p->ws_expert = o.ws_stride * dims->N;
  p->rows = static_cast<int>(dims->tokens * dims->k);
  p->a_rows = static_cast<int>(rows == EGS_ROWS_TOKENS ? dims->tokens : dims->tokens * dims->k);
  p->E = static_cast<int>(dims->E); p->C = static_cast<int>(dims->C); p->N = static_cast<int>(dims->N);
  p->by_k = Div(dims->k > 0 ? static_cast<int>(dims->k) : 1);
  return EGS_OK;
}
// Whether the kernel for few rows takes this, by the caller's wish or because it is faster; `able`: the tensor cores could.
bool takes_few(const Fp4Params& p, int path, bool able) { return !able || path == EGS_PATH_GENERIC || (path == EGS_PATH_AUTO && few_fp4_fit(p)); }
bool tensor_able(const egs_ragged& d) { return device_is_sm100() && d.C > 0 && tiles_fit(d); }

int check_layer(const egs_route* r, int64_t I, int64_t J) {
  if (!r || r->tokens < 0 || r->E < 1 || r->top_k < 1 || r->groups < 1 || r->E % r->groups || r->top_groups < 1 || r->top_groups > r->groups ||
      (r->group_top != 1 && r->group_top != 2) || r->top_k > r->E / r->groups * r->top_groups || (r->score != EGS_SCORE_SOFTMAX && r->score != EGS_SCORE_SIGMOID) ||
      I < 1 || J < 1)
    return EGS_ERR_INVALID_ARGUMENT;
  if (r->E > EGS_MAX_EXPERTS || r->top_k > EGS_MAX_CHOICES || r->groups > EGS_MAX_GROUPS || r->tokens > EGS_MAX_FEW_TOKENS || r->tokens * r->top_k > EGS_MAX_FEW_SLOTS ||
      I > kMaxWidth || J > kMaxWidth)
    return EGS_ERR_TOO_LARGE;
  return EGS_OK;
}
int layer(const FewLayer& f, const egs_route* r, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_dtype(dtype) || f.x_row < 0) return EGS_ERR_INVALID_ARGUMENT;
  if (int rc = check_layer(r, f.I, f.J)) return rc;
  if (r->tokens == 0) return EGS_OK;
  if (!f.X || !f.router || !f.up || !f.down || !f.out || !f.weights || !f.experts) return EGS_ERR_INVALID_ARGUMENT;
  const uintptr_t element = dtype == EGS_F32 ? 4 : 2, addresses = reinterpret_cast<uintptr_t>(f.X) | reinterpret_cast<uintptr_t>(f.router) | reinterpret_cast<uintptr_t>(f.out);
  if ((addresses | (f.up_scale ? 0u : reinterpret_cast<uintptr_t>(f.up) | reinterpret_cast<uintptr_t>(f.down))) % element) return EGS_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < few_layer_workspace(*r, f.I, f.J) || !on16(workspace)) return EGS_ERR_WORKSPACE;
  return done(launch_few_layer(f, *r, dtype, workspace, stream_of(stream)), "routed_experts_few launch");
}

}  // namespace
}  // namespace egs

using namespace egs;

extern "C" {

int egs_quantize_rows_fp4(const void* X, uint8_t* q, uint8_t* scale, int64_t rows, int64_t C, int64_t x_stride, int64_t q_stride, int64_t s_stride,
                          int activation, int dtype, void* cuda_stream) {
  if (!valid_dtype(dtype) || !valid_act(activation) || rows < 0 || C < 0 || x_stride < 0) return EGS_ERR_INVALID_ARGUMENT;
  if (rows > kMaxRows || C > kMaxWidth) return EGS_ERR_TOO_LARGE;
  if (!strides_hold(q_stride, s_stride, C, true)) return EGS_ERR_INVALID_ARGUMENT;
  if (rows == 0 || C == 0) return EGS_OK;
  if (!X || !q || !scale || !on16(q)) return EGS_ERR_INVALID_ARGUMENT;
  return done(launch_quantize_fp4(X, q, scale, rows, static_cast<int>(C), x_stride, q_stride, s_stride, activation, dtype, stream_of(cuda_stream)),
              "quantize_rows_fp4 launch");
}

int egs_dequantize_rows_fp4(const uint8_t* q, const uint8_t* scale, void* X, int64_t rows, int64_t C, int64_t q_stride, int64_t s_stride, int dtype,
                            void* cuda_stream) {
  if (!valid_dtype(dtype) || rows < 0 || C < 0) return EGS_ERR_INVALID_ARGUMENT;
  if (rows > kMaxRows || C > kMaxWidth) return EGS_ERR_TOO_LARGE;
  if (!strides_hold(q_stride, s_stride, C, false)) return EGS_ERR_INVALID_ARGUMENT;
  if (rows == 0 || C == 0) return EGS_OK;
  if (!X || !q || !scale || !on16(q)) return EGS_ERR_INVALID_ARGUMENT;
  return done(launch_dequantize_fp4(q, scale, X, rows, static_cast<int>(C), q_stride, s_stride, dtype, stream_of(cuda_stream)), "dequantize_rows_fp4 launch");
}

int egs_expert_matmul_fp4(const uint8_t* q, const uint8_t* q_scale, int64_t q_stride, int64_t qs_stride, const uint8_t* Wq, const uint8_t* w_scale,
                          int64_t w_stride, int64_t ws_stride, const int32_t* offsets, const int32_t* slots, void* Y, const egs_ragged* dims, int rows,
                          int out_dtype, int path, int32_t* status_word, void* cuda_stream) {
  if (!valid_dtype(out_dtype)) return EGS_ERR_INVALID_ARGUMENT;
  bool nothing;
  Fp4Params p{};
  if (int rc = product({q, q_scale, q_stride, qs_stride, Wq, w_scale, w_stride, ws_stride, offsets, slots}, dims, rows, path, status_word, &nothing, &p); rc || nothing) return rc;
  if (!Y) return EGS_ERR_INVALID_ARGUMENT;
  p.Out = Y;
  p.y_row = p.N;
  const bool able = tensor_able(*dims);
  if (path == EGS_PATH_TENSOR && !able) return EGS_ERR_UNSUPPORTED;
  const cudaStream_t st = stream_of(cuda_stream);
  return done(takes_few(p, path, able) ? launch_few_fp4(p, out_dtype, st) : launch_fp4_rows_tensor(p, out_dtype, st), "expert_matmul_fp4 launch");
}

size_t egs_expert_matmul_fp4_rows_workspace_bytes(const egs_ragged* dims, int path) {
  if (check_dims(dims) != EGS_OK || !valid_path(path) || dims->tokens * dims->k == 0 || dims->N == 0) return 0;
  Fp4Params p{};
  p.rows = static_cast<int>(dims->tokens * dims->k);
  p.E = static_cast<int>(dims->E);
  p.by_k = Div(static_cast<int>(dims->k));
  return takes_few(p, path, tensor_able(*dims)) ? static_cast<size_t>(p.rows) * dims->N * sizeof(float) : 0;
}

int egs_expert_matmul_fp4_rows(const uint8_t* q, const uint8_t* q_scale, int64_t q_stride, int64_t qs_stride, const uint8_t* Wq, const uint8_t* w_scale,
                               int64_t w_stride, int64_t ws_stride, const int32_t* offsets, const int32_t* slots, uint8_t* y, uint8_t* y_scale,
                               int64_t y_stride, int64_t ys_stride, const egs_ragged* dims, int rows, int activation, int path, void* workspace,
                               size_t workspace_bytes, int32_t* status_word, void* cuda_stream) {
  if (!valid_act(activation)) return EGS_ERR_INVALID_ARGUMENT;
  bool nothing;
  Fp4Params p{};
  if (int rc = product({q, q_scale, q_stride, qs_stride, Wq, w_scale, w_stride, ws_stride, offsets, slots}, dims, rows, path, status_word, &nothing, &p); rc || nothing) return rc;
  if (!strides_hold(y_stride, ys_stride, dims->N, true) || !y || !y_scale || !on16(y) || !on16(y_scale)) return EGS_ERR_INVALID_ARGUMENT;
  const bool able = tensor_able(*dims);
  if (path == EGS_PATH_TENSOR && !able) return EGS_ERR_UNSUPPORTED;
  const cudaStream_t st = stream_of(cuda_stream);
  p.act = activation;
  if (!takes_few(p, path, able)) {
    p.Out = y; p.OutScale = y_scale; p.y_row = y_stride; p.ys_row = ys_stride;
    return done(launch_fp4_rows_tensor(p, EGS_F32, st), "expert_matmul_fp4_rows launch");
  }
  const size_t need = static_cast<size_t>(p.rows) * p.N * sizeof(float);
  if (!workspace || workspace_bytes < need || !on16(workspace)) return EGS_ERR_WORKSPACE;
  p.Out = workspace;
  p.y_row = p.N;
  if (cudaError_t err = launch_few_fp4(p, EGS_F32, st); err != cudaSuccess) return fail_cuda(err, "expert_matmul_fp4_rows launch");
  return done(launch_quantize_fp4(workspace, y, y_scale, p.rows, p.N, p.N, y_stride, ys_stride, activation, EGS_F32, st), "expert_matmul_fp4_rows in 4 bits");
}

size_t egs_routed_experts_few_workspace_bytes(const egs_route* route, int64_t I, int64_t J) {
  return check_layer(route, I, J) == EGS_OK && route->tokens ? few_layer_workspace(*route, static_cast<int>(I), static_cast<int>(J)) : 0;
}

int egs_routed_experts_few(const void* X, const void* router, const float* bias, const void* up, const void* down, void* out, float* weights,
                           int32_t* experts, const egs_route* route, int64_t I, int64_t J, int64_t x_stride, int dtype, void* workspace,
                           size_t workspace_bytes, void* cuda_stream) {
  if (int rc = check_layer(route, I, J)) return rc;
  const FewLayer f{X, router, bias, up, down, nullptr, nullptr, out, weights, experts, x_stride, 0, 0, 0, 0, static_cast<int>(I), static_cast<int>(J), 0, 0, false, false};
  return layer(f, route, dtype, workspace, workspace_bytes, cuda_stream);
}

int egs_routed_experts_few_fp4(const void* X, const void* router, const float* bias, const uint8_t* up, const uint8_t* up_scale, int64_t up_stride,
                               int64_t up_far, int64_t us_stride, int up_layout, const uint8_t* down, const uint8_t* down_scale, int64_t down_stride,
                               int64_t down_far, int64_t ds_stride, int down_layout, void* out,
                               float* weights, int32_t* experts, const egs_route* route, int64_t I, int64_t J, int64_t x_stride, int dtype,
                               void* workspace, size_t workspace_bytes, void* cuda_stream) {
  if (int rc = check_layer(route, I, J)) return rc;
  // an expert's [N, C / 2], or [C / 2, N]
  auto holds = [&](const uint8_t* w, int64_t stride, int64_t far, int64_t s_stride, int layout, int64_t C, int64_t N) {
    if (stride > 0xffffffffll || s_stride > 0xffffffffll) return false;
    if (layout == EGS_W_NC) return strides_hold(stride, s_stride, C, false) && far >= stride * (N - 1) + (C + 1) / 2 && far % 16 == 0 && on16(w);
    return layout == EGS_W_CN && s_stride >= (C + 31) / 32 && stride >= N && far >= stride * ((C + 1) / 2 - 1) + N;
  };
  if (!holds(up, up_stride, up_far, us_stride, up_layout, I, J) || !holds(down, down_stride, down_far, ds_stride, down_layout, J, I)) return EGS_ERR_INVALID_ARGUMENT;
  if (route->tokens && (!up_scale || !down_scale)) return EGS_ERR_INVALID_ARGUMENT;
  const FewLayer f{X, router, bias, up, down, up_scale, down_scale, out, weights, experts, x_stride, up_stride, us_stride, down_stride, ds_stride, static_cast<int>(I), static_cast<int>(J),
                   up_far, down_far, up_layout == EGS_W_CN, down_layout == EGS_W_CN};
  return layer(f, route, dtype, workspace, workspace_bytes, cuda_stream);
}

}  // extern "C"
