// Operators on rows in 4 bits (included by egs_host.cpp behind egs_host_choice.h, whose helpers it uses).

int activation_id(const std::optional<std::string>& s) {
  if (!s) return EGS_ACT_NONE;
  if (*s == "silu") return EGS_ACT_SILU;
  value_error("activation must be None or 'silu'");
}
int64_t rows_ahead(const Tensor& t) {          // rows of a [..., n], n may be 0
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  return n;
}
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// Rows for 4-bit results: [.., ceil(C / 2)] bytes and [.., ceil(C / 32)] scales, both a multiple of 16 bytes apart
struct Rows4 {
  Tensor q, scale;
  int64_t pitch, scale_pitch;
};
Rows4 empty_rows4(std::vector<int64_t> shape, int64_t C, int idx) {
  const int64_t blocks = (C + 31) / 32, bytes = (C + 1) / 2;
  Rows4 r;
  r.pitch = 16 * blocks;
  r.scale_pitch = up16(blocks);
  shape.push_back(r.pitch);
  r.q = empty(shape, at::kByte, idx);
  shape.back() = r.scale_pitch;
  r.scale = empty(shape, at::kByte, idx);
  if (r.pitch != bytes) r.q = r.q.narrow(-1, 0, bytes);
  if (r.scale_pitch != blocks) r.scale = r.scale.narrow(-1, 0, blocks);
  return r;
}
// Bytes and scales that belong together, rows 16 bytes apart: what does not lie so is copied
struct Given4 {
  Rows8 q, scale;
  int64_t C, rows;
};
Given4 given_rows4(const Tensor& q, const Tensor& scale, const char* name) {
  if (q.dim() < 1 || scale.dim() != q.dim() || q.sizes().slice(0, q.dim() - 1) != scale.sizes().slice(0, q.dim() - 1) ||
      scale.size(-1) != (q.size(-1) + 15) / 16)
    value_error(std::string(name) + " in 4 bits are [..., C / 2] with scales [..., ceil(C / 32)], got " + shape_of(q) + " and " + shape_of(scale));
  if (q.scalar_type() != at::kByte || scale.scalar_type() != at::kByte) value_error(std::string(name) + " in 4 bits and their scales must be uint8");
  return {rows8_of(q), rows8_of(scale), 2 * q.size(-1), rows_ahead(q)};
}
const uint8_t* bytes_of(const Rows8& r) { return static_cast<const uint8_t*>(ptr(r.t)); }

std::tuple<Tensor, Tensor> quantize_rows_fp4(const Tensor& X, const std::optional<std::string>& activation) {
  if (X.dim() < 1) value_error("expected X[..., C]");
  const int dt = type_id(X.scalar_type()), act = activation_id(activation);
  Call c(X);
  const Rows r = rows_of(X);
  auto shape = X.sizes().vec();
  shape.pop_back();
  const Rows4 out = empty_rows4(shape, X.size(-1), c.idx);
  check(api.egs_quantize_rows_fp4(ptr(r.t), static_cast<uint8_t*>(ptr(out.q)), static_cast<uint8_t*>(ptr(out.scale)), rows_ahead(X), X.size(-1), r.stride,
                                  out.pitch, out.scale_pitch, act, dt, c.stream),
        "egs_quantize_rows_fp4");
  c.debug();
  return {out.q, out.scale};
}

Tensor dequantize_rows_fp4(const Tensor& q, const Tensor& scale, std::optional<int64_t> C, at::ScalarType dtype) {
  const int dt = type_id(dtype);
  Call c(q, scale);
  const Given4 a = given_rows4(q, scale, "rows");
  const int64_t width = C.value_or(a.C);
  if (width != a.C && width != a.C - 1) value_error("rows of " + std::to_string(q.size(-1)) + " bytes do not hold " + std::to_string(width) + " values");
  auto shape = q.sizes().vec();
  shape.back() = width;
  Tensor X = empty(shape, dtype, c.idx);
  check(api.egs_dequantize_rows_fp4(bytes_of(a.q), bytes_of(a.scale), ptr(X), a.rows, width, a.q.pitch, a.scale.pitch, dt, c.stream), "egs_dequantize_rows_fp4");
  c.debug();
  return X;
}

// The operands of a product in 4 bits; offsets undefined: one expert that has all rows.
struct Product4 {
  Given4 a, b;
  egs_ragged d;
  const int *offsets, *slots;
};
Product4 product4(const Call& c, const Tensor& q, const Tensor& q_scale, const Tensor& Wq, const Tensor& w_scale, const OptTensor& offsets,
                  const OptTensor& slots, int64_t tokens, int64_t k, int rid) {
  const bool dense = !offsets || !offsets->defined();
  if (Wq.dim() != (dense ? 2 : 3)) value_error(dense ? "expected q[..., C / 2], Wq[N, C / 2]" : "expected q[..., C / 2], Wq[E, N, C / 2]");
  Product4 p{given_rows4(q, q_scale, "rows"), given_rows4(Wq, w_scale, "weights"), {}, nullptr, nullptr};
  const int64_t E = dense ? 1 : Wq.size(0), N = Wq.size(-2);
  if (dense) {
    tokens = p.a.rows, k = 1;
  } else {
    check_plan(c, *offsets, *slots, E, tokens * k);
    p.offsets = offsets->data_ptr<int>();
    p.slots = slots->data_ptr<int>();
  }
  const int64_t want = rid == EGS_ROWS_TOKENS ? tokens : tokens * k;
  if (p.a.C != p.b.C || p.a.rows != want)
    value_error("shape mismatch: q" + shape_of(q) + " Wq" + shape_of(Wq) + " for " + std::to_string(want) + " rows");
  p.d = {tokens, k, E, p.a.C, N};
  return p;
}

Tensor matmul_fp4(const Tensor& q, const Tensor& q_scale, const Tensor& Wq, const Tensor& w_scale, const OptTensor& offsets, const OptTensor& slots,
                  int64_t tokens, int64_t k, const std::string& rows, at::ScalarType out_dtype, int path) {
  const int dt = type_id(out_dtype), rid = rows_id(rows);
  Call c(q, Wq, q_scale, w_scale);
  const Product4 p = product4(c, q, q_scale, Wq, w_scale, offsets, slots, tokens, k, rid);
  auto shape = q.sizes().vec();
  shape.back() = p.d.N;
  if (p.offsets) shape = {tokens * k, p.d.N};
  Tensor Y = empty(shape, out_dtype, c.idx);
  check(api.egs_expert_matmul_fp4(bytes_of(p.a.q), bytes_of(p.a.scale), p.a.q.pitch, p.a.scale.pitch, bytes_of(p.b.q), bytes_of(p.b.scale), p.b.q.pitch,
                                  p.b.scale.pitch, p.offsets, p.slots, ptr(Y), &p.d, rid, dt, path_of(path), c.status(), c.stream),
        "egs_expert_matmul_fp4");
  c.debug();
  return Y;
}

std::tuple<Tensor, Tensor> matmul_fp4_rows(const Tensor& q, const Tensor& q_scale, const Tensor& Wq, const Tensor& w_scale, const OptTensor& offsets,
                                           const OptTensor& slots, int64_t tokens, int64_t k, const std::string& rows,
                                           const std::optional<std::string>& activation, int path) {
  const int rid = rows_id(rows), act = activation_id(activation);
  Call c(q, Wq, q_scale, w_scale);
  const Product4 p = product4(c, q, q_scale, Wq, w_scale, offsets, slots, tokens, k, rid);
  const Rows4 y = empty_rows4({p.d.tokens * p.d.k}, p.d.N, c.idx);
  const size_t bytes = api.egs_expert_matmul_fp4_rows_workspace_bytes(&p.d, path_of(path));
  const Tensor ws = scratch(bytes, c.idx);
  check(api.egs_expert_matmul_fp4_rows(bytes_of(p.a.q), bytes_of(p.a.scale), p.a.q.pitch, p.a.scale.pitch, bytes_of(p.b.q), bytes_of(p.b.scale), p.b.q.pitch,
                                       p.b.scale.pitch, p.offsets, p.slots, static_cast<uint8_t*>(ptr(y.q)), static_cast<uint8_t*>(ptr(y.scale)), y.pitch,
                                       y.scale_pitch, &p.d, rid, act, path_of(path), ptr(ws), bytes, c.status(), c.stream),
        "egs_expert_matmul_fp4_rows");
  c.debug();
  return {y.q, y.scale};
}
