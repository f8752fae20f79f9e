// Operators on rows in 4 bits and the whole layer for a few tokens (included by egs_host.cpp behind egs_host_choice.h, whose helpers it uses).

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
// [shape.., width] of rows `pitch` bytes apart, behind the last one too.  (Sizes and strides are set: a view by the dispatcher took 1.7 us.)
Tensor empty_padded(std::vector<int64_t>& shape, int64_t width, int64_t pitch, int idx) {
  shape.back() = pitch;
  Tensor t = empty(shape, at::kByte, idx);
  if (pitch == width) return t;
  if (torch::jit::tracer::isTracing()) return t.narrow(-1, 0, width);
  const std::vector<int64_t> strides = t.strides().vec();
  shape.back() = width;
  t.unsafeGetTensorImpl()->set_sizes_and_strides(shape, strides);
  return t;
}
Rows4 empty_rows4(std::vector<int64_t> shape, int64_t C, int idx) {
  const int64_t blocks = (C + 31) / 32;
  Rows4 r;
  r.pitch = 16 * blocks;
  r.scale_pitch = up16(blocks);
  shape.push_back(0);
  r.q = empty_padded(shape, (C + 1) / 2, r.pitch, idx);
  r.scale = empty_padded(shape, blocks, r.scale_pitch, idx);
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
  Given4 g{rows8_of(q), rows8_of(scale), 2 * q.size(-1), rows_ahead(q)};
  // the products read a row's scales 16 bytes at a time, to the end of the last of them
  const Tensor& s = g.scale.t;
  if (s.data_ptr() == scale.data_ptr() && g.rows > 0 &&
      static_cast<size_t>(s.storage_offset() + (g.rows - 1) * g.scale.pitch + up16(s.size(-1))) > s.storage().nbytes()) {
    auto shape = scale.sizes().vec();
    shape.back() = g.scale.pitch = up16(scale.size(-1));
    g.scale.t = at::empty(shape, scale.options());
    g.scale.t.narrow(-1, 0, scale.size(-1)).copy_(scale);
  }
  return g;
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

// An expert's weights in 4 bits for the layer below, [E, N, C / 2] with the bytes of a channel or those of all channels together; others are copied.
struct Matrices4 {
  Tensor q;
  Rows8 scale;
  int64_t stride, far;
  int layout;
  const uint8_t* bytes() const { return static_cast<const uint8_t*>(ptr(q)); }
};
Matrices4 matrices4(const Tensor& q, const Tensor& scale) {
  if (q.scalar_type() == at::kByte && q.size(2) > 1 && q.size(1) > 1 && q.stride(1) == 1 && q.stride(2) >= q.size(1) &&
      q.stride(0) >= q.stride(2) * (q.size(2) - 1) + q.size(1)) {
    if (scale.dim() != 3 || scale.scalar_type() != at::kByte || scale.size(0) != q.size(0) || scale.size(1) != q.size(1) || scale.size(2) != (q.size(2) + 15) / 16)
      value_error("weights in 4 bits are [E, N, C / 2] with scales [E, N, ceil(C / 32)], got " + shape_of(q) + " and " + shape_of(scale));
    return {q, rows8_of(scale), q.stride(2), q.stride(0), EGS_W_CN};
  }
  const Given4 g = given_rows4(q, scale, "weights");
  return {g.q.t, g.scale, g.q.pitch, g.q.pitch * q.size(1), EGS_W_NC};
}

// The whole layer for a few tokens; up_scale and down_scale given: weights in 4 bits.
std::tuple<Tensor, Tensor, Tensor> routed_experts_few(const Tensor& x, const Tensor& router, const Tensor& up, const Tensor& down, int64_t k, const OptTensor& bias,
                                                      const OptTensor& up_scale, const OptTensor& down_scale, const std::string& score, int64_t groups,
                                                      int64_t top_groups, int64_t group_top, bool renormalize, double scale) {
  const bool fp4 = up_scale && up_scale->defined();
  if (fp4 != (down_scale && down_scale->defined())) value_error("up_scale and down_scale belong together");
  if (x.dim() < 1 || router.dim() != 2 || up.dim() != 3 || down.dim() != 3) value_error("expected x[..., I], router[E, I], up and down [E, ., .]");
  const int dt = type_id(x.scalar_type()), sc = score_id(score);
  if (router.scalar_type() != x.scalar_type() || (!fp4 && (up.scalar_type() != x.scalar_type() || down.scalar_type() != x.scalar_type())))
    value_error("x, router and weights must have the same dtype");
  Call c(x, router, up, down);
  const int64_t I = x.size(-1), E = router.size(0), J = fp4 ? up.size(1) : up.size(2), tokens = rows_ahead(x);
  const auto wrong = [&] {
    value_error("shape mismatch: x" + shape_of(x) + " router" + shape_of(router) + " up" + shape_of(up) + " down" + shape_of(down) +
                (fp4 ? " ([E, J, I / 2] and [E, I, J / 2] in 4 bits)" : " ([E, I, J] and [E, J, I])"));
  };
  if (router.size(1) != I || up.size(0) != E || down.size(0) != E) wrong();
  if (fp4 ? up.size(2) != (I + 1) / 2 || down.size(1) != I || down.size(2) != (J + 1) / 2 : up.size(1) != I || down.size(1) != J || down.size(2) != I) wrong();
  if (E < 1 || groups < 1 || E % groups || top_groups < 1 || top_groups > groups || (group_top != 1 && group_top != 2) || k < 1 || k > E / groups * top_groups)
    value_error("routed_experts_few: E = " + std::to_string(E) + " experts in " + std::to_string(groups) + " groups, " + std::to_string(top_groups) +
                " of them kept, do not give " + std::to_string(k) + " experts (group_top is 1 or 2)");
  if (E > EGS_MAX_EXPERTS || k > EGS_MAX_CHOICES || groups > EGS_MAX_GROUPS || tokens > EGS_MAX_FEW_TOKENS || tokens * k > EGS_MAX_FEW_SLOTS)
    value_error("routed_experts_few: at most " + std::to_string(int(EGS_MAX_FEW_TOKENS)) + " tokens, " + std::to_string(int(EGS_MAX_FEW_SLOTS)) + " of tokens * top_k, " +
                std::to_string(int(EGS_MAX_EXPERTS)) + " experts, " + std::to_string(int(EGS_MAX_CHOICES)) + " choices and " + std::to_string(int(EGS_MAX_GROUPS)) + " groups");
  Tensor b;
  if (bias && bias->defined()) {
    if (bias->numel() != E || !bias->is_floating_point()) value_error("bias must be a floating tensor of E elements");
    if (!bias->is_cuda() || bias->get_device() != c.idx) throw std::runtime_error("bias must be on x's CUDA device");
    b = bias->reshape({E}).to(at::kFloat).contiguous();
  }
  const Rows r = rows_of(x);
  const Tensor w = router.contiguous();
  auto shape = x.sizes().vec();
  Tensor out = empty(shape, x.scalar_type(), c.idx);
  shape.back() = k;
  Tensor weights = empty(shape, at::kFloat, c.idx), experts = empty(shape, at::kInt, c.idx);
  if (I == 0 || J == 0) value_error("routed_experts_few: no features");
  const egs_route spec{tokens, int(E), int(k), int(groups), int(top_groups), int(group_top), sc, renormalize ? 1 : 0, float(scale)};
  const size_t bytes = api.egs_routed_experts_few_workspace_bytes(&spec, I, J);
  const Tensor ws = scratch(bytes, c.idx);
  if (fp4) {
    for (const Tensor* t : {&*up_scale, &*down_scale})
      if (!t->is_cuda() || t->get_device() != c.idx) throw std::runtime_error("all tensors must be on the same CUDA device");
    const Matrices4 u = matrices4(up, *up_scale), d = matrices4(down, *down_scale);
    check(api.egs_routed_experts_few_fp4(ptr(r.t), ptr(w), static_cast<const float*>(ptr(b)), u.bytes(), bytes_of(u.scale), u.stride, u.far, u.scale.pitch, u.layout, d.bytes(),
                                         bytes_of(d.scale), d.stride, d.far, d.scale.pitch, d.layout, ptr(out), weights.data_ptr<float>(), experts.data_ptr<int>(), &spec, I, J,
                                         r.stride, dt, ptr(ws), bytes, c.stream),
          "egs_routed_experts_few_fp4");
  } else {
    const Tensor u = up.contiguous(), d = down.contiguous();
    check(api.egs_routed_experts_few(ptr(r.t), ptr(w), static_cast<const float*>(ptr(b)), ptr(u), ptr(d), ptr(out), weights.data_ptr<float>(), experts.data_ptr<int>(), &spec, I, J,
                                     r.stride, dt, ptr(ws), bytes, c.stream),
          "egs_routed_experts_few");
  }
  c.debug();
  return {out, weights, experts};
}
