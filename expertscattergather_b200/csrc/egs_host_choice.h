// Operators for tokens that choose experts (included by egs_host.cpp, whose conventions hold here).

// A matrix [..., n] as rows that lie `stride` elements apart, copied where its layout is another one.
struct Rows {
  Tensor t;
  int64_t count, stride;
};
Rows rows_of(const Tensor& t) {
  const int64_t n = t.size(-1);
  const int64_t count = n ? t.numel() / n : (t.dim() > 1 ? t.numel() : 0);
  if (t.dim() == 2 && (t.stride(1) == 1 || n == 1) && t.stride(0) >= n) return {t, t.size(0), t.stride(0)};
  if (t.dim() == 1 && (n <= 1 || t.stride(0) == 1)) return {t, 1, n};
  return {t.contiguous(), n ? count : t.numel(), n};
}
// 16-byte copies and loads want aligned tensors: one that begins elsewhere in its storage is copied.
Tensor whole(const Tensor& t) {
  const Tensor c = t.contiguous();
  return c.numel() && (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) ? c.clone() : c;
}
int score_id(const std::string& s) {
  if (s == "softmax") return EGS_SCORE_SOFTMAX;
  if (s == "sigmoid") return EGS_SCORE_SIGMOID;
  value_error("score must be 'softmax' or 'sigmoid'");
}
int rows_id(const std::string& s) {
  if (s == "tokens") return EGS_ROWS_TOKENS;
  if (s == "sorted") return EGS_ROWS_SORTED;
  value_error("rows must be 'tokens' or 'sorted'");
}
Tensor int_ids(const Tensor& ids, int64_t E) {
  switch (ids.scalar_type()) {
    case at::kInt: return ids.contiguous();
    case at::kLong: return ids.clamp(-2, E).to(at::kInt).contiguous();       // (ids beyond 32 bits stay outside)
    case at::kShort:
    case at::kChar:
    case at::kByte: return ids.to(at::kInt).contiguous();
    default: value_error(std::string("experts must be an integer tensor, got ") + toString(ids.scalar_type()));
  }
}

std::tuple<Tensor, Tensor> route_tokens(const Tensor& logits, int64_t k, const OptTensor& bias, const std::string& score, int64_t groups,
                                        int64_t top_groups, int64_t group_top, bool renormalize, double scale) {
  if (logits.dim() < 1) value_error("expected logits[..., E]");
  const int dt = type_id(logits.scalar_type());
  const int sc = score_id(score);
  Call c(logits);
  const int64_t E = logits.size(-1);
  if (E < 1 || groups < 1 || E % groups || top_groups < 1 || top_groups > groups || (group_top != 1 && group_top != 2) || k < 1 ||
      k > E / groups * top_groups)
    value_error("route_tokens: E = " + std::to_string(E) + " experts in " + std::to_string(groups) + " groups, " + std::to_string(top_groups) +
                " of them kept, do not give " + std::to_string(k) + " experts (group_top is 1 or 2)");
  if (E > EGS_MAX_EXPERTS || k > EGS_MAX_CHOICES || groups > EGS_MAX_GROUPS)
    value_error("route_tokens: at most " + std::to_string(int(EGS_MAX_EXPERTS)) + " experts, " + std::to_string(int(EGS_MAX_CHOICES)) +
                " choices and " + std::to_string(int(EGS_MAX_GROUPS)) + " groups");
  Tensor b;
  if (bias && bias->defined()) {
    if (bias->numel() != E || !bias->is_floating_point()) value_error("bias must be a floating tensor of E elements");
    if (!bias->is_cuda() || bias->get_device() != c.idx) throw std::runtime_error("bias must be on the logits' CUDA device");
    b = bias->reshape({E}).to(at::kFloat).contiguous();
  }
  const Rows r = rows_of(logits);
  auto shape = logits.sizes().vec();
  shape.back() = k;
  Tensor w = empty(shape, at::kFloat, c.idx), e = empty(shape, at::kInt, c.idx);
  const egs_route spec{r.count, int(E), int(k), int(groups), int(top_groups), int(group_top), sc, renormalize ? 1 : 0, float(scale)};
  check(api.egs_route_tokens(ptr(r.t), static_cast<const float*>(ptr(b)), w.data_ptr<float>(), e.data_ptr<int>(), &spec, r.stride, dt, c.stream),
        "egs_route_tokens");
  c.debug();
  return {w, e};
}

Tensor route_tokens_backward(const Tensor& dweights, const Tensor& logits, const Tensor& experts, const std::string& score, bool renormalize,
                             double scale) {
  if (logits.dim() < 1 || dweights.dim() != logits.dim() || experts.sizes() != dweights.sizes() ||
      logits.sizes().slice(0, logits.dim() - 1) != dweights.sizes().slice(0, logits.dim() - 1))
    value_error("expected dweights[..., k], logits[..., E], experts[..., k]");
  const int dt = type_id(logits.scalar_type());
  const int sc = score_id(score);
  Call c(logits, dweights, experts);
  const int64_t E = logits.size(-1), k = dweights.size(-1);
  if (E < 1 || E > EGS_MAX_EXPERTS || k < 1 || k > EGS_MAX_CHOICES) value_error("route_tokens_backward: unsupported E or k");
  const Tensor g = dweights.to(at::kFloat).contiguous(), ids = int_ids(experts, E);
  const Rows r = rows_of(logits);
  Tensor d = empty(logits.sizes(), logits.scalar_type(), c.idx);
  const egs_route spec{r.count, int(E), int(k), 1, 1, 1, sc, renormalize ? 1 : 0, float(scale)};
  check(api.egs_route_tokens_backward(g.data_ptr<float>(), ptr(r.t), ids.data_ptr<int>(), ptr(d), &spec, r.stride, dt, c.stream),
        "egs_route_tokens_backward");
  c.debug();
  return d;
}

// `n` integers of `all` from `first` on (three allocations instead of one took a microsecond of the plan's six)
Tensor part_of(const Tensor& all, int64_t first, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(first);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

std::tuple<Tensor, Tensor, Tensor> plan_experts(const Tensor& experts, int64_t E) {
  if (experts.dim() < 1) value_error("expected experts[..., k]");
  if (E < 1 || E > EGS_MAX_EXPERTS) value_error("plan_experts: E must be between 1 and " + std::to_string(int(EGS_MAX_EXPERTS)));
  Call c(experts);
  const Tensor ids = int_ids(experts, E);
  const int64_t n = ids.numel();
  const int64_t at_slots = (E + 4) / 4 * 4, at_position = at_slots + (n + 3) / 4 * 4;        // (each begins on 16 bytes)
  const Tensor all = empty({at_position + n}, at::kInt, c.idx);
  const Tensor offsets = part_of(all, 0, E + 1), slots = part_of(all, at_slots, n), position = part_of(all, at_position, n);
  const size_t bytes = api.egs_plan_workspace_bytes(n, int(E));
  const Tensor ws = scratch(bytes, c.idx);
  check(api.egs_plan_experts(ids.data_ptr<int>(), n, int(E), offsets.data_ptr<int>(), slots.data_ptr<int>(), position.data_ptr<int>(), ptr(ws),
                             bytes, c.status(), c.stream),
        "egs_plan_experts");
  c.debug();
  return {offsets, slots, position};
}

// The plan's arrays belong together, [E + 1], [tokens * k], [tokens * k], and lie where the tensors do.
void check_plan(const Call& c, const Tensor& offsets, const Tensor& slots, int64_t E, int64_t n) {
  for (const Tensor* t : {&offsets, &slots})
    if (!t->is_cuda() || t->get_device() != c.idx) throw std::runtime_error("the plan must be on the tensors' CUDA device");
  if (offsets.scalar_type() != at::kInt || slots.scalar_type() != at::kInt || offsets.numel() != E + 1 || slots.numel() != n ||
      !offsets.is_contiguous() || !slots.is_contiguous())
    value_error("the plan was made for " + std::to_string(offsets.numel() - 1) + " experts and " + std::to_string(slots.numel()) +
                " slots, not for " + std::to_string(E) + " and " + std::to_string(n));
}

Tensor expert_matmul(const Tensor& X, const Tensor& W, const Tensor& offsets, const Tensor& slots, int64_t tokens, int64_t k,
                     const std::string& rows, int layout, int path, std::optional<at::ScalarType> out_dtype) {
  if (X.dim() < 1 || W.dim() != 3) value_error("expected X[..., C], W[E,.,.]");
  if (W.scalar_type() != X.scalar_type()) value_error("X and W must have the same dtype");
  const int dt = type_id(X.scalar_type()), rid = rows_id(rows);
  const at::ScalarType out = out_dtype.value_or(X.scalar_type());
  if (out != X.scalar_type() && out != at::kFloat) value_error("out_dtype must be X's dtype or float32");
  Call c(X, W);
  const WDims w = w_dims(W, layout);
  check_plan(c, offsets, slots, w.E, tokens * k);
  const int64_t want = rid == EGS_ROWS_TOKENS ? tokens : tokens * k;
  if (X.size(-1) != w.C || X.numel() != want * w.C)
    value_error("shape mismatch: X" + shape_of(X) + " W" + shape_of(W) + " (" + layout_name(layout) + ") for " + std::to_string(want) + " rows");
  const Tensor Xc = whole(X), Wc = whole(W);
  Tensor Y = empty({tokens * k, w.N}, out, c.idx);
  const egs_ragged d{tokens, k, w.E, w.C, w.N};
  const size_t bytes = api.egs_expert_matmul_workspace_bytes(&d, rid, layout, dt);
  const Tensor ws = scratch(bytes, c.idx);
  check(api.egs_expert_matmul_out(ptr(Xc), ptr(Wc), offsets.data_ptr<int>(), slots.data_ptr<int>(), ptr(Y), &d, rid, layout, dt, type_id(out),
                                  path_of(path), ptr(ws), bytes, c.status(), c.stream),
        "egs_expert_matmul");
  c.debug();
  return Y;
}

Tensor expert_dweight(const Tensor& X, const Tensor& dY, const Tensor& offsets, const Tensor& slots, int64_t tokens, int64_t k,
                      const std::string& rows, int path) {
  if (X.dim() < 1 || dY.dim() != 2) value_error("expected X[..., C], dY[tokens * k, N]");
  if (dY.scalar_type() != X.scalar_type()) value_error("X and dY must have the same dtype");
  const int dt = type_id(X.scalar_type()), rid = rows_id(rows);
  Call c(X, dY);
  const int64_t E = offsets.numel() - 1, C = X.size(-1), N = dY.size(1);
  check_plan(c, offsets, slots, E, tokens * k);
  const int64_t want = rid == EGS_ROWS_TOKENS ? tokens : tokens * k;
  if (X.numel() != want * C || dY.size(0) != tokens * k)
    value_error("shape mismatch: X" + shape_of(X) + " dY" + shape_of(dY) + " for " + std::to_string(want) + " and " + std::to_string(tokens * k) + " rows");
  const Tensor Xc = whole(X), Yc = whole(dY);
  Tensor dW = empty({E, C, N}, X.scalar_type(), c.idx);
  const egs_ragged d{tokens, k, E, C, N};
  const size_t bytes = api.egs_expert_dweight_workspace_bytes(&d, rid, dt);
  const Tensor ws = scratch(bytes, c.idx);
  check(api.egs_expert_dweight(ptr(Xc), ptr(Yc), offsets.data_ptr<int>(), slots.data_ptr<int>(), ptr(dW), &d, rid, dt, path_of(path), ptr(ws), bytes,
                               c.status(), c.stream),
        "egs_expert_dweight");
  c.debug();
  return dW;
}

// weights [.., k] in float32 or in `other`; undefined for none
Tensor choice_weights(const OptTensor& weights, const Tensor& Y, at::ScalarType other, int64_t n, int* type) {
  *type = EGS_F32;
  if (!weights || !weights->defined()) return Tensor();
  if (weights->numel() != n) value_error("weights must have one element a slot (" + std::to_string(n) + "), got " + shape_of(*weights));
  if (weights->scalar_type() != at::kFloat && weights->scalar_type() != other) value_error("weights must be float32 or of the rows' dtype");
  if (!weights->is_cuda() || weights->get_device() != Y.get_device()) throw std::runtime_error("all tensors must be on the same CUDA device");
  *type = type_id(weights->scalar_type());
  return weights->contiguous();
}

Tensor combine(const Tensor& Y, const OptTensor& weights, const Tensor& position, int64_t tokens, int64_t k, std::optional<at::ScalarType> out_dtype) {
  if (Y.dim() != 2 || Y.size(0) != tokens * k || position.numel() != tokens * k || position.scalar_type() != at::kInt || !position.is_contiguous())
    value_error("expected Y[" + std::to_string(tokens * k) + ", N], got " + shape_of(Y));
  const int dt = type_id(Y.scalar_type());
  const at::ScalarType type = out_dtype.value_or(Y.scalar_type());
  const int ot = type_id(type);
  if (ot != dt && dt != EGS_F32) value_error("out_dtype must be Y's dtype, or any where Y is float32");
  Call c(Y, position);
  int wt;
  const Tensor w = choice_weights(weights, Y, type, tokens * k, &wt), Yc = whole(Y);
  Tensor out = empty({tokens, Y.size(1)}, type, c.idx);
  check(api.egs_combine_out(ptr(Yc), ptr(w), position.data_ptr<int>(), ptr(out), tokens, k, Y.size(1), dt, wt, ot, c.stream), "egs_combine");
  c.debug();
  return out;
}

std::tuple<Tensor, OptTensor> combine_backward(const Tensor& dOut, const Tensor& Y, const OptTensor& weights, const Tensor& position, int64_t tokens,
                                               int64_t k) {
  if (Y.dim() != 2 || Y.size(0) != tokens * k || dOut.dim() != 2 || dOut.size(0) != tokens || dOut.size(1) != Y.size(1) ||
      position.numel() != tokens * k || position.scalar_type() != at::kInt || !position.is_contiguous())
    value_error("expected dOut[" + std::to_string(tokens) + ", N], Y[" + std::to_string(tokens * k) + ", N], got " + shape_of(dOut) + " " + shape_of(Y));
  if (dOut.scalar_type() != Y.scalar_type()) value_error("dOut and Y must have the same dtype");
  const int dt = type_id(Y.scalar_type());
  Call c(Y, dOut, position);
  int wt;
  const Tensor w = choice_weights(weights, Y, Y.scalar_type(), tokens * k, &wt), Yc = whole(Y), g = whole(dOut);
  Tensor dY = empty({tokens * k, Y.size(1)}, Y.scalar_type(), c.idx);
  OptTensor dw;
  if (w.defined()) dw = empty(weights->sizes(), weights->scalar_type(), c.idx);
  check(api.egs_combine_backward(ptr(g), ptr(Yc), ptr(w), position.data_ptr<int>(), ptr(dY), dw ? ptr(*dw) : nullptr, tokens, k, Y.size(1), dt, wt,
                                 c.stream),
        "egs_combine_backward");
  c.debug();
  return {dY, dw};
}

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& X) {
  if (X.dim() < 1) value_error("expected X[..., C]");
  const int dt = type_id(X.scalar_type());
  Call c(X);
  const Rows r = rows_of(X);
  const int64_t C = X.size(-1), pitch = (C + 15) / 16 * 16;
  auto shape = X.sizes().vec();
  shape.pop_back();
  Tensor scale = empty(shape, at::kFloat, c.idx);
  shape.push_back(pitch);
  Tensor q = empty(shape, at::kChar, c.idx);
  check(api.egs_quantize_rows(ptr(r.t), q.data_ptr<int8_t>(), scale.data_ptr<float>(), scale.numel(), C, r.stride, pitch, dt, c.stream),
        "egs_quantize_rows");
  c.debug();
  return {pitch == C ? q : q.narrow(-1, 0, C), scale};
}

// 8-bit rows [.., C] with elements together and rows of one pitch, a multiple of 16 from a multiple of 16; copied where they are not.
struct Rows8 {
  Tensor t;
  int64_t pitch;
};
Rows8 rows8_of(const Tensor& t) {
  const int64_t C = t.size(-1);
  bool even = (C <= 1 || t.stride(-1) == 1) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
  int64_t pitch = t.dim() > 1 ? t.stride(-2) : (C + 15) / 16 * 16;
  for (int64_t i = t.dim() - 3, p = t.dim() > 1 ? pitch * t.size(-2) : 0; i >= 0; --i) {
    even = even && (t.size(i) == 1 || t.stride(i) == p);
    p *= t.size(i);
  }
  if (t.dim() > 1 && t.size(-2) == 1 && t.dim() == 2) pitch = (C + 15) / 16 * 16;      // one row: any pitch is right
  if (even && pitch >= C && pitch % 16 == 0) return {t, pitch};
  auto shape = t.sizes().vec();
  pitch = shape.back() = (C + 15) / 16 * 16;
  Tensor padded = at::empty(shape, t.options());
  padded.narrow(-1, 0, C).copy_(t);
  return {padded, pitch};
}

// offsets undefined: one expert that has all rows
Tensor matmul_int8(const Tensor& q, const Tensor& q_scale, const Tensor& Wq, const Tensor& w_scale, const OptTensor& offsets, const OptTensor& slots,
                   int64_t tokens, int64_t k, const std::string& rows, at::ScalarType out_dtype, int path) {
  const bool dense = !offsets || !offsets->defined();
  if (q.dim() < 1 || Wq.dim() != (dense ? 2 : 3)) value_error(dense ? "expected q[..., C], Wq[N, C]" : "expected q[..., C], Wq[E, N, C]");
  if (q.scalar_type() != at::kChar || Wq.scalar_type() != at::kChar) value_error("q and Wq must be int8");
  if (q_scale.scalar_type() != at::kFloat || w_scale.scalar_type() != at::kFloat) value_error("the scales must be float32");
  const int dt = type_id(out_dtype), rid = rows_id(rows);
  Call c(q, Wq, q_scale, w_scale);
  const int64_t C = q.size(-1), E = dense ? 1 : Wq.size(0), N = Wq.size(-2), n = C ? q.numel() / C : 0;
  const int64_t row_count = q_scale.numel();
  if (dense) tokens = row_count, k = 1;
  else check_plan(c, *offsets, *slots, E, tokens * k);
  const int64_t want = rid == EGS_ROWS_TOKENS ? tokens : tokens * k;
  if (Wq.size(-1) != C || row_count != want || (C && n != want) || w_scale.numel() != E * N)
    value_error("shape mismatch: q" + shape_of(q) + " scale" + shape_of(q_scale) + " Wq" + shape_of(Wq) + " scale" + shape_of(w_scale) + " for " +
                std::to_string(want) + " rows");
  const Rows8 a = rows8_of(q), b = rows8_of(Wq);
  const Tensor as = q_scale.contiguous(), bs = w_scale.contiguous();
  auto shape = q.sizes().vec();
  shape.back() = N;
  if (!dense) shape = {tokens * k, N};
  Tensor Y = empty(shape, out_dtype, c.idx);
  const egs_ragged d{tokens, k, E, C, N};
  check(api.egs_expert_matmul_int8(static_cast<const int8_t*>(ptr(a.t)), as.data_ptr<float>(), a.pitch, static_cast<const int8_t*>(ptr(b.t)),
                                   bs.data_ptr<float>(), b.pitch, dense ? nullptr : offsets->data_ptr<int>(),
                                   dense ? nullptr : slots->data_ptr<int>(), ptr(Y), &d, rid, dt, path_of(path), c.status(), c.stream),
        "egs_expert_matmul_int8");
  c.debug();
  return Y;
}
