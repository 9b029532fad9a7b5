// torch_step.hpp -- the part of torch_ops.cpp that binds the token embedding,
// dropout, the layer norm and the masked self-attention (included inside its
// namespace, behind what the layers share).

// ------------------------------------------------------------- embedding
orda_embedding_t embedding_problem(int64_t tokens, const Tensor& ids, int64_t vocab, int64_t hidden, ScalarType weight, ScalarType type, double scale,
                                   int64_t padding) {
  orda_embedding_t p{};
  p.abi_version = ORDA_ABI_VERSION;
  p.dtype = code(weight);
  p.out_dtype = code(type);
  p.wide_ids = ids.scalar_type() == at::kLong;
  p.tokens = tokens;
  p.vocab = vocab;
  p.hidden = hidden;
  p.padding_idx = padding;
  p.scale = (float)scale;
  return p;
}
Tensor embedding_run(const Tensor& ids, const Tensor& weight, double scale, int64_t padding, ScalarType type) {
  const c10::DeviceGuard guard(weight.device());
  const Tensor w = rows_of(weight, weight.scalar_type());
  orda_embedding_t p = embedding_problem(ids.numel(), ids, w.size(0), w.size(1), w.scalar_type(), type, scale, padding);
  p.ldw = pitch(w);
  Tensor y = at::empty({ids.numel(), w.size(1)}, w.options().dtype(type));
  check(api.embedding_forward(&p, ptr(ids), ptr(w), out(y), stream_of(w)), "orda_embedding_forward");
  return y;
}

struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
  struct Kept {
    orda_embedding_t p;
    int64_t type, weight_type;
  };
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale, int64_t padding, int64_t type) {
    const Tensor y = embedding_run(ids, weight, scale, padding, static_cast<ScalarType>(type));
    ctx->save_for_backward({ids});
    ctx->saved_data["kept"] = packed(Kept{embedding_problem(ids.numel(), ids, weight.size(0), weight.size(1), weight.scalar_type(),
                                                            static_cast<ScalarType>(type), scale, padding), type, (int64_t)weight.scalar_type()});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list g(5);
    if (!grads[0].defined() || !ctx->needs_input_grad(1)) return g;
    const bool graph = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const c10::DeviceGuard guard(grads[0].device());
    check_capture("token_embedding");
    const Kept kept = unpacked<Kept>(ctx->saved_data["kept"].toStringRef());
    orda_embedding_t p = kept.p;
    Tensor ids = restored(ctx->get_saved_variables()[0], {p.tokens}, grads[0].device());
    if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) ids = ids.to(at::kLong);
    ids = ids.contiguous();
    p.wide_ids = ids.scalar_type() == at::kLong;
    const Tensor dy = rows_of(grads[0], static_cast<ScalarType>(kept.type));
    p.ldg = pitch(dy);
    g[1] = at::empty({p.vocab, p.hidden}, dy.options().dtype(static_cast<ScalarType>(kept.weight_type)));
    const size_t bytes_needed = size_of(api.embedding_workspace_bytes(&p), "orda_embedding_workspace_bytes");
    const Tensor ws = bytes(bytes_needed, dy);
    check(api.embedding_backward(&p, ptr(ids), ptr(dy), out(g[1]), out(ws), bytes_needed, stream_of(dy)), "orda_embedding_backward");
    return once(std::move(g), graph);
  }
};

// ids 1-D, int32 or int64, at least one.
Tensor embedding(const Tensor& ids_, const Tensor& weight, double scale, int64_t padding, ScalarType type, bool record) {
  const Tensor ids = ids_.contiguous();
  if (record) return EmbeddingNode::apply(ids, weight, scale, padding, (int64_t)type);
  const at::AutoGradMode off(false);
  return embedding_run(ids, weight, scale, padding, type);
}

// ------------------------------------------------------------- dropout
struct Drop {
  double p;
  uint64_t seed, site;
  Tensor on_device;  // or undefined
  orda_dropout_t c() const { return {p, seed, on_device.defined() ? on_device.const_data_ptr<int64_t>() : nullptr, site}; }
};
// What a node keeps of it beside the seed's tensor.
struct KeptDrop {
  double p;
  uint64_t seed, site;
  int64_t on_device;
};
KeptDrop kept_drop(const Drop& d) { return {d.p, d.seed, d.site, d.on_device.defined()}; }
// seed: what the node saved of the seed's tensor
Drop restored_drop(const KeptDrop& k, const Tensor& seed, const c10::Device& device) {
  return {k.p, k.seed, k.site, k.on_device ? restored_dense(seed, {1}, at::kLong, device) : Tensor()};
}

Tensor dropout_run(const Tensor& x_, const Tensor& res_, const Drop& d, ScalarType type) {
  const c10::DeviceGuard guard(x_.device());
  Tensor x = x_.scalar_type() == type ? x_ : x_.to(type), r = !res_.defined() || res_.scalar_type() == type ? res_ : res_.to(type);
  orda_rows_problem_t p{ORDA_ABI_VERSION, code(type), 1, x.numel(), 0, 0};
  Tensor y = at::empty(x.sizes(), x.options());
  if (x.size(-1) > (1 << 22)) {  // (rows longer than a pitch may be: one dense row)
    x = x.contiguous();
    if (r.defined()) r = r.contiguous();
  } else if (!x.is_contiguous() || (r.defined() && !r.is_contiguous())) {  // row by row
    x = rows_of(x.reshape({-1, x.size(-1)}), type);
    if (r.defined()) r = rows_of(r.reshape({-1, r.size(-1)}), type);
    p.rows = x.size(0);
    p.cols = x.size(1);
    p.ldx = pitch(x);
    p.ldr = r.defined() ? pitch(r) : 0;
  }
  const orda_dropout_t c = d.c();
  check(api.dropout_add(&p, &c, ptr(x), ptr(r), out(y), stream_of(x)), "orda_dropout_add");
  return y;
}

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  struct Kept {
    KeptDrop drop;
    int64_t types[4];
  };
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& res_, double p, int64_t seed, int64_t site, const OptTensor& on_device, int64_t type) {
    const ScalarType t = static_cast<ScalarType>(type);
    const Drop d{p, (uint64_t)seed, (uint64_t)site, given(on_device)};
    const Tensor res = given(res_);
    ctx->save_for_backward({d.on_device});
    ctx->saved_data["kept"] = packed(Kept{kept_drop(d), {type, type_or(x, t), type_or(res, t), res.defined()}});
    return dropout_run(x, res, d, t);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list g(7);
    if (!grads[0].defined()) return g;
    const bool graph = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const Kept kept = unpacked<Kept>(ctx->saved_data["kept"].toStringRef());
    auto type = [&](int i) { return static_cast<ScalarType>(kept.types[i]); };
    if (kept.types[3] && ctx->needs_input_grad(1)) g[1] = grads[0].to(type(2));
    if (ctx->needs_input_grad(0)) {
      const c10::DeviceGuard guard(grads[0].device());
      check_capture("counter_dropout");
      const Drop d = restored_drop(kept.drop, ctx->get_saved_variables()[0], grads[0].device());
      g[0] = as_type(dropout_run(grads[0], Tensor(), d, type(0)), type(1));
    }
    return once(std::move(g), graph);
  }
};

Tensor dropout(const Tensor& x, const OptTensor& res, double p, uint64_t seed, uint64_t site, const OptTensor& on_device, ScalarType type, bool record) {
  if (record) return DropoutNode::apply(x, res, p, (int64_t)seed, (int64_t)site, on_device, (int64_t)type);
  const at::AutoGradMode off(false);
  return dropout_run(x, given(res), Drop{p, seed, site, given(on_device)}, type);
}

// ------------------------------------------------------------- layer norm
// Weight and bias in one type that the kernels take: the tensors', or fp32.
ScalarType param_type(ScalarType type, const Tensor& w, const Tensor& b) {
  return w.scalar_type() == type && (!b.defined() || b.scalar_type() == type) ? type : at::kFloat;
}
struct NormCall {
  Tensor s, r, w, y, stats;  // with r: the backward pass computes s again from x (in s) and r
  Tensor stream;             // s as the call returns it
  orda_layer_norm_t p{};
};
NormCall norm_run(const Tensor& x_, const Tensor& w, const Tensor& b_, const Tensor& res, double eps, const Drop& d, ScalarType type, bool keep) {
  const c10::DeviceGuard guard(x_.device());
  NormCall c;
  const Tensor x = rows_of(x_, type), r = res.defined() ? rows_of(res, type) : Tensor();
  const ScalarType pt = param_type(type, w, b_);
  c.w = w.to(pt).contiguous();
  const Tensor b = b_.defined() ? b_.to(pt).contiguous() : Tensor();
  c.p.abi_version = ORDA_ABI_VERSION;
  c.p.dtype = code(type);
  c.p.param_dtype = code(pt);
  c.p.eps = (float)eps;
  c.p.rows = x.size(0);
  c.p.cols = x.size(1);
  c.p.ldx = pitch(x);
  c.p.ldr = r.defined() ? pitch(r) : 0;
  c.y = at::empty(x.sizes(), x.options());
  if (r.defined()) c.stream = at::empty(x.sizes(), x.options());
  if (keep) c.stats = at::empty({x.size(0), 2}, x.options().dtype(at::kFloat));
  const orda_dropout_t drop = d.c();
  check(api.layer_norm_forward(&c.p, &drop, ptr(x), ptr(r), ptr(c.w), ptr(b), out(c.y), out(c.stream), static_cast<float*>(out(c.stats)), stream_of(x)),
        "orda_layer_norm_forward");
  const bool again = r.defined() && pt != type;
  c.s = r.defined() && !again ? c.stream : x;
  if (again) c.r = r;
  return c;
}

struct NormNode : torch::autograd::Function<NormNode> {
  struct Kept {
    orda_layer_norm_t p;
    KeptDrop drop;
    int64_t types[7];
  };
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b_, const OptTensor& res_, double eps, double p,
                               int64_t seed, int64_t site, const OptTensor& on_device, int64_t type) {
    const ScalarType t = static_cast<ScalarType>(type);
    const Tensor b = given(b_), res = given(res_);
    const Drop d{p, (uint64_t)seed, (uint64_t)site, given(on_device)};
    NormCall c = norm_run(x, w, b, res, eps, d, t, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({c.s, c.stats, c.w, d.on_device, c.r});
    ctx->saved_data["kept"] = packed(Kept{c.p, kept_drop(d), {type, type_or(x, t), type_or(w, t), type_or(b, t), type_or(res, t), b.defined(), res.defined()}});
    return res.defined() ? variable_list{c.y, c.stream} : variable_list{c.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list g(10);
    const Tensor& any = grads[0].defined() ? grads[0] : grads.back();
    if (!any.defined()) return g;
    const bool graph = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const c10::Device device = any.device();
    const c10::DeviceGuard guard(device);
    const Kept kept = unpacked<Kept>(ctx->saved_data["kept"].toStringRef());
    orda_layer_norm_t p = kept.p;
    auto type = [&](int i) { return static_cast<ScalarType>(kept.types[i]); };
    const ScalarType t = type(0), pt = p.param_dtype == ORDA_F32 ? at::kFloat : t;
    const bool has_b = kept.types[5] != 0, has_r = kept.types[6] != 0;
    // (edges are numbered over the tensors that were given)
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = has_b && ctx->needs_input_grad(2);
    const bool nr = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    if (!nx && !nw && !nb && !nr) return g;
    check_capture("layer_norm");
    const variable_list v = ctx->get_saved_variables();
    const Tensor s = rows_of(restored(v[0], {p.rows, p.cols}, device), t);
    const Tensor stats = restored_dense(v[1], {p.rows, 2}, at::kFloat, device), w = restored_dense(v[2], {p.cols}, pt, device);
    const Tensor r = has_r && pt != t ? rows_of(restored(v[4], {p.rows, p.cols}, device), t) : Tensor();
    const Drop d = restored_drop(kept.drop, v[3], device);
    const Tensor dy = grads[0].defined() ? rows_of(grads[0], t) : at::zeros({p.rows, p.cols}, any.options().dtype(t));
    const Tensor ds = has_r && grads[1].defined() ? rows_of(grads[1], t) : Tensor();
    p.ld_s = pitch(s);
    p.ldr = r.defined() ? pitch(r) : 0;
    p.ld_dy = pitch(dy);
    p.ld_ds = ds.defined() ? pitch(ds) : 0;
    const bool drops = std::floor(d.p * 65536.0 + 0.5) > 0.0;  // (else dx and dr are one)
    Tensor dx, dr, dw, db;
    if (nx || (nr && !drops)) dx = at::empty({p.rows, p.cols}, dy.options());
    if (nr && drops) dr = at::empty({p.rows, p.cols}, dy.options());
    if (nw) dw = at::empty({p.cols}, dy.options().dtype(pt));
    if (nb) db = at::empty({p.cols}, dy.options().dtype(pt));
    const size_t n = size_of(api.layer_norm_workspace_bytes(&p), "orda_layer_norm_workspace_bytes");
    const Tensor ws = nw || nb ? bytes(n, dy) : Tensor();
    const orda_dropout_t drop = d.c();
    check(api.layer_norm_backward(&p, &drop, ptr(s), ptr(r), static_cast<const float*>(ptr(stats)), ptr(w), ptr(dy), ptr(ds), out(dx), out(dr), out(dw), out(db),
                                  out(ws), ws.defined() ? n : 0, stream_of(dy)), "orda_layer_norm_backward");
    if (nx) g[0] = as_type(dx, type(1));
    if (nr) g[3] = as_type(drops ? dr : dx, type(4));
    g[1] = as_type(dw, type(2));
    g[2] = as_type(db, type(3));
    return once(std::move(g), graph);
  }
};

// x and residual 2-D, at least one row: {y}, with a residual {y, s}.
std::vector<Tensor> layer_norm(const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& res, double eps, double p, uint64_t seed, uint64_t site,
                               const OptTensor& on_device, ScalarType type, bool record) {
  if (record) return NormNode::apply(x, w, b, res, eps, p, (int64_t)seed, (int64_t)site, on_device, (int64_t)type);
  const at::AutoGradMode off(false);
  NormCall c = norm_run(x, w, given(b), given(res), eps, Drop{p, seed, site, given(on_device)}, type, false);
  return given(res).defined() ? std::vector<Tensor>{c.y, c.stream} : std::vector<Tensor>{c.y};
}

// ------------------------------------------------------------- attention
// (batch, length, heads, D) as the kernels read it: D padded with zeros to a
// multiple of 8 (`width`), rows of a head 16-byte aligned, positions at most
// 2^22 elements apart.
Tensor head_rows(const Tensor& given, ScalarType type, int64_t width) {
  Tensor t = given.scalar_type() == type ? given : given.to(type);
  if (t.size(3) != width) return at::constant_pad_nd(t, {0, width - t.size(3)}).contiguous();
  bool fits = aligned(t) && (t.stride(3) == 1 || width == 1) && (t.size(1) == 1 || t.stride(1) <= (1 << 22));
  for (int i = 0; i < 3; ++i) fits = fits && (t.size(i) == 1 || (t.stride(i) >= 0 && t.stride(i) % 8 == 0));
  if (fits) return t;
  t = t.contiguous();
  return aligned(t) ? t : t.clone();
}
void set_strides(int64_t (&s)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}

struct AttentionCall {
  Tensor q, k, v, o, saved;  // o: with padded heads
  orda_attention_t p{};
};
AttentionCall attention_run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& slopes, const Tensor& docs, const Tensor& prefix, bool causal,
                            double scale, double softcap, ScalarType type, bool keep) {
  const c10::DeviceGuard guard(q.device());
  AttentionCall c;
  const int64_t D = q.size(3), width = padded(D, type);
  c.q = head_rows(q, type, width);
  c.k = head_rows(k, type, width);
  c.v = head_rows(v, type, width);
  orda_attention_t& p = c.p;
  p.abi_version = ORDA_ABI_VERSION;
  p.dtype = code(type);
  p.heads = (int32_t)q.size(2);
  p.kv_heads = (int32_t)k.size(2);
  p.head_dim = (int32_t)width;
  p.causal = causal;
  p.batch = q.size(0);
  p.length = q.size(1);
  p.scale = scale;
  p.softcap = softcap;
  set_strides(p.q_stride, c.q);
  set_strides(p.k_stride, c.k);
  set_strides(p.v_stride, c.v);
  if (docs.defined()) p.documents_stride = docs.stride(0);
  c.o = at::empty({q.size(0), q.size(1), q.size(2), width}, c.q.options());
  const size_t n = size_of(api.attention_saved_bytes(&p, docs.defined(), keep), "orda_attention_saved_bytes");
  if (docs.defined() || keep) c.saved = bytes(n, c.q);
  check(api.attention_forward(&p, ptr(c.q), ptr(c.k), ptr(c.v), static_cast<const float*>(ptr(slopes)), static_cast<const int32_t*>(ptr(docs)),
                              static_cast<const int32_t*>(ptr(prefix)), out(c.o), out(c.saved), n, keep, stream_of(c.q)), "orda_attention_forward");
  return c;
}
Tensor without_padding(const Tensor& t, int64_t D) { return t.size(3) == D ? t : t.narrow(3, 0, D).contiguous(); }

struct AttentionNode : torch::autograd::Function<AttentionNode> {
  struct Kept {
    orda_attention_t p;
    int64_t types[8];
  };
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& slopes_, const OptTensor& docs_,
                        const OptTensor& prefix_, bool causal, double scale, double softcap, int64_t type) {
    const ScalarType t = static_cast<ScalarType>(type);
    const Tensor slopes = given(slopes_), docs = given(docs_), prefix = given(prefix_);
    AttentionCall c = attention_run(q, k, v, slopes, docs, prefix, causal, scale, softcap, t, true);
    const Tensor y = without_padding(c.o, q.size(3));
    ctx->save_for_backward({c.q, c.k, c.v, c.o, c.saved, slopes, prefix});
    ctx->saved_data["kept"] = packed(Kept{c.p, {type, type_or(q, t), type_or(k, t), type_or(v, t), docs.defined(), slopes.defined(), prefix.defined(), q.size(3)}});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list g(10);
    if (!grads[0].defined()) return g;
    const bool graph = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const c10::Device device = grads[0].device();
    const c10::DeviceGuard guard(device);
    const bool n[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
    if (!n[0] && !n[1] && !n[2]) return g;
    check_capture("masked_attention");
    const Kept node = unpacked<Kept>(ctx->saved_data["kept"].toStringRef());
    orda_attention_t p = node.p;
    const int64_t(&types)[8] = node.types;
    const ScalarType t = static_cast<ScalarType>(types[0]);
    const variable_list s = ctx->get_saved_variables();
    const int64_t width = p.head_dim, rows[4] = {p.batch, p.length, p.heads, width}, kv[4] = {p.batch, p.length, p.kv_heads, width};
    const Tensor q = head_rows(restored(s[0], rows, device), t, width), k = head_rows(restored(s[1], kv, device), t, width);
    const Tensor v = head_rows(restored(s[2], kv, device), t, width), o = restored_dense(s[3], rows, t, device);
    const int64_t kept = (int64_t)size_of(api.attention_saved_bytes(&p, types[4] != 0, 1), "orda_attention_saved_bytes");
    const Tensor saved = restored_dense(s[4], {kept}, at::kByte, device);
    const Tensor slopes = types[5] ? restored_dense(s[5], {p.heads}, at::kFloat, device) : Tensor();
    const Tensor prefix = types[6] ? restored_dense(s[6], {p.batch}, at::kInt, device) : Tensor();
    const Tensor dy = head_rows(grads[0], t, width);
    set_strides(p.q_stride, q);
    set_strides(p.k_stride, k);
    set_strides(p.v_stride, v);
    set_strides(p.g_stride, dy);
    Tensor d[3];
    for (int i = 0; i < 3; ++i)
      if (n[i]) d[i] = at::empty(at::IntArrayRef(i ? kv : rows, 4), dy.options());
    const size_t need = size_of(api.attention_workspace_bytes(&p), "orda_attention_workspace_bytes");
    const Tensor ws = bytes(need, dy);
    check(api.attention_backward(&p, ptr(q), ptr(k), ptr(v), static_cast<const float*>(ptr(slopes)), types[4] != 0, static_cast<const int32_t*>(ptr(prefix)),
                                 ptr(o), ptr(saved), (size_t)kept, ptr(dy), out(d[0]), out(d[1]), out(d[2]), out(ws), need, stream_of(dy)),
          "orda_attention_backward");
    for (int i = 0; i < 3; ++i)
      if (n[i]) g[i] = as_type(without_padding(d[i], types[7]), static_cast<ScalarType>(types[1 + i]));
    return once(std::move(g), graph);
  }
};

// q (batch, length, heads, D), k and v (batch, length, kv_heads, D), none empty;
// slopes fp32, documents and prefix int32, rows of documents contiguous.
Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& slopes, const OptTensor& docs, const OptTensor& prefix, bool causal,
                 double scale, double softcap, ScalarType type, bool record) {
  if (record) return AttentionNode::apply(q, k, v, slopes, docs, prefix, causal, scale, softcap, (int64_t)type);
  const at::AutoGradMode off(false);
  AttentionCall c = attention_run(q, k, v, given(slopes), given(docs), given(prefix), causal, scale, softcap, type, false);
  return without_padding(c.o, q.size(3));
}
