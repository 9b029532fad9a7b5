// torch_ops.cpp -- the binding of orda_linear_*, orda_ffn_*, orda_grad_norm and
// orda_clip_grads to torch: operands as the kernels read them, workspaces and
// outputs from torch's allocator, autograd nodes, tables of gradients.  Host
// code only; it reaches the C entry points through the addresses that
// _native.py hands over, so one library is loaded.  Measured against the same
// steps in Python (ctypes and a Python autograd Function): forward and backward
// of a 4 x 64 x 64 projection 81 us instead of 195, most of which was Python on
// the autograd engine's thread.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPGraphsC10Utils.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <map>
#include <optional>
#include <string>
#include <tuple>
#include <unordered_map>
#include <utility>
#include <vector>

#include "../../include/orda_ce.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------- the library
struct Api {
  decltype(&orda_last_error) last_error;
  decltype(&orda_pad_rows) pad_rows;
  decltype(&orda_linear_saved_bytes) linear_saved_bytes;
  decltype(&orda_linear_workspace_bytes) linear_workspace_bytes;
  decltype(&orda_linear_forward) linear_forward;
  decltype(&orda_linear_backward) linear_backward;
  decltype(&orda_ffn_inner_pitch) ffn_inner_pitch;
  decltype(&orda_ffn_saved_bytes) ffn_saved_bytes;
  decltype(&orda_ffn_workspace_bytes) ffn_workspace_bytes;
  decltype(&orda_ffn_forward) ffn_forward;
  decltype(&orda_ffn_backward) ffn_backward;
  decltype(&orda_grad_norm_workspace_bytes) grad_norm_workspace_bytes;
  decltype(&orda_grad_norm) grad_norm;
  decltype(&orda_clip_grads) clip_grads;
  decltype(&orda_clip_grad_norm) clip_grad_norm;
} api;

void bind(const std::map<std::string, uintptr_t>& at) {
#define ORDA_BIND(name) api.name = reinterpret_cast<decltype(api.name)>(at.at("orda_" #name))
  ORDA_BIND(last_error);
  ORDA_BIND(pad_rows);
  ORDA_BIND(linear_saved_bytes);
  ORDA_BIND(linear_workspace_bytes);
  ORDA_BIND(linear_forward);
  ORDA_BIND(linear_backward);
  ORDA_BIND(ffn_inner_pitch);
  ORDA_BIND(ffn_saved_bytes);
  ORDA_BIND(ffn_workspace_bytes);
  ORDA_BIND(ffn_forward);
  ORDA_BIND(ffn_backward);
  ORDA_BIND(grad_norm_workspace_bytes);
  ORDA_BIND(grad_norm);
  ORDA_BIND(clip_grads);
  ORDA_BIND(clip_grad_norm);
#undef ORDA_BIND
}

// The errors _native.py raises: ORDA_EINVAL a ValueError, others RuntimeError.
void check(int rc, const char* what) {
  if (rc == ORDA_OK) return;
  const std::string msg = api.last_error();
  TORCH_CHECK_VALUE(rc != ORDA_EINVAL, what, ": ", msg);
  TORCH_CHECK(false, what, " failed (", rc, "): ", msg);
}
size_t size_of(size_t n, const char* what) {
  if (n == 0) check(ORDA_EINVAL, what);
  return n;
}

int32_t code(ScalarType t) {
  switch (t) {
    case at::kBFloat16: return ORDA_BF16;
    case at::kHalf: return ORDA_F16;
    case at::kFloat: return ORDA_F32;
    default: TORCH_CHECK_VALUE(false, "expected bfloat16, float16 or float32, got ", t);
  }
}
int64_t granule(ScalarType t) { return t == at::kFloat ? 4 : 8; }
int64_t padded(int64_t n, ScalarType t) { return (n + granule(t) - 1) / granule(t) * granule(t); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }
Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}
void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// ------------------------------------------------------------- operands
// 2-D operands as the kernels read them: contiguous rows, a multiple of 16
// bytes apart, 16-byte aligned, zero-padded.  Tensors that are so stay where
// they are; those that lack padding or alignment are copied, up to four in one
// launch.
struct Operands {
  ScalarType type;
  std::vector<orda_rows_t> copies;
  std::vector<Tensor> alive;
  explicit Operands(ScalarType t) : type(t) {}
  Tensor add(const Tensor& given) {
    Tensor t = given.scalar_type() == type ? given : given.to(type);
    const int64_t rows = t.size(0), cols = t.size(1), g = granule(type);
    // (a pitch past 2^22 is more than the C entry points take)
    if ((t.stride(1) != 1 && cols > 1) || (rows > 1 && (t.stride(0) < cols || t.stride(0) > (1 << 22)))) t = t.contiguous();
    const int64_t ld = rows > 1 ? t.stride(0) : cols;
    if (cols % g == 0 && (rows == 1 || ld % g == 0) && aligned(t)) return t;
    Tensor p = at::empty({rows, padded(cols, type)}, t.options());
    copies.push_back({t.const_data_ptr(), p.data_ptr(), rows, cols, ld, p.size(1)});
    alive.push_back(t);
    return p;
  }
  void copy(void* stream) {
    constexpr size_t kMost = 4;  // of one orda_pad_rows call
    for (size_t i = 0; i < copies.size(); i += kMost)
      check(api.pad_rows(code(type), copies.data() + i, (int64_t)std::min(kMost, copies.size() - i), stream), "orda_pad_rows");
  }
};
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Two weights of one shape with one pitch (a row-strided one beside another is
// copied).
std::pair<Tensor, Tensor> add_pair(Operands& ops, const Tensor& a, const Tensor& b) {
  const bool same = a.size(0) == 1 || a.strides() == b.strides();
  std::pair<Tensor, Tensor> p(ops.add(same ? a : a.contiguous()), ops.add(same ? b : b.contiguous()));
  if (pitch(p.first) != pitch(p.second)) {
    p.first = p.first.contiguous();
    p.second = p.second.contiguous();
  }
  return p;
}

// What a node saved, as the backward pass reads it.  Saved-tensor hooks
// (offloading to the host, for one) may hand back a copy, dense where the saved
// tensor's rows were apart, so that pitches, alignment and dtype are taken from
// what they hand back; its shape and device have to be the saved one's.
const Tensor& restored(const Tensor& t, at::IntArrayRef sizes, const c10::Device& device) {
  TORCH_CHECK(t.defined() && t.sizes() == sizes && t.device() == device, "a saved tensor of shape ", sizes, " on ", device,
              " came back from its hooks ", t.defined() ? "with another shape or on another device" : "undefined");
  return t;
}
// Kept factors and h: dense and 16-byte aligned.
Tensor restored_dense(const Tensor& t, at::IntArrayRef sizes, ScalarType type, const c10::Device& device) {
  Tensor d = restored(t, sizes, device).to(type).contiguous();
  return aligned(d) ? d : d.clone();
}

// Contiguous rows of any pitch up to 2^22 and any alignment.
Tensor rows_of(const Tensor& given, ScalarType type) {
  Tensor t = given.scalar_type() == type ? given : given.to(type);
  if ((t.stride(1) != 1 && t.size(1) > 1) || (t.size(0) > 1 && (t.stride(0) < t.size(1) || t.stride(0) > (1 << 22)))) t = t.contiguous();
  return t;
}

// Dense, so that accumulating it into a leaf copies nothing.
Tensor gradient(const Tensor& like, int64_t rows, int64_t cols, ScalarType type) {
  return at::empty({rows, cols}, like.options().dtype(type));
}
// A gradient in its own tensor's dtype.  Beside 16-bit operands that of an fp32
// tensor has the compute dtype's value, as under torch's autocast: a second set
// of epilogues would be needed to write the accumulators themselves.
Tensor as_type(const Tensor& g, ScalarType type) { return !g.defined() || g.scalar_type() == type ? g : g.to(type); }

// Gradients of a node that is differentiable once: with create_graph (`graph`)
// a second backward through them raises.
variable_list once(variable_list grads, bool graph) {
  if (!graph) return grads;
  const at::AutoGradMode on(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)grads.size());
  variable_list in;
  for (Tensor& g : grads) in.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
  return (*node)(std::move(in));
}

// A leaf's gradient is accumulated on the stream where its first live graph was
// made.  If that is the default stream and this backward pass is being captured,
// autograd would draw the default stream into the capture, which no capture
// allows, and end the process: the call is refused here instead, while the
// capture is whole.
void check_capture(const char* entry) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node();
  if (!node) return;
  for (const torch::autograd::Edge& e : node->next_edges()) {
    if (!dynamic_cast<torch::autograd::AccumulateGrad*>(e.function.get())) continue;
    const std::optional<c10::Stream> s = e.function->stream();
    TORCH_CHECK(!s || c10::hip::HIPStreamMasqueradingAsCUDA(*s).stream() != nullptr, entry,
                ": this backward pass is being captured, and a graph of the same leaf made on the default stream is alive; delete "
                "what holds it (an earlier output or loss), or give the captured call leaf.detach().requires_grad_()");
  }
}

template <class P>
std::string packed(const P& p) { return std::string(reinterpret_cast<const char*>(&p), sizeof(p)); }
template <class P>
P unpacked(const std::string& s) {
  P p;
  memcpy(&p, s.data(), sizeof(p));
  return p;
}
int64_t type_or(const Tensor& t, ScalarType other) { return (int64_t)(t.defined() ? t.scalar_type() : other); }

// ------------------------------------------------------------- projection
struct LinearCall {
  Tensor x, w, d, y;
  orda_linear_t p{};
};
LinearCall linear_run(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& res, int64_t act, ScalarType type, bool keep) {
  const c10::DeviceGuard guard(x.device());
  void* s = stream_of(x);
  LinearCall c;
  Operands ops(type);
  c.x = ops.add(x);
  c.w = ops.add(w);
  ops.copy(s);
  const Tensor b = bias.defined() ? bias.to(type).contiguous() : Tensor();
  const Tensor r = res.defined() ? rows_of(res, type) : Tensor();
  c.p = {ORDA_ABI_VERSION, code(type), (int32_t)act, 0, x.size(0), x.size(1), w.size(0), pitch(c.x), pitch(c.w),
         r.defined() ? pitch(r) : 0, x.size(1), x.size(1)};
  c.y = at::empty({x.size(0), w.size(0)}, x.options().dtype(type));
  if (keep && act != ORDA_ACT_NONE) c.d = bytes(size_of(api.linear_saved_bytes(&c.p), "orda_linear_saved_bytes"), x);
  const size_t n = size_of(api.linear_workspace_bytes(&c.p, 0), "orda_linear_workspace_bytes");
  const Tensor ws = bytes(n, x);
  check(api.linear_forward(&c.p, ptr(c.x), ptr(c.w), ptr(b), ptr(r), out(c.y), out(c.d), out(ws), n, s), "orda_linear_forward");
  return c;
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias_, const OptTensor& res_, int64_t act, int64_t type) {
    const ScalarType t = static_cast<ScalarType>(type);
    const Tensor bias = given(bias_), res = given(res_);
    LinearCall c = linear_run(x, w, bias, res, act, t, true);
    ctx->save_for_backward({c.x, c.w, c.d});
    ctx->saved_data["p"] = packed(c.p);
    ctx->saved_data["types"] = std::vector<int64_t>{type, type_or(x, t), type_or(w, t), type_or(bias, t), type_or(res, t), bias.defined(), res.defined()};
    return c.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list g(6);
    if (!grads[0].defined()) return g;
    const bool graph = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const variable_list saved = ctx->get_saved_variables();
    orda_linear_t p = unpacked<orda_linear_t>(ctx->saved_data["p"].toStringRef());
    const std::vector<int64_t> types = ctx->saved_data["types"].toIntVector();
    auto type = [&](int i) { return static_cast<ScalarType>(types[i]); };
    const ScalarType t = type(0);
    // (edges are numbered over the tensors that were given)
    const bool has_b = types[5] != 0, has_r = types[6] != 0;
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = has_b && ctx->needs_input_grad(2);
    if (has_r && ctx->needs_input_grad(has_b ? 3 : 2)) g[3] = grads[0].to(type(4));
    if (nx || nw || nb) {
      const c10::DeviceGuard guard(grads[0].device());
      check_capture("fused_linear");
      const Tensor dy = grads[0].to(t).contiguous();
      void* s = stream_of(dy);
      const int64_t kp = padded(p.in_features, t);
      Operands ops(t);
      Tensor x, w, d;
      if (nw) p.ldx = pitch(x = ops.add(restored(saved[0], {p.tokens, kp}, dy.device())));
      if (nx) p.ldw = pitch(w = ops.add(restored(saved[1], {p.out_features, kp}, dy.device())));
      ops.copy(s);
      if (p.activation != ORDA_ACT_NONE)
        d = restored_dense(saved[2], {(int64_t)size_of(api.linear_saved_bytes(&p), "orda_linear_saved_bytes")}, at::kByte, dy.device());
      if (nx) g[0] = gradient(dy, p.tokens, p.in_features, t);
      if (nw) g[1] = gradient(dy, p.out_features, p.in_features, t);
      if (nb) g[2] = at::empty({p.out_features}, dy.options());
      const size_t n = size_of(api.linear_workspace_bytes(&p, 1), "orda_linear_workspace_bytes");
      const Tensor ws = bytes(n, dy);
      check(api.linear_backward(&p, ptr(x), ptr(w), ptr(d), ptr(dy), out(g[0]), out(g[1]), out(g[2]), out(ws), n, s), "orda_linear_backward");
      for (int i = 0; i < 3; ++i) g[i] = as_type(g[i], type(i + 1));
    }
    return once(std::move(g), graph);
  }
};

// x and residual 2-D, at least one row.  record: autograd sees the call.
Tensor linear(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& res, int64_t act, ScalarType type, bool record) {
  if (record) return LinearNode::apply(x, w, bias, res, act, (int64_t)type);
  const at::AutoGradMode off(false);
  return linear_run(x, w, given(bias), given(res), act, type, false).y;
}

// ------------------------------------------------------------- feed-forward
struct FfnCall {
  Tensor x, gate, up, down, h, da, db, y;
  orda_ffn_t p{};
};
FfnCall ffn_run(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const Tensor& res, int64_t act, ScalarType type, bool keep) {
  const c10::DeviceGuard guard(x.device());
  void* s = stream_of(x);
  FfnCall c;
  Operands ops(type);
  c.x = ops.add(x);
  std::tie(c.gate, c.up) = add_pair(ops, wg, wu);
  c.down = ops.add(wd);
  ops.copy(s);
  const Tensor r = res.defined() ? rows_of(res, type) : Tensor();
  const int64_t N = x.size(0), H = x.size(1), F = wg.size(0), O = wd.size(0);
  c.p = {ORDA_ABI_VERSION, code(type), (int32_t)act, 0, N, H, F, O, pitch(c.x), pitch(c.gate), pitch(c.down),
         r.defined() ? pitch(r) : 0, padded(O, type), H, H, F};
  c.y = at::empty({N, O}, x.options().dtype(type));
  c.h = at::empty({N, (int64_t)size_of((size_t)api.ffn_inner_pitch(&c.p), "orda_ffn_inner_pitch")}, c.y.options());
  if (keep) {
    const size_t n = size_of(api.ffn_saved_bytes(&c.p), "orda_ffn_saved_bytes");
    c.da = bytes(n, x);
    c.db = bytes(n, x);
  }
  const size_t n = size_of(api.ffn_workspace_bytes(&c.p, 0), "orda_ffn_workspace_bytes");
  const Tensor ws = bytes(n, x);
  check(api.ffn_forward(&c.p, ptr(c.x), ptr(c.gate), ptr(c.up), ptr(c.down), ptr(r), out(c.y), out(c.h), out(c.da), out(c.db), out(ws), n, s),
        "orda_ffn_forward");
  return c;
}

struct FfnNode : torch::autograd::Function<FfnNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const OptTensor& res_, int64_t act, int64_t type) {
    const ScalarType t = static_cast<ScalarType>(type);
    const Tensor res = given(res_);
    FfnCall c = ffn_run(x, wg, wu, wd, res, act, t, true);
    ctx->save_for_backward({c.x, c.gate, c.up, c.down, c.h, c.da, c.db});
    ctx->saved_data["p"] = packed(c.p);
    ctx->saved_data["types"] = std::vector<int64_t>{type, type_or(x, t), type_or(wg, t), type_or(wu, t), type_or(wd, t), type_or(res, t), res.defined()};
    return c.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list g(7);
    if (!grads[0].defined()) return g;
    const bool graph = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const variable_list v = ctx->get_saved_variables();
    orda_ffn_t p = unpacked<orda_ffn_t>(ctx->saved_data["p"].toStringRef());
    const std::vector<int64_t> types = ctx->saved_data["types"].toIntVector();
    auto type = [&](int i) { return static_cast<ScalarType>(types[i]); };
    const ScalarType t = type(0);
    bool any = false;
    const int64_t rows[4] = {p.tokens, p.inner, p.inner, p.out_features}, cols[4] = {p.hidden, p.hidden, p.hidden, p.inner};
    if (types[6] != 0 && ctx->needs_input_grad(4)) g[4] = grads[0].to(type(5));
    const c10::Device device = grads[0].device();
    for (int i = 0; i < 4; ++i) any = any || ctx->needs_input_grad(i);
    if (any) {
      const c10::DeviceGuard guard(device);
      check_capture("gated_feed_forward");
      void* s = stream_of(grads[0]);
      const int64_t hp = padded(p.hidden, t), kept = (int64_t)size_of(api.ffn_saved_bytes(&p), "orda_ffn_saved_bytes");
      Operands ops(t);
      const Tensor dy = ops.add(grads[0]), x = ops.add(restored(v[0], {p.tokens, hp}, device));
      const auto [gate, up] = add_pair(ops, restored(v[1], {p.inner, hp}, device), restored(v[2], {p.inner, hp}, device));
      const Tensor down = ops.add(restored(v[3], {p.out_features, padded(p.inner, t)}, device));
      ops.copy(s);
      const Tensor h = restored_dense(v[4], {p.tokens, api.ffn_inner_pitch(&p)}, t, device);
      const Tensor da = restored_dense(v[5], {kept}, at::kByte, device), db = restored_dense(v[6], {kept}, at::kByte, device);
      p.ldg = pitch(dy);
      p.ldx = pitch(x);
      p.ldw = pitch(gate);
      p.ldd = pitch(down);
      for (int i = 0; i < 4; ++i)
        if (ctx->needs_input_grad(i)) g[i] = gradient(dy, rows[i], cols[i], t);
      const size_t n = size_of(api.ffn_workspace_bytes(&p, 1), "orda_ffn_workspace_bytes");
      const Tensor ws = bytes(n, dy);
      check(api.ffn_backward(&p, ptr(x), ptr(gate), ptr(up), ptr(down), ptr(h), ptr(da), ptr(db), ptr(dy), out(g[0]), out(g[1]), out(g[2]),
                             out(g[3]), out(ws), n, s), "orda_ffn_backward");
      for (int i = 0; i < 4; ++i) g[i] = as_type(g[i], type(i + 1));
    }
    return once(std::move(g), graph);
  }
};

Tensor feed_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const OptTensor& res, int64_t act, ScalarType type, bool record) {
  if (record) return FfnNode::apply(x, wg, wu, wd, res, act, (int64_t)type);
  const at::AutoGradMode off(false);
  return ffn_run(x, wg, wu, wd, given(res), act, type, false).y;
}

// ------------------------------------------------------------- gradients
void check_grad(const char* entry, const Tensor& g, const c10::Device& device) {
  TORCH_CHECK_VALUE(g.layout() == at::kStrided, entry, ": gradients must be dense, got layout ", g.layout());
  TORCH_CHECK_VALUE(g.device() == device, entry, ": gradients must be on one device, got ", device, " and ", g.device());
  const ScalarType t = g.scalar_type();
  TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, entry, ": gradients must be bfloat16, float16 or float32, got ", t);
}

// (rows, cols, ld) of a tensor that the kernels walk in place, in row-major
// order; false for other strides.
bool walk(const Tensor& g, int64_t& rows, int64_t& cols, int64_t& ld) {
  if (g.is_contiguous()) {
    rows = 1;
    cols = ld = g.numel();
    return true;
  }
  if (g.dim() == 2 && g.stride(1) == 1 && g.stride(0) >= g.size(1)) {
    rows = g.size(0);
    cols = g.size(1);
    ld = g.stride(0);
    return true;
  }
  return false;
}
bool walks(const Tensor& g) {
  int64_t a, b, c;
  return walk(g, a, b, c);
}

orda_grad_t entry_of(const Tensor& g, const Tensor* dst) {
  orda_grad_t e{};
  walk(g, e.rows, e.cols, e.ld);
  e.data = g.data_ptr();
  e.dtype = e.out_dtype = code(g.scalar_type());
  e.ld_out = e.ld;
  if (dst) {
    int64_t r, c;
    walk(*dst, r, c, e.ld_out);
    if (r != e.rows) {  // a dense side beside a row-strided one: rows both
      e.rows = g.size(0);
      e.cols = g.size(1);
      e.ld = e.rows > 1 ? g.stride(0) : e.cols;
      e.ld_out = e.rows > 1 ? dst->stride(0) : e.cols;
    }
    e.out = dst->data_ptr();
    e.out_dtype = code(dst->scalar_type());
  }
  return e;
}

Tensor norm_of(const std::vector<orda_grad_t>& table, double norm_type, const Tensor& like, void* s) {
  const Tensor total = at::empty({}, like.options().dtype(at::kFloat));
  const size_t n = api.grad_norm_workspace_bytes();
  const Tensor ws = bytes(n, like);
  check(api.grad_norm(table.data(), (int64_t)table.size(), norm_type, static_cast<float*>(total.data_ptr()), out(ws), n, s), "orda_grad_norm");
  return total;
}

Tensor grad_norm(const std::vector<Tensor>& grads, double norm_type) {
  const c10::DeviceGuard guard(grads[0].device());
  std::vector<orda_grad_t> table;
  std::vector<Tensor> alive;
  table.reserve(grads.size());
  for (const Tensor& g : grads) {
    check_grad("grad_norm", g, grads[0].device());
    if (!walks(g)) alive.push_back(g.contiguous());
    table.push_back(entry_of(walks(g) ? g : alive.back(), nullptr));
  }
  return norm_of(table, norm_type, grads[0], stream_of(grads[0]));
}

// The gradients of the parameters (each parameter once) and, with outs, where
// they go; undefined where there is none.
Tensor clip(const std::vector<Tensor>& params, double max_norm, double norm_type, bool raise, const OptTensor& given_total,
            const std::optional<std::vector<Tensor>>& outs) {
  static const char* entry = "clip_grad_norm_";
  std::vector<Tensor> grads, dests;
  std::unordered_map<const void*, size_t> seen;
  grads.reserve(params.size());
  seen.reserve(params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    const Tensor& g = params[i].grad();
    if (!g.defined()) continue;
    const auto [at, fresh] = seen.emplace(params[i].unsafeGetTensorImpl(), i);
    if (!fresh) {
      if (outs) {
        const Tensor &a = (*outs)[at->second], &b = (*outs)[i];
        TORCH_CHECK_VALUE(a.is_same(b) || (a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides() &&
                                           a.scalar_type() == b.scalar_type() && a.device() == b.device()),
                          entry, ": parameters ", at->second, " and ", i, " are one, their out tensors are not");
      }
      continue;
    }
    check_grad(entry, g, grads.empty() ? g.device() : grads[0].device());
    if (outs) {
      const Tensor& o = (*outs)[i];
      const ScalarType t = o.scalar_type();
      TORCH_CHECK_VALUE(o.sizes() == g.sizes() && o.device() == g.device() && o.layout() == at::kStrided &&
                            (t == at::kBFloat16 || t == at::kHalf || t == at::kFloat),
                        entry, ": out[", i, "] must be a bfloat16, float16 or float32 tensor of shape ", g.sizes(), " on ", g.device());
      dests.push_back(o);
    }
    grads.push_back(g);
  }
  if (grads.empty()) return Tensor();
  TORCH_CHECK_VALUE(grads[0].device().is_cuda(), entry, ": gradients must be on a HIP device, got ", grads[0].device());
  const c10::DeviceGuard guard(grads[0].device());
  const at::AutoGradMode off(false);
  void* s = stream_of(grads[0]);
  std::vector<orda_grad_t> table;
  std::vector<std::pair<Tensor, Tensor>> back;  // (dense copy, where it goes afterwards)
  table.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    Tensor g = grads[i], o = outs ? dests[i] : Tensor();
    if (!walks(g)) {  // strides that the kernels do not walk: through a dense copy
      g = g.contiguous();
      if (!outs) back.emplace_back(g, grads[i]);
    }
    if (outs && !walks(o)) {
      o = at::empty(o.sizes(), o.options());
      back.emplace_back(o, dests[i]);
    }
    table.push_back(entry_of(g, outs ? &o : nullptr));
    if (g.unsafeGetTensorImpl() != grads[i].unsafeGetTensorImpl()) grads[i] = g;  // (kept alive)
  }
  Tensor total;
  if (!given_total && !raise) {
    total = at::empty({}, grads[0].options().dtype(at::kFloat));
    const size_t n = api.grad_norm_workspace_bytes();
    const Tensor ws = bytes(n, grads[0]);
    check(api.clip_grad_norm(table.data(), (int64_t)table.size(), norm_type, max_norm, static_cast<float*>(total.data_ptr()), out(ws), n, s),
          "orda_clip_grad_norm");
  } else {
    if (given_total) {
      TORCH_CHECK_VALUE(given_total->numel() == 1 && given_total->device() == grads[0].device(), entry,
                        ": total_norm must be a one-element tensor on ", grads[0].device());
      total = given_total->detach().to(at::kFloat).reshape({});
    } else {
      total = norm_of(table, norm_type, grads[0], s);
    }
    if (raise) {
      TORCH_CHECK(std::isfinite(total.item<float>()), "The total norm of order ", norm_type,
                  " for gradients from `parameters` is non-finite, so it cannot be clipped. To disable this error and scale the "
                  "gradients by the non-finite norm anyway, set `error_if_nonfinite=False`");
    }
    check(api.clip_grads(table.data(), (int64_t)table.size(), static_cast<const float*>(total.const_data_ptr()), max_norm, s), "orda_clip_grads");
  }
  for (auto& [made, want] : back) want.copy_(made);
  for (size_t i = 0; i < params.size(); ++i)
    if (params[i].grad().defined()) {
      const Tensor& t = outs ? (*outs)[i] : params[i].grad();
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
  return total;
}

}  // namespace

PYBIND11_MODULE(orda_torch, m) {
  m.def("bind", &bind);
  m.def("linear", &linear);
  m.def("feed_forward", &feed_forward);
  m.def("grad_norm", &grad_norm);
  m.def("clip", &clip);
}
