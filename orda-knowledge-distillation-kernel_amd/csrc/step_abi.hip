// step_abi.hip -- the C entry points of the token embedding, dropout, the layer
// norm and the masked self-attention: argument checks and launch sequences.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/orda_ce.h"
#include "step_launch.hpp"

using namespace orda;

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_last_error(code, buf);
}
#define STEP_TRY(expr)                   \
  do {                                   \
    const int rc_ = (expr);              \
    if (rc_ != ORDA_OK) return rc_;      \
  } while (0)
#define STEP_LAUNCH(expr)                                                                     \
  do {                                                                                        \
    const hipError_t e_ = (expr);                                                             \
    if (e_ != hipSuccess) return fail(ORDA_ELAUNCH, "%s: %s", #expr, hipGetErrorString(e_));  \
  } while (0)

inline int64_t esize(int dtype) { return dtype == ORDA_F32 ? 4 : 2; }
inline bool on(const void* q, int64_t bytes) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; }
inline char* base256(const void* ws) { return reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(ws) + 255) / 256 * 256); }
inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }
inline hipStream_t stream_of(void* s) { return static_cast<hipStream_t>(s); }

constexpr int64_t kMaxTokens = 1ll << 30, kMaxWidth = 1ll << 21, kMaxPitch = 1ll << 22;

int check_dtype(const char* what, const char* name, int32_t dtype) {
  if (dtype < ORDA_BF16 || dtype > ORDA_F32) return fail(ORDA_EINVAL, "%s: unknown %s %d", what, name, dtype);
  return ORDA_OK;
}
int check_version(const char* what, int32_t version) {
  if (version != ORDA_ABI_VERSION) return fail(ORDA_EINVAL, "%s: abi_version %d, library has %d", what, version, ORDA_ABI_VERSION);
  return ORDA_OK;
}
int check_pitch(const char* what, const char* name, int64_t ld, int64_t rows, int64_t cols) {
  if (rows > 1 && (ld < cols || ld > kMaxPitch)) return fail(ORDA_EINVAL, "%s: %s must be in [%lld, 2^22], got %lld", what, name, (long long)cols, (long long)ld);
  return ORDA_OK;
}
int check_size(const char* what, const char* name, int64_t n, int64_t most) {
  if (n < 1 || n > most) return fail(ORDA_EINVAL, "%s: %s must be in [1, %lld], got %lld", what, name, (long long)most, (long long)n);
  return ORDA_OK;
}
int check_tensor(const char* what, const char* name, const void* t, int64_t bytes, bool required = true) {
  if (!t) return required ? fail(ORDA_EINVAL, "%s: %s is required", what, name) : ORDA_OK;
  if (!on(t, bytes)) return fail(ORDA_EINVAL, "%s: %s must be aligned to %lld bytes", what, name, (long long)bytes);
  return ORDA_OK;
}
int check_workspace(const char* what, const char* name, const void* ws, size_t given, size_t needed) {
  if (!ws || given < needed) return fail(ORDA_EWORKSPACE, "%s: %s has %zu bytes, needs %zu", what, name, ws ? given : (size_t)0, needed);
  return ORDA_OK;
}

int drop_params(const char* what, const orda_dropout_t* d, DropParams& out) {
  out = DropParams{0, nullptr, 0, 0, 1.0f};
  if (!d) return ORDA_OK;
  if (!(d->p >= 0.0 && d->p <= 1.0)) return fail(ORDA_EINVAL, "%s: p must be in [0, 1], got %g", what, d->p);
  if (!on(d->seed_on_device, 8)) return fail(ORDA_EINVAL, "%s: seed_on_device must be aligned to 8 bytes", what);
  out.seed = d->seed;
  out.seed_ptr = d->seed_on_device;
  out.site = d->site;
  out.threshold = (uint32_t)std::floor(d->p * 65536.0 + 0.5);
  out.factor = out.threshold < 65536 ? (float)(65536.0 / (65536.0 - out.threshold)) : 0.0f;
  return ORDA_OK;
}

int check_embedding(const char* what, const orda_embedding_t* p) {
  if (!p) return fail(ORDA_EINVAL, "%s: the problem is NULL", what);
  STEP_TRY(check_version(what, p->abi_version));
  STEP_TRY(check_dtype(what, "dtype", p->dtype));
  STEP_TRY(check_dtype(what, "out_dtype", p->out_dtype));
  if (p->reserved != 0) return fail(ORDA_EINVAL, "%s: reserved must be 0", what);
  STEP_TRY(check_size(what, "tokens", p->tokens, kMaxTokens));
  STEP_TRY(check_size(what, "vocab", p->vocab, 0x7ffffffell));
  STEP_TRY(check_size(what, "hidden", p->hidden, kMaxWidth));
  if (!std::isfinite(p->scale)) return fail(ORDA_EINVAL, "%s: scale must be finite, got %g", what, p->scale);
  return ORDA_OK;
}
size_t embedding_bytes(const orda_embedding_t* p) { return embed_grad_workspace(p->tokens, p->hidden) + 256; }

int check_layer_norm(const char* what, const orda_layer_norm_t* p) {
  if (!p) return fail(ORDA_EINVAL, "%s: the problem is NULL", what);
  STEP_TRY(check_version(what, p->abi_version));
  STEP_TRY(check_dtype(what, "dtype", p->dtype));
  if (p->param_dtype != p->dtype && p->param_dtype != ORDA_F32)
    return fail(ORDA_EINVAL, "%s: param_dtype must be dtype or fp32, got %d", what, p->param_dtype);
  STEP_TRY(check_size(what, "rows", p->rows, kMaxTokens));
  STEP_TRY(check_size(what, "cols", p->cols, kMaxWidth));
  if (!(p->eps >= 0.0f) || !std::isfinite(p->eps)) return fail(ORDA_EINVAL, "%s: eps must be finite and >= 0, got %g", what, p->eps);
  return ORDA_OK;
}
size_t layer_norm_bytes(const orda_layer_norm_t* p) { return (size_t)layer_norm_groups(p->rows, p->cols) * 2 * p->cols * 4 + 256; }

int64_t padded_length(const orda_attention_t* p) { return (p->length + 127) / 128 * 128; }
int check_strides(const char* what, const char* name, const int64_t (&s)[3], const orda_attention_t* p, int64_t heads) {
  const int64_t n[3] = {p->batch, p->length, heads};
  for (int i = 0; i < 3; ++i) {
    if (n[i] == 1) continue;
    if (s[i] < 0 || s[i] % 8 != 0) return fail(ORDA_EINVAL, "%s: strides of %s must be multiples of 8, got %lld", what, name, (long long)s[i]);
    if (i == 1 && s[i] > kMaxPitch) return fail(ORDA_EINVAL, "%s: rows of %s are more than 2^22 elements apart (%lld)", what, name, (long long)s[i]);
  }
  return ORDA_OK;
}
int check_attention(const char* what, const orda_attention_t* p) {
  if (!p) return fail(ORDA_EINVAL, "%s: the problem is NULL", what);
  STEP_TRY(check_version(what, p->abi_version));
  if (p->dtype != ORDA_BF16 && p->dtype != ORDA_F16) return fail(ORDA_EINVAL, "%s: dtype must be bf16 or fp16, got %d", what, p->dtype);
  STEP_TRY(check_size(what, "length", p->length, 1ll << 24));
  STEP_TRY(check_size(what, "batch", p->batch, 65535));  // (a grid's second dimension)
  STEP_TRY(check_size(what, "heads", p->heads, 1 << 16));
  STEP_TRY(check_size(what, "kv_heads", p->kv_heads, p->heads));
  if (p->heads % p->kv_heads != 0) return fail(ORDA_EINVAL, "%s: heads (%d) must be a multiple of kv_heads (%d)", what, p->heads, p->kv_heads);
  if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8 != 0)
    return fail(ORDA_EINVAL, "%s: head_dim must be a multiple of 8 in [8, 128], got %d", what, p->head_dim);
  if (p->causal != 0 && p->causal != 1) return fail(ORDA_EINVAL, "%s: causal must be 0 or 1, got %d", what, p->causal);
  if (!(std::fabs(p->scale) <= 1e38)) return fail(ORDA_EINVAL, "%s: scale must be finite in fp32, up to 1e38, got %g", what, p->scale);
  if (!(p->softcap >= 0.0) || !std::isfinite(p->softcap)) return fail(ORDA_EINVAL, "%s: softcap must be finite and >= 0, got %g", what, p->softcap);
  // (a launch has fewer than 2^32 threads, a tile 256 of them, of dk and dv 512)
  if (padded_length(p) / 128 * p->batch * std::max(p->heads, 2 * p->kv_heads) >= (1ll << 24))
    return fail(ORDA_EINVAL, "%s: %lld x %lld x %d rows are more tiles than a launch has workgroups", what, (long long)p->batch, (long long)p->length, p->heads);
  STEP_TRY(check_strides(what, "q", p->q_stride, p, p->heads));
  STEP_TRY(check_strides(what, "k", p->k_stride, p, p->kv_heads));
  return check_strides(what, "v", p->v_stride, p, p->kv_heads);
}

// The pieces of `saved`: ranges of document numbers, the numbers, L, what the
// rounding of the output left.
struct Kept {
  size_t docs, lse, low, bytes;
};
Kept kept_of(const orda_attention_t* p, bool documents, bool training) {
  const size_t L = (size_t)padded_length(p);
  Kept k{};
  k.docs = documents ? up256((size_t)p->batch * (L / 32) * sizeof(int4)) : 0;
  k.lse = k.docs + (documents ? up256((size_t)p->batch * L * 4) : 0);
  k.low = k.lse + (training ? up256((size_t)p->batch * p->heads * L * 4) : 0);
  k.bytes = k.low + (training ? (size_t)p->batch * p->length * p->heads * p->head_dim * 2 : 0) + 256;
  return k;
}
// Parts that the heads of a tile of 128 keys are taken in, each by a workgroup of
// its own: as many as bring two workgroups to a CU.  One whose keys' heads are one
// after the other takes long on a card that these do not fill (3 x 1777 rows, 12
// heads of 80, 4 of keys, documents: 111 us, by parts of one head 74 and 9 to add
// them up).
struct Parts {
  int count, share;
};
Parts parts_of(const orda_attention_t* p) {
  const int64_t full = 512, tiles = padded_length(p) / 128 * p->batch * p->kv_heads;
  const int group = p->heads / p->kv_heads, want = (int)std::min<int64_t>(group, (full + tiles - 1) / tiles);
  const int share = (group + want - 1) / want;
  return {(group + share - 1) / share, share};
}
// delta of the queries, dk and dv of the parts
size_t delta_bytes(const orda_attention_t* p) { return up256((size_t)p->batch * p->heads * padded_length(p) * 4); }
size_t attention_bytes(const orda_attention_t* p) {
  const int parts = parts_of(p).count;
  return delta_bytes(p) + (parts > 1 ? (size_t)2 * parts * p->batch * p->length * p->kv_heads * p->head_dim * 4 : 0) + 256;
}

// Caps up to which the shorter tanh serves (attn.hpp, scores: its error grows with
// the cap; 2e-5 here, the other's time is 1.4 to 1.7 times as long).
constexpr double kSmallCap = 128.0;

AttnParams attn_params(const orda_attention_t* p, const void* q, const void* k, const void* v, const float* slopes, const int32_t* prefix) {
  AttnParams a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.slopes = slopes;
  a.prefix = prefix;
  a.S = p->length;
  a.padded = padded_length(p);
  const int64_t n[3] = {p->batch, p->length, p->heads}, kv[3] = {p->batch, p->length, p->kv_heads};
  // (the stride of a dimension of one element says nothing)
  auto set = [](const int64_t (&s)[3], const int64_t (&size)[3], int64_t& b, int64_t& r, int64_t& h) {
    b = size[0] == 1 ? 0 : s[0];
    r = size[1] == 1 ? 0 : s[1];
    h = size[2] == 1 ? 0 : s[2];
  };
  set(p->q_stride, n, a.qb, a.qs, a.qh);
  set(p->k_stride, kv, a.kb, a.ks, a.kh);
  set(p->v_stride, kv, a.vb, a.vs, a.vh);
  set(p->g_stride, n, a.gb, a.gs, a.gh);
  a.B = (int)p->batch;
  a.H = p->heads;
  a.KV = p->kv_heads;
  a.group = p->heads / p->kv_heads;
  // dz rounded to 16 bits as an operand leaves dq and dk in bf16 off by 2.4e-3 of their
  // norm at any length (1.7e-3 are their own rounding), in two halves by 1.7e-3 to
  // 1.8e-3.  The second halves' products cost 0.3 us of 6 to 9 while a call is one
  // tile of keys, from there on 3 to 15 % of either kernel (16 x 256 rows, 8 heads of
  // 64 and of 128), up to 19 to 28 % of dq and 12 to 21 % of dk and dv (8 heads of 128,
  // 4096 rows: 106 -> 136 and 135 -> 155 us).  Documents packed into longer rows have
  // the one operand, however short they are.
  a.fine = p->length <= 64;
  a.parts = parts_of(p).count;
  a.share = parts_of(p).share;
  a.D = p->head_dim;
  a.causal = p->causal;
  const double log2e = 1.4426950408889634;
  // (magnitudes: the kernels turn the sign of one operand; a scale of 0 is 1e-24,
  // so that the -inf of what is not seen stays one)
  const double size = std::fmax(std::fabs(p->scale), 1e-24);
  a.scale = (float)p->scale;
  a.scale_log2 = (float)(size * log2e);
  a.slope_mul = (float)(p->softcap > 0.0 ? log2e : 1.0 / size);
  const double far = p->length * (p->softcap > 0.0 ? 1.0 : size * log2e);
  a.slope_low = (float)std::fmax(-0x1p22 / far, -1e30);
  a.slope_high = (float)std::fmin(0x1p30 / far, 1e30);
  a.cap = CAP_NONE;
  if (p->softcap > 0.0) {
    // (a cap below 1e-24 leaves scores of 0 and one past 1e30 the scores as they are, in fp32)
    const double cap = std::fmin(std::fmax(p->softcap, 1e-24), 1e30);
    a.cap = cap <= kSmallCap ? CAP_SMALL : CAP_ANY;
    a.cap_in = (float)std::fmin(2.0 * log2e * size / cap, 3e38);
    a.cap_out = (float)(cap * log2e);
  }
  return a;
}
// The columns that go through the products, in steps of 32 from 64 on (heads of 80
// in the 128 columns: forward 47.0 us instead of 44.5, dq 54 instead of 51, for 3 x
// 1777 rows of 12 heads in documents).
template <class T>
hipError_t attn(const AttnParams& a, AttnPass pass, hipStream_t s) {
  return a.D <= 64 ? launch_attn<T, 64>(a, pass, s) : a.D <= 96 ? launch_attn<T, 96>(a, pass, s) : launch_attn<T, 128>(a, pass, s);
}
hipError_t attn(const AttnParams& a, int32_t dtype, AttnPass pass, hipStream_t s) {
  return dtype == ORDA_BF16 ? attn<bf16>(a, pass, s) : attn<f16>(a, pass, s);
}

}  // namespace

extern "C" {

int orda_embedding_forward(const orda_embedding_t* p, const void* ids, const void* weight, void* y, void* stream) {
  static const char* what = "orda_embedding_forward";
  set_last_error(0, nullptr);
  STEP_TRY(check_embedding(what, p));
  STEP_TRY(check_pitch(what, "ldw", p->ldw, p->vocab, p->hidden));
  STEP_TRY(check_tensor(what, "ids", ids, p->wide_ids ? 8 : 4));
  STEP_TRY(check_tensor(what, "weight", weight, esize(p->dtype)));
  STEP_TRY(check_tensor(what, "y", y, esize(p->out_dtype)));
  const EmbedParams e{ids, weight, y, p->tokens, p->vocab, p->hidden, p->ldw, p->scale, p->wide_ids != 0};
  STEP_LAUNCH(launch_embed(e, p->dtype, p->out_dtype, stream_of(stream)));
  return ORDA_OK;
}

size_t orda_embedding_workspace_bytes(const orda_embedding_t* p) {
  set_last_error(0, nullptr);
  return check_embedding("orda_embedding_workspace_bytes", p) == ORDA_OK ? embedding_bytes(p) : 0;
}

int orda_embedding_backward(const orda_embedding_t* p, const void* ids, const void* grad_output, void* grad_weight, void* workspace,
                            size_t workspace_bytes, void* stream) {
  static const char* what = "orda_embedding_backward";
  set_last_error(0, nullptr);
  STEP_TRY(check_embedding(what, p));
  STEP_TRY(check_pitch(what, "ldg", p->ldg, p->tokens, p->hidden));
  STEP_TRY(check_tensor(what, "ids", ids, p->wide_ids ? 8 : 4));
  STEP_TRY(check_tensor(what, "grad_output", grad_output, esize(p->out_dtype)));
  STEP_TRY(check_tensor(what, "grad_weight", grad_weight, 16));
  STEP_TRY(check_workspace(what, "the workspace", workspace, workspace_bytes, embedding_bytes(p)));
  const EmbedGradParams e{ids, grad_output, grad_weight, p->tokens, p->vocab, p->hidden, p->ldg, p->padding_idx, p->scale, p->wide_ids != 0};
  STEP_LAUNCH(launch_embed_grad(e, p->dtype, p->out_dtype, base256(workspace), stream_of(stream)));
  return ORDA_OK;
}

int orda_dropout_add(const orda_rows_problem_t* p, const orda_dropout_t* d, const void* x, const void* residual, void* y, void* stream) {
  static const char* what = "orda_dropout_add";
  set_last_error(0, nullptr);
  if (!p || !d) return fail(ORDA_EINVAL, "%s: the problem is NULL", what);
  STEP_TRY(check_version(what, p->abi_version));
  STEP_TRY(check_dtype(what, "dtype", p->dtype));
  STEP_TRY(check_size(what, "rows", p->rows, kMaxTokens));
  STEP_TRY(check_size(what, "cols", p->cols, 1ll << 40));
  if (p->cols > (1ll << 42) / p->rows) return fail(ORDA_EINVAL, "%s: %lld x %lld are more than 2^42 elements", what, (long long)p->rows, (long long)p->cols);
  STEP_TRY(check_pitch(what, "ldx", p->ldx, p->rows, p->cols));
  if (residual) STEP_TRY(check_pitch(what, "ldr", p->ldr, p->rows, p->cols));
  STEP_TRY(check_tensor(what, "x", x, esize(p->dtype)));
  STEP_TRY(check_tensor(what, "residual", residual, esize(p->dtype), false));
  STEP_TRY(check_tensor(what, "y", y, esize(p->dtype)));
  DropoutParams e{x, residual, y, p->rows, p->cols, p->ldx, p->ldr, {}};
  STEP_TRY(drop_params(what, d, e.drop));
  STEP_LAUNCH(launch_dropout(e, p->dtype, stream_of(stream)));
  return ORDA_OK;
}

int orda_layer_norm_forward(const orda_layer_norm_t* p, const orda_dropout_t* d, const void* x, const void* residual, const void* weight,
                            const void* bias, void* y, void* s, float* stats, void* stream) {
  static const char* what = "orda_layer_norm_forward";
  set_last_error(0, nullptr);
  STEP_TRY(check_layer_norm(what, p));
  const int64_t es = esize(p->dtype), ps = esize(p->param_dtype);
  STEP_TRY(check_pitch(what, "ldx", p->ldx, p->rows, p->cols));
  if (residual) STEP_TRY(check_pitch(what, "ldr", p->ldr, p->rows, p->cols));
  STEP_TRY(check_tensor(what, "x", x, es));
  STEP_TRY(check_tensor(what, "residual", residual, es, false));
  STEP_TRY(check_tensor(what, "weight", weight, ps));
  STEP_TRY(check_tensor(what, "bias", bias, ps, false));
  STEP_TRY(check_tensor(what, "y", y, es));
  STEP_TRY(check_tensor(what, "s", s, es, false));
  STEP_TRY(check_tensor(what, "stats", stats, 8, false));
  LayerNormParams e{x, residual, weight, bias, y, s, stats, p->rows, p->cols, p->ldx, p->ldr, p->eps, {}};
  STEP_TRY(drop_params(what, d, e.drop));
  STEP_LAUNCH(launch_layer_norm(e, p->dtype, p->param_dtype, stream_of(stream)));
  return ORDA_OK;
}

size_t orda_layer_norm_workspace_bytes(const orda_layer_norm_t* p) {
  set_last_error(0, nullptr);
  return check_layer_norm("orda_layer_norm_workspace_bytes", p) == ORDA_OK ? layer_norm_bytes(p) : 0;
}

int orda_layer_norm_backward(const orda_layer_norm_t* p, const orda_dropout_t* d, const void* s, const void* residual, const float* stats,
                             const void* weight, const void* grad_y, const void* grad_s, void* grad_x, void* grad_residual, void* grad_weight, void* grad_bias,
                             void* workspace, size_t workspace_bytes, void* stream) {
  static const char* what = "orda_layer_norm_backward";
  set_last_error(0, nullptr);
  STEP_TRY(check_layer_norm(what, p));
  const int64_t es = esize(p->dtype), ps = esize(p->param_dtype);
  STEP_TRY(check_pitch(what, "ld_s", p->ld_s, p->rows, p->cols));
  STEP_TRY(check_pitch(what, "ld_dy", p->ld_dy, p->rows, p->cols));
  if (grad_s) STEP_TRY(check_pitch(what, "ld_ds", p->ld_ds, p->rows, p->cols));
  STEP_TRY(check_tensor(what, "s", s, es));
  STEP_TRY(check_tensor(what, "residual", residual, es, false));
  if (residual) {
    if (p->param_dtype == p->dtype) return fail(ORDA_EINVAL, "%s: s is computed again only for fp32 parameters beside 16-bit tensors", what);
    STEP_TRY(check_pitch(what, "ldr", p->ldr, p->rows, p->cols));
  }
  STEP_TRY(check_tensor(what, "stats", stats, 8));
  STEP_TRY(check_tensor(what, "weight", weight, ps));
  STEP_TRY(check_tensor(what, "grad_y", grad_y, es));
  STEP_TRY(check_tensor(what, "grad_s", grad_s, es, false));
  STEP_TRY(check_tensor(what, "grad_x", grad_x, es, false));
  STEP_TRY(check_tensor(what, "grad_residual", grad_residual, es, false));
  STEP_TRY(check_tensor(what, "grad_weight", grad_weight, ps, false));
  STEP_TRY(check_tensor(what, "grad_bias", grad_bias, ps, false));
  const bool params = grad_weight || grad_bias;
  if (params) STEP_TRY(check_workspace(what, "the workspace", workspace, workspace_bytes, layer_norm_bytes(p)));
  float* partial = params ? reinterpret_cast<float*>(base256(workspace)) : nullptr;
  LayerNormGradParams e{s, residual, stats, weight, grad_y, grad_s, grad_x, grad_residual, partial, p->rows, p->cols, p->ld_s, p->ldr, p->ld_dy, p->ld_ds, {}};
  STEP_TRY(drop_params(what, d, e.drop));
  if (e.drop.threshold == 0 && grad_x && grad_residual) return fail(ORDA_EINVAL, "%s: without dropout grad_x and grad_residual are one", what);
  STEP_LAUNCH(launch_layer_norm_grad(e, p->dtype, p->param_dtype, stream_of(stream)));
  if (params)
    STEP_LAUNCH(launch_layer_norm_params(partial, layer_norm_groups(p->rows, p->cols), p->cols, grad_weight, grad_bias, p->param_dtype, stream_of(stream)));
  return ORDA_OK;
}

size_t orda_attention_saved_bytes(const orda_attention_t* p, int32_t with_documents, int32_t training) {
  set_last_error(0, nullptr);
  return check_attention("orda_attention_saved_bytes", p) == ORDA_OK ? kept_of(p, with_documents != 0, training != 0).bytes : 0;
}

int orda_attention_forward(const orda_attention_t* p, const void* q, const void* k, const void* v, const float* slopes, const int32_t* documents,
                           const int32_t* prefix, void* out, void* saved, size_t saved_bytes, int32_t training, void* stream) {
  static const char* what = "orda_attention_forward";
  set_last_error(0, nullptr);
  STEP_TRY(check_attention(what, p));
  STEP_TRY(check_tensor(what, "q", q, 16));
  STEP_TRY(check_tensor(what, "k", k, 16));
  STEP_TRY(check_tensor(what, "v", v, 16));
  STEP_TRY(check_tensor(what, "slopes", slopes, 4, false));
  STEP_TRY(check_tensor(what, "documents", documents, 4, false));
  STEP_TRY(check_tensor(what, "prefix", prefix, 4, false));
  STEP_TRY(check_tensor(what, "out", out, 16));
  if (documents && p->batch > 1 && p->documents_stride < p->length)
    return fail(ORDA_EINVAL, "%s: documents_stride must be at least the length, got %lld", what, (long long)p->documents_stride);
  const Kept kept = kept_of(p, documents != nullptr, training != 0);
  if (documents || training) {
    STEP_TRY(check_workspace(what, "saved", saved, saved_bytes, kept.bytes));
    STEP_TRY(check_tensor(what, "saved", saved, 16));
  }
  char* base = static_cast<char*>(saved);
  AttnParams a = attn_params(p, q, k, v, slopes, prefix);
  a.o = out;
  if (training) {
    a.lse = reinterpret_cast<float*>(base + kept.lse);
    a.o_low = base + kept.low;
  }
  if (documents) {
    int* docs = reinterpret_cast<int*>(base + kept.docs);
    int4* ranges = reinterpret_cast<int4*>(base);
    STEP_LAUNCH(launch_attn_docs(documents, p->documents_stride, p->batch, p->length, a.padded, docs, ranges, stream_of(stream)));
    a.docs = docs;
    a.ranges = ranges;
  }
  STEP_LAUNCH(attn(a, p->dtype, ATTN_FORWARD, stream_of(stream)));
  return ORDA_OK;
}

size_t orda_attention_workspace_bytes(const orda_attention_t* p) {
  set_last_error(0, nullptr);
  return check_attention("orda_attention_workspace_bytes", p) == ORDA_OK ? attention_bytes(p) : 0;
}

int orda_attention_backward(const orda_attention_t* p, const void* q, const void* k, const void* v, const float* slopes, int32_t with_documents,
                            const int32_t* prefix, const void* out, const void* saved, size_t saved_bytes, const void* grad_output, void* grad_q,
                            void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes, void* stream) {
  static const char* what = "orda_attention_backward";
  set_last_error(0, nullptr);
  STEP_TRY(check_attention(what, p));
  STEP_TRY(check_strides(what, "grad_output", p->g_stride, p, p->heads));
  STEP_TRY(check_tensor(what, "q", q, 16));
  STEP_TRY(check_tensor(what, "k", k, 16));
  STEP_TRY(check_tensor(what, "v", v, 16));
  STEP_TRY(check_tensor(what, "out", out, 16));
  STEP_TRY(check_tensor(what, "grad_output", grad_output, 16));
  STEP_TRY(check_tensor(what, "slopes", slopes, 4, false));
  STEP_TRY(check_tensor(what, "prefix", prefix, 4, false));
  STEP_TRY(check_tensor(what, "grad_q", grad_q, 16, false));
  STEP_TRY(check_tensor(what, "grad_k", grad_k, 16, false));
  STEP_TRY(check_tensor(what, "grad_v", grad_v, 16, false));
  const Kept kept = kept_of(p, with_documents != 0, true);
  STEP_TRY(check_workspace(what, "saved", saved, saved_bytes, kept.bytes));
  STEP_TRY(check_tensor(what, "saved", saved, 16));
  STEP_TRY(check_workspace(what, "the workspace", workspace, workspace_bytes, attention_bytes(p)));
  char* base = static_cast<char*>(const_cast<void*>(saved));
  AttnParams a = attn_params(p, q, k, v, slopes, prefix);
  a.o = const_cast<void*>(out);
  a.dout = grad_output;
  a.dq = grad_q;
  a.dk = grad_k;
  a.dv = grad_v;
  a.lse = reinterpret_cast<float*>(base + kept.lse);
  a.o_low = base + kept.low;
  a.delta = reinterpret_cast<float*>(base256(workspace));
  if (a.parts > 1) a.partial = reinterpret_cast<float*>(static_cast<char*>(base256(workspace)) + delta_bytes(p));
  if (with_documents) {
    a.docs = reinterpret_cast<const int*>(base + kept.docs);
    a.ranges = reinterpret_cast<const int4*>(base);
  }
  STEP_LAUNCH(attn(a, p->dtype, ATTN_DQ, stream_of(stream)));  // (delta too)
  if (grad_k || grad_v) STEP_LAUNCH(attn(a, p->dtype, ATTN_DKV, stream_of(stream)));
  if ((grad_k || grad_v) && a.parts > 1) STEP_LAUNCH(launch_attn_join(a, p->dtype, stream_of(stream)));
  return ORDA_OK;
}

}  // extern "C"
