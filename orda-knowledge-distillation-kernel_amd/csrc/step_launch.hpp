// step_launch.hpp -- launcher declarations of a student's embedding, dropout,
// layer norm and attention, shared between their C entry points (step_abi.hip)
// and the kernels (rownorm.hip, embed.hip, k_attn_*.hip).
#pragma once
#include "launch.hpp"
#include "philox.hpp"

namespace orda {

// orda_last_error()'s message on this thread (abi.hip).
int set_last_error(int code, const char* msg);

// y = residual + keep(x) factor, row by row.
struct DropoutParams {
  const void* x;
  const void* residual;  // or null
  void* y;               // dense
  int64_t rows, cols, ldx, ldr;
  DropParams drop;
};
hipError_t launch_dropout(const DropoutParams& P, int dtype, hipStream_t s);

// s = residual + keep(x) factor; y = (s - mean) rstd w + b.
struct LayerNormParams {
  const void* x;
  const void* residual;  // or null
  const void* weight;
  const void* bias;      // or null
  void* y;
  void* s;               // or null
  float* stats;          // (mean, rstd) of each row, or null
  int64_t rows, cols, ldx, ldr;
  float eps;
  DropParams drop;
};
struct LayerNormGradParams {
  const void* s;
  const void* residual;  // or null; else s holds x, and s = residual + keep(x) factor is computed again
  const float* stats;
  const void* weight;
  const void* dy;
  const void* ds;        // or null
  void* dx;              // or null
  void* dr;              // or null; without dropout dx serves for both
  float* partial;        // [groups][2][cols] sums of dw and db, or null
  int64_t rows, cols, ld_s, ldr, ldy, ldd;
  DropParams drop;
};
// How many workgroups walk the rows of a backward pass (each with sums of dw
// and db of its own).
int64_t layer_norm_groups(int64_t rows, int64_t cols);
hipError_t launch_layer_norm(const LayerNormParams& P, int dtype, int param_dtype, hipStream_t s);
hipError_t launch_layer_norm_grad(const LayerNormGradParams& P, int dtype, int param_dtype, hipStream_t s);
// dw and db (either may be null) from the partial sums
hipError_t launch_layer_norm_params(const float* partial, int64_t groups, int64_t cols, void* dw, void* db, int param_dtype, hipStream_t s);

// y[n] = scale W[t_n]
struct EmbedParams {
  const void* ids;
  const void* weight;
  void* y;
  int64_t tokens, vocab, hidden, ldw;
  float scale;
  int wide;  // ids of 64 bits
};
// dw[v] = scale sum of dy[n] over t_n = v, 0 for v = padding
struct EmbedGradParams {
  const void* ids;
  const void* dy;
  void* dw;  // dense, 16-byte aligned
  int64_t tokens, vocab, hidden, ldg, padding;
  float scale;
  int wide;
};
hipError_t launch_embed(const EmbedParams& P, int dtype, int out_dtype, hipStream_t s);
size_t embed_grad_workspace(int64_t tokens, int64_t hidden);
hipError_t launch_embed_grad(const EmbedGradParams& P, int dtype, int out_dtype, void* workspace, hipStream_t s);

// Masked self-attention (attn.hpp).  Strides in elements; o, dq, dk and dv are
// dense.  Rows of a head are 16-byte aligned, D a multiple of 8 up to 128.
struct AttnParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  void* o_low;  // what o's rounding left, or null (no backward pass)
  const void* dout;
  void* dq;
  void* dk;  // or null
  void* dv;  // or null
  float* lse;    // [B][H][padded], or null (no backward pass)
  float* delta;  // the same
  const float* slopes;    // [H], or null
  const int32_t* prefix;  // [B], or null
  const int* docs;        // [B][padded], or null
  const int4* ranges;     // [B][padded / 32]
  int64_t S, padded;      // padded: S up to a multiple of 128
  int64_t qb, qs, qh, kb, ks, kh, vb, vs, vh, gb, gs, gh;
  float* partial;         // dk and dv of each part, [2][parts][B S KV D], or null (one part)
  int B, H, KV, group, D, causal, tiles;
  int cap;                  // AttnCap
  int fine;                 // dz goes into its products in two halves
  int parts, share;         // workgroups that take the heads of a tile of keys, heads of each
  float scale, scale_log2;  // scale_log2 = |scale| log2(e)
  float slope_mul;          // 1 / |scale|, with a cap log2(e)
  float slope_low, slope_high;  // what it is then taken for at least and at most
  float cap_in, cap_out;    // 2 |scale| log2(e) / cap and cap log2(e)
};
enum AttnCap { CAP_NONE, CAP_SMALL, CAP_ANY };  // (attn.hpp: scores)
enum AttnPass { ATTN_FORWARD, ATTN_DQ, ATTN_DKV };
template <class T, int HD> hipError_t launch_attn(const AttnParams& P, AttnPass pass, hipStream_t s);
hipError_t launch_attn_join(const AttnParams& P, int dtype, hipStream_t s);
hipError_t launch_attn_docs(const int32_t* ids, int64_t ld, int64_t B, int64_t S, int64_t padded, int* docs, int4* ranges, hipStream_t s);

}  // namespace orda
