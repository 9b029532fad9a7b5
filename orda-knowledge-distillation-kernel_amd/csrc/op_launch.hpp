// op_launch.hpp -- plan and launcher declarations of the projection, the gated
// feed-forward block and the gradient norm, shared between their C entry
// points (ops_abi.hip) and the per-dtype kernel objects (k_op_*.hip).
#pragma once
#include "launch.hpp"
#include "skinny.hpp"
#include "tile16.hpp"

namespace orda {

// orda_last_error()'s message on this thread (abi.hip).
int set_last_error(int code, const char* msg);

enum OpEngine { OP_SKINNY = 0, OP_TILE = 1, OP_RING = 2, OP_SPLIT3 = 3, OP_NONE = -1 };

// How one product runs: the engine, its tile, and K in `splits` ranges of kps.
struct OpPlan {
  int engine;
  int tile;  // OP_TILE: 1000 rows + columns; OP_SPLIT3: 64 (small) or 256 (large)
  int splits;
  int64_t kps;
};

// The product of one launch.  Layouts as GemmParams has them.
template <class T> hipError_t launch_op_linear(const OpPlan& pl, int la, int lb, TileParams P, const EpiLinear<T>& E, float* part, hipStream_t s);
template <class T> hipError_t launch_op_gate(const OpPlan& pl, TileParams P, const EpiGate<T>& E, float* part, hipStream_t s);
template <class T> hipError_t launch_op_gate_grad(const OpPlan& pl, TileParams P, const EpiGateGrad<T>& E, float* part, hipStream_t s);

// dz = dy d (d: the kept act'(z)) into dz ([rows x ldz], columns up to ldz
// written, zeros past cols) and, with partial, its column sums per block of
// rows.
struct DzParams {
  const void* dy;
  Planes d;        // as keep() wrote it, in rows of ldz; null: dz = dy
  void* dz;        // null: only the sums
  float* partial;  // [row blocks][cols], or null
  int64_t rows, cols, ldy, ldz;
  int64_t rows_per_block;
};
template <class T> hipError_t launch_dz(const DzParams& P, hipStream_t s);
// out[c] = sum over b of partial[b][c], in order
template <class T> hipError_t launch_colsum(const float* partial, int64_t blocks, int64_t cols, void* out, hipStream_t s);

// Rows copied and zero-padded, up to kPadMax tensors of one element size.
constexpr int kPadMax = 4;
struct PadParams {
  struct Item {
    const char* src;
    char* dst;
    int64_t rows, cols, ld_src, ld_dst;  // elements
    int64_t first;                       // its first 16-byte piece of dst
  } t[kPadMax];
  int n;
  int64_t pieces;
};
hipError_t launch_pad_rows(const PadParams& P, int esize, hipStream_t s);

// Norm and clipping of many tensors (norms.hip).
struct GradSpan {  // rows x cols elements, ld apart; dense: one row
  void* p;
  void* out;
  int64_t rows, cols, ld, ld_out;
  int in_dtype, out_dtype;
};
constexpr int kNormPartials = 2048;  // fp64 partials of one kernel, added up by the next
hipError_t launch_grad_norm(const GradSpan* g, int64_t n, int kind, double* partials, int max_partials, float* total, hipStream_t s);
hipError_t launch_clip_grad_norm(const GradSpan* g, int64_t n, int kind, double* partials, int max_partials, float* total, float max_norm, hipStream_t s);
hipError_t launch_clip_grads(const GradSpan* g, int64_t n, const float* total, float max_norm, hipStream_t s);

}  // namespace orda
