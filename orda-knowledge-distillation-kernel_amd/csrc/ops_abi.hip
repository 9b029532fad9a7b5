// ops_abi.hip -- the C entry points of the projection (orda_linear_*), the
// gated feed-forward block (orda_ffn_*) and the gradient norm: argument
// checks, the choice of engine, and the launch sequences.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <vector>

#include "../../include/orda_ce.h"
#include "op_launch.hpp"

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
#define OP_LAUNCH(expr)                                                                       \
  do {                                                                                        \
    const hipError_t e_ = (expr);                                                             \
    if (e_ != hipSuccess) return fail(ORDA_ELAUNCH, "%s: %s", #expr, hipGetErrorString(e_));  \
  } while (0)

inline int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t esize(int dtype) { return dtype == ORDA_F32 ? 4 : 2; }
inline int64_t kept_bytes(int dtype) { return dtype == ORDA_F32 ? kKeptBytes<float> : kKeptBytes<bf16>; }
inline int64_t granule(int dtype) { return dtype == ORDA_F32 ? 4 : 8; }  // elements of 16 bytes
inline bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }
inline char* base256(void* ws) { return reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(ws) + 255) / 256 * 256); }

constexpr int64_t kMaxTokens = 1ll << 30;
// A launch has fewer than 2^32 threads, a tile 256 of them: 2^30 tokens on 64
// columns are 2^24 tiles of 64 rows, one too many, and half as many of 128.
constexpr double kMaxItems = 16777216.0;
// (128 rows of a K-major operand in one buffer resource, 256 rows of an output
// within 2^32 bytes)
constexpr int64_t kMaxWidth = 1ll << 21, kMaxPitch = 1ll << 22;

// ------------------------------------------------------------- the engine
// One product C[M x cols] = A B^T over K; dual: two weights.
struct Shape {
  int dtype, la, lb;
  bool dual;
  int64_t M, cols, K;
  int64_t lda, ldb;   // pitches of MN-major operands
  bool pair;          // two products side by side (A's columns)
};

// Splits without which a split's MN-major K rows would pass 2^30 bytes: the
// offset of a step and the one that marks a chunk as out of range (2^31) add up
// in 32 bits.
int64_t splits_needed(const Shape& q) {
  const int64_t row = std::max<int64_t>(q.la == MNMAJ ? q.lda : 0, q.lb == MNMAJ ? q.ldb : 0) * 2;
  const int64_t rows = std::max<int64_t>(64, row ? (0x3fffffffll / row) / 64 * 64 : up(q.K, 64));
  return cdiv(q.K, rows);
}

// Estimated microseconds of a 16-bit product, from a sweep of 18 shapes (20 x
// 1024 x 1024 to 8192 x 4096 x 2048) in the three layouts over tiles and
// splits.  A K step of 64 takes the CU `step` per workgroup on it, and at least
// `alone`; the ring engine 1.45 us per step of its 256 x 256 tiles (one
// workgroup per CU) and 8 per tile for the epilogue.  Partials go out and back
// at 8 TB/s (they stay in the caches), their sum is one more launch.
//   1024^3: 64 x 64 8.2 us (model 8.1), 64 x 128 10.2, 128 x 128 14.5
//   2048 x 4096 x 1024: 128 x 128 23.6 us (22), 64 x 64 30.8 (27), ring 37 (39)
//   8192 x 4096 x 2048: ring 118 us (116), 128 x 128 135 (132)
//   512 x 1024 x 2736: 64 x 64 in 2 ranges 13.1 us (13.9), in one 14.9 (15.7)
struct TileCost {
  int bm, bn;
  double fixed, step, alone;
};
constexpr TileCost kTileCosts[] = {{64, 64, 3.8, 0.19, 0.27}, {64, 128, 4.8, 0.33, 0.33}, {128, 128, 6.0, 0.49, 0.58}};
constexpr double kCus = 256.0;

int64_t products(const Shape& q) { return q.pair ? 2 : 1; }
double split_cost(const Shape& q, int64_t sp) {
  return sp == 1 ? 0.0 : 3.0 + (double)sp * q.M * products(q) * q.cols * (q.dual ? 2 : 1) * 8.0 / 8e6;
}
// Tiles of bm x bn (dual: half of them of each weight) times splits.
double items_of(const Shape& q, int64_t bm, int64_t bn, int64_t sp) {
  return (double)(cdiv(q.M, bm) * products(q) * cdiv(q.cols, q.dual ? bn / 2 : bn) * sp);
}
double tile_cost(const Shape& q, const TileCost& t, int64_t sp) {
  const double per_cu = std::ceil(items_of(q, t.bm, t.bn, sp) / kCus), steps = (double)cdiv(cdiv(q.K, sp), 64);
  return t.fixed + steps * (per_cu <= 1 ? std::max(t.alone, t.step) : per_cu * t.step) + split_cost(q, sp);
}
double ring_cost(const Shape& q, int64_t sp) {
  const double rounds = std::ceil(items_of(q, 256, 256, sp) / kCus);
  return 8.0 + rounds * ((double)cdiv(cdiv(q.K, sp), 64) * 1.45 + 8.0) + split_cost(q, sp);
}
// The ring engine takes more than one K step, and of a K-major operand whole
// K ranges only.
bool ring_fits(const Shape& q, int64_t sp) {
  if (q.K <= 64 * sp || sp < splits_needed(q)) return false;
  return sp == 1 || q.la == MNMAJ || q.K % (64 * sp) == 0;
}
// fp32, K steps of 32 on the split-operand engine: 1.9 to 2.4 us per step of a
// 256 x 128 tile (one to a CU; the clock falls with the load) and 8 per tile; 64 x 64 tiles, up to three to a CU, by
// how many there are and whether an operand is MN-major (a sweep of 13 shapes;
// 2048^3 in 2 ranges 92 us, model 96; 1000 x 2668 x 777 in 3 ranges of large
// tiles 41 us, 44; 300 x 300 x 4096 in 16 of small ones 17.6 us, 17.6).
double s3_op_cost(const Shape& q, int64_t sp, bool large) {
  const double steps = (double)cdiv(cdiv(q.K, sp), 32), part = split_cost(q, sp);
  if (large) {
    const double fill = items_of(q, 256, 128, sp) / kCus;
    return std::ceil(fill) * (steps * (1.9 + 0.5 * std::min(1.0, fill)) + 8.0) + part;
  }
  const double items = items_of(q, 64, 64, sp), rounds = std::ceil(items / (3 * kCus));
  constexpr double kStep[2][3] = {{0.75, 1.0, 1.45}, {1.15, 1.55, 2.0}};
  const int load = rounds > 1 ? 2 : (int)std::ceil(items / kCus) - 1;
  return 5.0 + rounds * steps * kStep[q.la == MNMAJ || q.lb == MNMAJ][load] + part;
}

OpPlan plan_of(const Shape& q) {
  OpPlan pl{};
  pl.engine = OP_NONE;
  pl.splits = 1;
  pl.kps = up(q.K, 64);
  if (q.M <= 16 && q.la == KMAJ && q.lb == KMAJ) {
    pl.engine = OP_SKINNY;
    return pl;
  }
  const int64_t steps = cdiv(q.K, 64);
  const int64_t need = q.dtype == ORDA_F32 ? 1 : splits_needed(q);
  const int64_t most = std::max<int64_t>(need, std::min<int64_t>(16, std::max<int64_t>(1, steps / 2)));
  int64_t splits = 1;
  double best = 1e300;
  auto take = [&](double cost, int engine, int tile, int64_t sp) {
    if (cost >= best) return;
    best = cost;
    pl.engine = engine;
    pl.tile = tile;
    splits = sp;
  };
  for (int64_t sp = need; sp <= most; ++sp) {
    if (q.dtype == ORDA_F32) {
      take(s3_op_cost(q, sp, true), OP_SPLIT3, 256, sp);
      take(s3_op_cost(q, sp, false), OP_SPLIT3, 64, sp);
      continue;
    }
    for (const TileCost& t : kTileCosts)
      if (items_of(q, t.bm, t.bn, sp) < kMaxItems) take(tile_cost(q, t, sp), OP_TILE, t.bm * 1000 + t.bn, sp);
    if (ring_fits(q, sp)) take(ring_cost(q, sp), OP_RING, 256, sp);
  }
  if (pl.engine == OP_RING && splits == 1) pl.kps = q.K;
  if (splits > 1) {
    pl.kps = up(cdiv(q.K, splits), 64);
    pl.splits = (int)cdiv(q.K, pl.kps);
  }
  return pl;
}

// Whether a launch has the workgroups for a product (looked at where it is
// near: 2^24 tiles of 128 x 64 are at least 2^36 elements).
int check_launch(const char* what, const Shape& q) {
  if ((double)q.M * (double)q.cols >= 34359738368.0 && plan_of(q).engine == OP_NONE)
    return fail(ORDA_EINVAL, "%s: %lld x %lld outputs are more tiles than a launch has workgroups", what, (long long)q.M, (long long)q.cols);
  return ORDA_OK;
}

// Rows and columns of the output that a workgroup (or one turn of a persistent
// one) takes.
void tile_of(const OpPlan& pl, int& rows, int& cols) {
  rows = cols = 16;
  if (pl.engine == OP_TILE) {
    rows = pl.tile / 1000;
    cols = pl.tile % 1000;
  } else if (pl.engine == OP_RING) {
    rows = cols = 256;
  } else if (pl.engine == OP_SPLIT3) {
    rows = pl.tile;
    cols = pl.tile == 256 ? 128 : 64;
  }
}
void fill_plan(const Shape& q, orda_product_plan_t* out) {
  const OpPlan pl = plan_of(q);
  int rows, cols;
  tile_of(pl, rows, cols);
  *out = {pl.engine, rows, cols, pl.splits,
          pl.engine == OP_SKINNY ? cdiv(q.cols, cols) : (int64_t)items_of(q, rows, cols, pl.splits)};
}

// fp32 partials of a product in K ranges
size_t part_bytes(const Shape& q) {
  const OpPlan pl = plan_of(q);
  return pl.splits > 1 ? (size_t)pl.splits * q.M * products(q) * up(q.cols, 4) * (q.dual ? 2 : 1) * 4 : 0;
}

bool rows_aligned(const void* p, int64_t ld, int dtype) { return !p || (aligned16(p) && ld % granule(dtype) == 0); }

// Dispatch on the dtype: f(T{}).
template <class F>
int by_dtype(int dtype, const F& f) {
  switch (dtype) {
    case ORDA_BF16: return f(bf16{});
    case ORDA_F16: return f(f16{});
    default: return f(float{});
  }
}

int check_common(const char* what, int32_t abi, int32_t dtype, int32_t act, int32_t reserved) {
  if (abi != ORDA_ABI_VERSION) return fail(ORDA_EINVAL, "%s: abi_version %d, library has %d", what, abi, ORDA_ABI_VERSION);
  if (dtype < ORDA_BF16 || dtype > ORDA_F32) return fail(ORDA_EINVAL, "%s: unknown dtype %d", what, dtype);
  if (act < 0 || act >= ACT_COUNT) return fail(ORDA_EINVAL, "%s: unknown activation %d", what, act);
  if (reserved != 0) return fail(ORDA_EINVAL, "%s: reserved must be 0", what);
  return ORDA_OK;
}
int check_width(const char* what, const char* name, int64_t v) {
  if (v <= 0 || v > kMaxWidth) return fail(ORDA_EINVAL, "%s: %s must be in [1, 2^21], got %lld", what, name, (long long)v);
  return ORDA_OK;
}
int check_pitch(const char* what, const char* name, int64_t ld, int64_t width, int dtype) {
  const int64_t g = granule(dtype);
  if (ld < up(width, g) || ld % g != 0 || ld > kMaxPitch)
    return fail(ORDA_EINVAL, "%s: %s must be a multiple of %lld in [%lld, 2^22], got %lld", what, name, (long long)g,
                (long long)up(width, g), (long long)ld);
  return ORDA_OK;
}
// Of a gradient: dense rows, or as an operand's; its columns are written up to
// grad_cols.
int check_grad_pitch(const char* what, const char* name, int64_t ld, int64_t width, int dtype) {
  return ld == width ? ORDA_OK : check_pitch(what, name, ld, width, dtype);
}
int64_t grad_cols(int64_t ld, int64_t width, int dtype) { return ld == width ? width : up(width, granule(dtype)); }
int check_residual(const char* what, int64_t ld, int64_t width) {
  if (ld < width || ld > kMaxPitch) return fail(ORDA_EINVAL, "%s: ldr must be in [%lld, 2^22], got %lld", what, (long long)width, (long long)ld);
  return ORDA_OK;
}
#define OP_TRY(expr)                 \
  do {                               \
    const int rc_ = (expr);          \
    if (rc_ != ORDA_OK) return rc_;  \
  } while (0)

int check_workspace(const char* what, void* ws, size_t have, size_t need) {
  if (need > 0 && (!ws || have < need)) return fail(ORDA_EWORKSPACE, "%s: workspace of %zu bytes, need %zu", what, have, need);
  return ORDA_OK;
}

// ----------------------------------------------------------------- linear
struct LinearShapes {
  Shape fwd, dx, dw;
  int64_t op;       // pitch of z and dz
  int64_t blocks;   // row blocks of the bias gradient's partial sums
  int64_t rows_per_block;
};
int linear_shapes(const orda_linear_t* p, LinearShapes& s) {
  const char* what = "orda_linear";
  if (!p) return fail(ORDA_EINVAL, "%s: problem is NULL", what);
  OP_TRY(check_common(what, p->abi_version, p->dtype, p->activation, p->reserved));
  if (p->tokens <= 0 || p->tokens > kMaxTokens) return fail(ORDA_EINVAL, "%s: tokens must be in [1, 2^30], got %lld", what, (long long)p->tokens);
  OP_TRY(check_width(what, "in_features", p->in_features));
  OP_TRY(check_width(what, "out_features", p->out_features));
  OP_TRY(check_pitch(what, "ldx", p->ldx, p->in_features, p->dtype));
  OP_TRY(check_pitch(what, "ldw", p->ldw, p->in_features, p->dtype));
  const int64_t g = granule(p->dtype), kp = up(p->in_features, g);
  s.op = up(p->out_features, g);
  s.fwd = {p->dtype, KMAJ, KMAJ, false, p->tokens, p->out_features, kp, 0, 0, false};
  s.dx = {p->dtype, KMAJ, MNMAJ, false, p->tokens, kp, s.op, 0, p->ldw, false};
  s.dw = {p->dtype, MNMAJ, MNMAJ, false, p->out_features, kp, p->tokens, s.op, p->ldx, false};
  for (const Shape* q : {&s.fwd, &s.dx}) OP_TRY(check_launch(what, *q));
  // about 1024 workgroups, at least 16 rows each (8192 x 4096 in bf16 with 512,
  // 1024, 2048, 4096: 63, 46, 52, 47 us)
  const int64_t per = 64 * g, cb = cdiv(s.op, per);
  s.rows_per_block = std::max<int64_t>(16, up(cdiv(p->tokens * cb, 1024), 4));
  s.blocks = cdiv(p->tokens, s.rows_per_block);
  return ORDA_OK;
}
size_t linear_part(const LinearShapes& s, bool backward) {
  return backward ? std::max(part_bytes(s.dx), part_bytes(s.dw)) : part_bytes(s.fwd);
}
size_t linear_ws(const orda_linear_t* p, const LinearShapes& s, bool backward) {
  if (!backward) return linear_part(s, false) + 256;
  return up((int64_t)linear_part(s, true), 256) + up(s.blocks * p->out_features * 4, 256) + p->tokens * s.op * esize(p->dtype) + 256;
}

template <class T>
TileParams product(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K) {
  TileParams t{};
  t.A = A; t.B = B;
  t.M = M; t.N = N; t.K = K; t.lda = lda; t.ldb = ldb;
  t.kseg = up(K, 64);
  t.kval = K;
  return t;
}
template <class T>
EpiLinear<T> store_to(void* y, int64_t ldy, int64_t cols) {
  EpiLinear<T> e{};
  e.y = static_cast<T*>(y);
  e.ldy = ldy;
  e.cols = cols;
  e.act = ACT_NONE;
  return e;
}

// ------------------------------------------------------------ feed-forward
struct FfnShapes {
  Shape gate, down, dh, dx, dw, dw2, dd;
  int64_t fp;  // pitch of h, a, b: inner rounded to 64 (the K step of dx, whose K has two segments of it)
};
int ffn_shapes(const orda_ffn_t* p, FfnShapes& s) {
  const char* what = "orda_ffn";
  if (!p) return fail(ORDA_EINVAL, "%s: problem is NULL", what);
  OP_TRY(check_common(what, p->abi_version, p->dtype, p->activation, p->reserved));
  if (p->tokens <= 0 || p->tokens > kMaxTokens) return fail(ORDA_EINVAL, "%s: tokens must be in [1, 2^30], got %lld", what, (long long)p->tokens);
  OP_TRY(check_width(what, "hidden", p->hidden));
  OP_TRY(check_width(what, "inner", p->inner));
  OP_TRY(check_width(what, "out_features", p->out_features));
  OP_TRY(check_pitch(what, "ldx", p->ldx, p->hidden, p->dtype));
  OP_TRY(check_pitch(what, "ldw", p->ldw, p->hidden, p->dtype));
  OP_TRY(check_pitch(what, "ldd", p->ldd, p->inner, p->dtype));
  const int64_t g = granule(p->dtype), hp = up(p->hidden, g), ip = up(p->inner, g);
  s.fp = up(p->inner, 64);
  s.gate = {p->dtype, KMAJ, KMAJ, true, p->tokens, s.fp, hp, 0, 0, false};
  s.down = {p->dtype, KMAJ, KMAJ, false, p->tokens, p->out_features, ip, 0, 0, false};
  s.dh = {p->dtype, KMAJ, MNMAJ, false, p->tokens, s.fp, up(p->out_features, g), 0, p->ldd, false};
  s.dx = {p->dtype, KMAJ, MNMAJ, false, p->tokens, hp, 2 * s.fp, 0, p->ldw, false};
  s.dw = {p->dtype, MNMAJ, MNMAJ, false, p->inner, hp, p->tokens, 2 * s.fp, p->ldx, false};
  s.dw2 = s.dw;
  s.dw2.pair = true;
  s.dd = {p->dtype, MNMAJ, MNMAJ, false, p->out_features, ip, p->tokens, p->ldg, s.fp, false};
  for (const Shape* q : {&s.gate, &s.down, &s.dh, &s.dx}) OP_TRY(check_launch(what, *q));
  return ORDA_OK;
}
size_t ffn_part(const FfnShapes& s, bool backward) {
  return backward ? std::max(std::max(part_bytes(s.dh), part_bytes(s.dx)), std::max(part_bytes(s.dw), std::max(part_bytes(s.dw2), part_bytes(s.dd))))
                  : std::max(part_bytes(s.gate), part_bytes(s.down));
}
size_t ffn_ws(const orda_ffn_t* p, const FfnShapes& s, bool backward) {
  if (!backward) return ffn_part(s, false) + 256;
  return up((int64_t)ffn_part(s, true), 256) + p->tokens * 2 * s.fp * esize(p->dtype) + 256;
}

}  // namespace

extern "C" {

int orda_pad_rows(int32_t dtype, const orda_rows_t* t, int64_t n, void* stream) {
  set_last_error(0, nullptr);
  if (dtype < ORDA_BF16 || dtype > ORDA_F32) return fail(ORDA_EINVAL, "orda_pad_rows: unknown dtype %d", dtype);
  if (n < 0 || n > kPadMax || (n > 0 && !t)) return fail(ORDA_EINVAL, "orda_pad_rows: n must be in [0, %d]", kPadMax);
  const int64_t es = esize(dtype), g = granule(dtype);
  PadParams P{};
  for (int64_t i = 0; i < n; ++i) {
    const orda_rows_t& x = t[i];
    if (x.rows < 0 || x.cols <= 0 || x.cols > kMaxPitch || x.rows > kMaxTokens) return fail(ORDA_EINVAL, "orda_pad_rows: tensor %lld has a size out of range", (long long)i);
    if (x.rows == 0) continue;
    if (!x.src || !x.dst || !aligned16(x.dst) || reinterpret_cast<uintptr_t>(x.src) % es) return fail(ORDA_EINVAL, "orda_pad_rows: tensor %lld is not aligned", (long long)i);
    if (x.ld_dst < x.cols || x.ld_dst % g || x.ld_dst > kMaxPitch || (x.rows > 1 && x.ld_src < x.cols)) return fail(ORDA_EINVAL, "orda_pad_rows: tensor %lld has a pitch out of range", (long long)i);
    P.t[P.n++] = {static_cast<const char*>(x.src), static_cast<char*>(x.dst), x.rows, x.cols, x.ld_src, x.ld_dst, P.pieces};
    P.pieces += x.rows * (x.ld_dst / g);
  }
  if (P.n == 0) return ORDA_OK;
  OP_LAUNCH(launch_pad_rows(P, (int)es, static_cast<hipStream_t>(stream)));
  return ORDA_OK;
}

size_t orda_linear_saved_bytes(const orda_linear_t* p) {
  set_last_error(0, nullptr);
  LinearShapes s;
  return linear_shapes(p, s) == ORDA_OK ? (size_t)(p->tokens * s.op * kept_bytes(p->dtype)) : 0;
}

size_t orda_linear_workspace_bytes(const orda_linear_t* p, int32_t backward) {
  set_last_error(0, nullptr);
  LinearShapes s;
  return linear_shapes(p, s) == ORDA_OK ? linear_ws(p, s, backward != 0) : 0;
}

int orda_linear_forward(const orda_linear_t* p, const void* x, const void* weight, const void* bias, const void* residual,
                        void* y, void* d, void* workspace, size_t workspace_bytes, void* stream) {
  set_last_error(0, nullptr);
  LinearShapes s;
  OP_TRY(linear_shapes(p, s));
  if (!x || !weight || !y) return fail(ORDA_EINVAL, "orda_linear_forward: x, weight and y are required");
  if (!aligned16(x) || !aligned16(weight) || !aligned16(d)) return fail(ORDA_EINVAL, "orda_linear_forward: x, weight and d must be 16-byte aligned");
  if (residual) OP_TRY(check_residual("orda_linear_forward", p->ldr, p->out_features));
  OP_TRY(check_workspace("orda_linear_forward", workspace, workspace_bytes, linear_ws(p, s, false)));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return by_dtype(p->dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    EpiLinear<T> e = store_to<T>(y, p->out_features, p->out_features);
    e.d = planes<T>(d, p->tokens * s.op);
    e.bias = static_cast<const T*>(bias);
    e.res = static_cast<const T*>(residual);
    e.ldd = s.op;
    e.ldr = p->ldr;
    e.act = p->activation;
    const TileParams t = product<T>(x, p->ldx, weight, p->ldw, p->tokens, p->out_features, s.fwd.K);
    OP_LAUNCH(launch_op_linear<T>(plan_of(s.fwd), KMAJ, KMAJ, t, e, reinterpret_cast<float*>(base256(workspace)), st));
    return ORDA_OK;
  });
}

int orda_linear_backward(const orda_linear_t* p, const void* x, const void* weight, const void* d, const void* grad_output,
                         void* grad_x, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                         void* stream) {
  set_last_error(0, nullptr);
  LinearShapes s;
  OP_TRY(linear_shapes(p, s));
  if (!grad_output) return fail(ORDA_EINVAL, "orda_linear_backward: grad_output is required");
  if (p->activation != ORDA_ACT_NONE && !d) return fail(ORDA_EINVAL, "orda_linear_backward: d is required with an activation");
  if ((grad_x && !weight) || (grad_weight && !x)) return fail(ORDA_EINVAL, "orda_linear_backward: grad_x needs weight, grad_weight needs x");
  if (!aligned16(x) || !aligned16(weight) || !aligned16(d) || !aligned16(grad_x) || !aligned16(grad_weight))
    return fail(ORDA_EINVAL, "orda_linear_backward: x, weight, d, grad_x and grad_weight must be 16-byte aligned");
  if (grad_x) OP_TRY(check_grad_pitch("orda_linear_backward", "ldgx", p->ldgx, p->in_features, p->dtype));
  if (grad_weight) OP_TRY(check_grad_pitch("orda_linear_backward", "ldgw", p->ldgw, p->in_features, p->dtype));
  OP_TRY(check_workspace("orda_linear_backward", workspace, workspace_bytes, linear_ws(p, s, true)));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = base256(workspace);
  float* part = reinterpret_cast<float*>(ws);
  float* sums = reinterpret_cast<float*>(ws + up((int64_t)linear_part(s, true), 256));
  void* own_dz = reinterpret_cast<char*>(sums) + up(s.blocks * p->out_features * 4, 256);
  return by_dtype(p->dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    // grad_output itself is dz where there is no activation and its rows are
    // aligned as operands are
    const bool act = p->activation != ORDA_ACT_NONE;
    const bool aligned = rows_aligned(grad_output, p->out_features, p->dtype);
    const bool direct = !act && aligned;
    const bool products = grad_x || grad_weight;
    const void* dz = direct ? grad_output : own_dz;
    if (grad_bias || (products && !direct)) {
      DzParams z{};
      z.dy = grad_output;
      z.d = planes<T>(act ? d : nullptr, p->tokens * s.op);
      z.dz = products && !direct ? own_dz : nullptr;
      z.partial = grad_bias ? sums : nullptr;
      z.rows = p->tokens;
      z.cols = p->out_features;
      z.ldy = p->out_features;
      z.ldz = s.op;
      z.rows_per_block = s.rows_per_block;
      OP_LAUNCH(launch_dz<T>(z, st));
      if (grad_bias) OP_LAUNCH(launch_colsum<T>(sums, s.blocks, p->out_features, grad_bias, st));
    }
    if (grad_x) {
      TileParams t = product<T>(dz, s.op, weight, p->ldw, p->tokens, s.dx.cols, s.dx.K);
      t.kval = p->out_features;
      OP_LAUNCH(launch_op_linear<T>(plan_of(s.dx), KMAJ, MNMAJ, t, store_to<T>(grad_x, p->ldgx, grad_cols(p->ldgx, p->in_features, p->dtype)), part, st));
    }
    if (grad_weight) {
      const TileParams t = product<T>(dz, s.op, x, p->ldx, p->out_features, s.dw.cols, p->tokens);
      OP_LAUNCH(launch_op_linear<T>(plan_of(s.dw), MNMAJ, MNMAJ, t, store_to<T>(grad_weight, p->ldgw, grad_cols(p->ldgw, p->in_features, p->dtype)), part, st));
    }
    return ORDA_OK;
  });
}

int orda_linear_plan(const orda_linear_t* p, int32_t product, orda_product_plan_t* out) {
  set_last_error(0, nullptr);
  LinearShapes s;
  OP_TRY(linear_shapes(p, s));
  const Shape* const all[] = {&s.fwd, &s.dx, &s.dw};
  if (!out || product < 0 || product > ORDA_LINEAR_GRAD_WEIGHT) return fail(ORDA_EINVAL, "orda_linear_plan: out is required and product one of orda_product");
  fill_plan(*all[product], out);
  return ORDA_OK;
}

int orda_ffn_plan(const orda_ffn_t* p, int32_t product, orda_product_plan_t* out) {
  set_last_error(0, nullptr);
  FfnShapes s;
  OP_TRY(ffn_shapes(p, s));
  const Shape* const all[] = {&s.gate, &s.down, &s.dh, &s.dx, &s.dw2, &s.dw, &s.dd};
  if (!out || product < 0 || product > ORDA_FFN_GRAD_DOWN) return fail(ORDA_EINVAL, "orda_ffn_plan: out is required and product one of orda_product");
  fill_plan(*all[product], out);
  return ORDA_OK;
}

int64_t orda_ffn_inner_pitch(const orda_ffn_t* p) {
  set_last_error(0, nullptr);
  FfnShapes s;
  return ffn_shapes(p, s) == ORDA_OK ? s.fp : 0;
}

size_t orda_ffn_saved_bytes(const orda_ffn_t* p) {
  set_last_error(0, nullptr);
  FfnShapes s;
  return ffn_shapes(p, s) == ORDA_OK ? (size_t)(p->tokens * s.fp * kept_bytes(p->dtype)) : 0;
}

size_t orda_ffn_workspace_bytes(const orda_ffn_t* p, int32_t backward) {
  set_last_error(0, nullptr);
  FfnShapes s;
  return ffn_shapes(p, s) == ORDA_OK ? ffn_ws(p, s, backward != 0) : 0;
}

int orda_ffn_forward(const orda_ffn_t* p, const void* x, const void* w_gate, const void* w_up, const void* w_down,
                     const void* residual, void* y, void* h, void* da_factor, void* db_factor, void* workspace, size_t workspace_bytes,
                     void* stream) {
  set_last_error(0, nullptr);
  FfnShapes s;
  OP_TRY(ffn_shapes(p, s));
  if (!x || !w_gate || !w_up || !w_down || !y || !h) return fail(ORDA_EINVAL, "orda_ffn_forward: x, the three weights, y and h are required");
  if ((da_factor == nullptr) != (db_factor == nullptr)) return fail(ORDA_EINVAL, "orda_ffn_forward: the two factors are kept together");
  for (const void* q : {x, w_gate, w_up, w_down, (const void*)h, (const void*)da_factor, (const void*)db_factor})
    if (!aligned16(q)) return fail(ORDA_EINVAL, "orda_ffn_forward: x, the weights, h and the factors must be 16-byte aligned");
  if (residual) OP_TRY(check_residual("orda_ffn_forward", p->ldr, p->out_features));
  OP_TRY(check_workspace("orda_ffn_forward", workspace, workspace_bytes, ffn_ws(p, s, false)));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  float* part = reinterpret_cast<float*>(base256(workspace));
  return by_dtype(p->dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    const int64_t kept = p->tokens * s.fp;
    EpiGate<T> g{static_cast<T*>(h), planes<T>(da_factor, kept), planes<T>(db_factor, kept), s.fp, s.fp, (int)p->inner, p->activation};
    TileParams t = product<T>(x, p->ldx, w_gate, p->ldw, p->tokens, p->inner, s.gate.K);
    t.B1 = w_up;
    OP_LAUNCH(launch_op_gate<T>(plan_of(s.gate), t, g, part, st));
    EpiLinear<T> e = store_to<T>(y, p->out_features, p->out_features);
    e.res = static_cast<const T*>(residual);
    e.ldr = p->ldr;
    t = product<T>(h, s.fp, w_down, p->ldd, p->tokens, p->out_features, s.down.K);
    OP_LAUNCH(launch_op_linear<T>(plan_of(s.down), KMAJ, KMAJ, t, e, part, st));
    return ORDA_OK;
  });
}

int orda_ffn_backward(const orda_ffn_t* p, const void* x, const void* w_gate, const void* w_up, const void* w_down,
                      const void* h, const void* da_factor, const void* db_factor, const void* grad_output, void* grad_x, void* grad_gate,
                      void* grad_up, void* grad_down, void* workspace, size_t workspace_bytes, void* stream) {
  set_last_error(0, nullptr);
  FfnShapes s;
  OP_TRY(ffn_shapes(p, s));
  if (!x || !w_gate || !w_up || !w_down || !h || !da_factor || !db_factor || !grad_output)
    return fail(ORDA_EINVAL, "orda_ffn_backward: x, the three weights, h, the two factors and grad_output are required");
  OP_TRY(check_pitch("orda_ffn_backward", "ldg", p->ldg, p->out_features, p->dtype));
  if (grad_x) OP_TRY(check_grad_pitch("orda_ffn_backward", "ldgx", p->ldgx, p->hidden, p->dtype));
  if (grad_gate || grad_up) OP_TRY(check_grad_pitch("orda_ffn_backward", "ldgw", p->ldgw, p->hidden, p->dtype));
  if (grad_down) OP_TRY(check_grad_pitch("orda_ffn_backward", "ldgd", p->ldgd, p->inner, p->dtype));
  for (const void* q : {x, w_gate, w_up, w_down, h, da_factor, db_factor, grad_output, (const void*)grad_x, (const void*)grad_gate, (const void*)grad_up, (const void*)grad_down})
    if (!aligned16(q)) return fail(ORDA_EINVAL, "orda_ffn_backward: every tensor must be 16-byte aligned");
  OP_TRY(check_workspace("orda_ffn_backward", workspace, workspace_bytes, ffn_ws(p, s, true)));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = base256(workspace);
  float* part = reinterpret_cast<float*>(ws);
  char* d = ws + up((int64_t)ffn_part(s, true), 256);  // [tokens x 2 fp]: da, db
  return by_dtype(p->dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    if (grad_x || grad_gate || grad_up) {
      T* const da = reinterpret_cast<T*>(d);
      const int64_t kept = p->tokens * s.fp;
      const EpiGateGrad<T> e{da, da + s.fp, planes<T>(da_factor, kept), planes<T>(db_factor, kept), 2 * s.fp, s.fp, s.fp, (int)p->inner};
      TileParams t = product<T>(grad_output, p->ldg, w_down, p->ldd, p->tokens, p->inner, s.dh.K);
      t.kval = p->out_features;
      OP_LAUNCH(launch_op_gate_grad<T>(plan_of(s.dh), t, e, part, st));
    }
    if (grad_x) {
      TileParams t = product<T>(d, 2 * s.fp, w_gate, p->ldw, p->tokens, s.dx.cols, s.dx.K);
      t.B1 = w_up;
      t.kseg = s.fp;
      t.kval = p->inner;
      OP_LAUNCH(launch_op_linear<T>(plan_of(s.dx), KMAJ, MNMAJ, t, store_to<T>(grad_x, p->ldgx, grad_cols(p->ldgx, p->hidden, p->dtype)), part, st));
    }
    if (grad_gate && grad_up) {  // one launch: its tiles fill the chip's last round better than two launches' do
      TileParams t = product<T>(d, 2 * s.fp, x, p->ldx, p->inner, s.dw2.cols, p->tokens);
      t.pair = s.fp;
      EpiLinear<T> e = store_to<T>(grad_gate, p->ldgw, grad_cols(p->ldgw, p->hidden, p->dtype));
      e.y1 = static_cast<T*>(grad_up);
      OP_LAUNCH(launch_op_linear<T>(plan_of(s.dw2), MNMAJ, MNMAJ, t, e, part, st));
    } else if (grad_gate || grad_up) {
      const TileParams t = product<T>(d + (grad_up ? s.fp * (int64_t)sizeof(T) : 0), 2 * s.fp, x, p->ldx, p->inner, s.dw.cols, p->tokens);
      OP_LAUNCH(launch_op_linear<T>(plan_of(s.dw), MNMAJ, MNMAJ, t, store_to<T>(grad_up ? grad_up : grad_gate, p->ldgw, grad_cols(p->ldgw, p->hidden, p->dtype)), part, st));
    }
    if (grad_down) {
      const TileParams t = product<T>(grad_output, p->ldg, h, s.fp, p->out_features, s.dd.cols, p->tokens);
      OP_LAUNCH(launch_op_linear<T>(plan_of(s.dd), MNMAJ, MNMAJ, t, store_to<T>(grad_down, p->ldgd, grad_cols(p->ldgd, p->inner, p->dtype)), part, st));
    }
    return ORDA_OK;
  });
}

// ------------------------------------------------------------ gradient norm
size_t orda_grad_norm_workspace_bytes(void) { return (size_t)kNormPartials * sizeof(double) + 256; }

}  // extern "C"

namespace {

int spans_of(const char* what, const orda_grad_t* g, int64_t n, bool outputs, std::vector<GradSpan>& v) {
  if (n < 0 || (n > 0 && !g)) return fail(ORDA_EINVAL, "%s: a table of n >= 0 gradients is required", what);
  v.reserve((size_t)n);
  for (int64_t i = 0; i < n; ++i) {
    const orda_grad_t& x = g[i];
    if (x.rows < 0 || x.cols < 0) return fail(ORDA_EINVAL, "%s: gradient %lld has a negative size", what, (long long)i);
    if (x.rows == 0 || x.cols == 0) continue;
    if (x.rows > (1ll << 40) / x.cols) return fail(ORDA_EINVAL, "%s: gradient %lld has more than 2^40 elements", what, (long long)i);
    if (!x.data) return fail(ORDA_EINVAL, "%s: gradient %lld has no data", what, (long long)i);
    if (x.dtype < ORDA_BF16 || x.dtype > ORDA_F32) return fail(ORDA_EINVAL, "%s: gradient %lld has unknown dtype %d", what, (long long)i, x.dtype);
    const int64_t es = esize(x.dtype);
    if (reinterpret_cast<uintptr_t>(x.data) % es != 0) return fail(ORDA_EINVAL, "%s: gradient %lld is not aligned to its elements", what, (long long)i);
    GradSpan s{x.data, x.data, x.rows, x.cols, x.ld, x.ld, x.dtype, x.dtype};
    if (outputs && x.out) {
      if (x.out_dtype < ORDA_BF16 || x.out_dtype > ORDA_F32) return fail(ORDA_EINVAL, "%s: gradient %lld has unknown out_dtype %d", what, (long long)i, x.out_dtype);
      if (reinterpret_cast<uintptr_t>(x.out) % esize(x.out_dtype) != 0) return fail(ORDA_EINVAL, "%s: out %lld is not aligned to its elements", what, (long long)i);
      s.out = x.out;
      s.ld_out = x.ld_out;
      s.out_dtype = x.out_dtype;
    }
    if (s.rows > 1 && (s.ld < s.cols || s.ld_out < s.cols)) return fail(ORDA_EINVAL, "%s: gradient %lld has rows that overlap", what, (long long)i);
    // a tensor whose rows follow one another is one row
    if (s.rows > 1 && s.ld == s.cols && s.ld_out == s.cols) {
      s.cols *= s.rows;
      s.rows = 1;
    }
    v.push_back(s);
  }
  return ORDA_OK;
}

int norm_kind_of(double p) { return p == 2.0 ? 2 : p == 1.0 ? 1 : (std::isinf(p) && p > 0) ? 0 : -1; }

// Whether the bytes of two row sets meet, a.lo <= b.lo < a's end.  Sets of the
// same pitch whose columns lie beside each other (two halves of one buffer)
// do not; anything else that is interleaved counts as meeting.
struct Extent {
  uintptr_t lo, hi;  // first byte, one past the last
  int64_t pitch, width;
  int64_t index;
  bool written;
};
bool meet(const Extent& a, const Extent& b) {
  if (b.lo >= a.hi) return false;
  if (a.pitch != b.pitch || a.pitch == 0) return true;
  const int64_t c = (int64_t)(b.lo - a.lo) % a.pitch;  // b's columns relative to a's
  return c < a.width || c + b.width > a.pitch;
}
// What one call writes may meet nothing else that it reads or writes, a
// gradient in place its own input alone.
int check_overlap(const char* what, const std::vector<GradSpan>& v) {
  std::vector<Extent> e;
  e.reserve(2 * v.size());
  auto add = [&](size_t i, const void* p, int64_t ld, int64_t es, bool written) {
    const GradSpan& s = v[i];
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    e.push_back({lo, lo + (uintptr_t)(((s.rows - 1) * ld + s.cols) * es), s.rows > 1 ? ld * es : 0, s.cols * es, (int64_t)i, written});
  };
  for (size_t i = 0; i < v.size(); ++i) {
    const GradSpan& s = v[i];
    add(i, s.out, s.ld_out, esize(s.out_dtype), true);
    if (s.out != s.p || s.out_dtype != s.in_dtype || (s.rows > 1 && s.ld != s.ld_out)) add(i, s.p, s.ld, esize(s.in_dtype), false);
  }
  std::sort(e.begin(), e.end(), [](const Extent& a, const Extent& b) { return a.lo < b.lo; });
  for (size_t i = 0; i < e.size(); ++i)
    for (size_t j = i + 1; j < e.size() && e[j].lo < e[i].hi; ++j)
      if ((e[i].written || e[j].written) && meet(e[i], e[j]))
        return fail(ORDA_EINVAL, "%s: gradients %lld and %lld meet in memory that is written", what, (long long)e[i].index, (long long)e[j].index);
  return ORDA_OK;
}

}  // namespace

extern "C" {

int orda_grad_norm(const orda_grad_t* grads, int64_t n, double norm_type, float* total, void* workspace,
                   size_t workspace_bytes, void* stream) {
  set_last_error(0, nullptr);
  try {
    if (!total) return fail(ORDA_EINVAL, "orda_grad_norm: total is required");
    const int kind = norm_kind_of(norm_type);
    if (kind < 0) return fail(ORDA_EINVAL, "orda_grad_norm: norm_type must be 1, 2 or infinity, got %g", norm_type);
    OP_TRY(check_workspace("orda_grad_norm", workspace, workspace_bytes, orda_grad_norm_workspace_bytes()));
    std::vector<GradSpan> v;
    OP_TRY(spans_of("orda_grad_norm", grads, n, false, v));
    OP_LAUNCH(launch_grad_norm(v.data(), (int64_t)v.size(), kind, reinterpret_cast<double*>(base256(workspace)), kNormPartials, total, static_cast<hipStream_t>(stream)));
    return ORDA_OK;
  } catch (const std::exception& e) {
    return fail(ORDA_EINVAL, "orda_grad_norm: %s", e.what());
  }
}

int orda_clip_grad_norm(const orda_grad_t* grads, int64_t n, double norm_type, double max_norm, float* total, void* workspace,
                        size_t workspace_bytes, void* stream) {
  set_last_error(0, nullptr);
  try {
    if (!total) return fail(ORDA_EINVAL, "orda_clip_grad_norm: total is required");
    const int kind = norm_kind_of(norm_type);
    if (kind < 0) return fail(ORDA_EINVAL, "orda_clip_grad_norm: norm_type must be 1, 2 or infinity, got %g", norm_type);
    if (!(max_norm >= 0.0)) return fail(ORDA_EINVAL, "orda_clip_grad_norm: max_norm must be >= 0, got %g", max_norm);
    OP_TRY(check_workspace("orda_clip_grad_norm", workspace, workspace_bytes, orda_grad_norm_workspace_bytes()));
    std::vector<GradSpan> v;
    OP_TRY(spans_of("orda_clip_grad_norm", grads, n, true, v));
    OP_TRY(check_overlap("orda_clip_grad_norm", v));
    OP_LAUNCH(launch_clip_grad_norm(v.data(), (int64_t)v.size(), kind, reinterpret_cast<double*>(base256(workspace)), kNormPartials, total,
                                    (float)max_norm, static_cast<hipStream_t>(stream)));
    return ORDA_OK;
  } catch (const std::exception& e) {
    return fail(ORDA_EINVAL, "orda_clip_grad_norm: %s", e.what());
  }
}

int orda_clip_grads(const orda_grad_t* grads, int64_t n, const float* total, double max_norm, void* stream) {
  set_last_error(0, nullptr);
  try {
    if (!total) return fail(ORDA_EINVAL, "orda_clip_grads: total is required");
    if (!(max_norm >= 0.0)) return fail(ORDA_EINVAL, "orda_clip_grads: max_norm must be >= 0, got %g", max_norm);
    std::vector<GradSpan> v;
    OP_TRY(spans_of("orda_clip_grads", grads, n, true, v));
    OP_TRY(check_overlap("orda_clip_grads", v));
    OP_LAUNCH(launch_clip_grads(v.data(), (int64_t)v.size(), total, (float)max_norm, static_cast<hipStream_t>(stream)));
    return ORDA_OK;
  } catch (const std::exception& e) {
    return fail(ORDA_EINVAL, "orda_clip_grads: %s", e.what());
  }
}

}  // extern "C"
