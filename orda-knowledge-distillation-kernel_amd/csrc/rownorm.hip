// rownorm.hip -- dropout and layer norm: passes over rows of a student's
// residual stream, bound by memory.
//
// Dropout's bits are made again in the backward pass (philox.hpp).  The norm's
// forward pass reads x and the residual once, holds the row in registers (two
// passes over them: the mean, then the squares of what is left, so that an
// offset cancels before it is squared) and writes s, y and the row's mean and
// 1 / sqrt(variance + eps).  Its backward pass reads s, dy and the gradient of s
// once:
//   h = (s - mean) rstd, g = dy w
//   ds' = ds + rstd (g - mean(g) - h mean(g h)), dx = keep(ds') factor, dr = ds'
// and adds up dw = sum dy h and db = sum dy on the way, each thread over its own
// columns of all rows that its workgroup walks, in fp32; a second kernel adds
// up the workgroups' sums in order.  No atomics: results do not depend on the
// run.
//
// A row has LPR lanes (8, a wave, 256 or 1024 threads) with NP pieces of 8
// consecutive elements each, the k-th of lane l piece l + k LPR.
#include <algorithm>

#include "pieces.hpp"
#include "step_launch.hpp"

namespace orda {

// ------------------------------------------------------------- dropout
// One piece a thread: 256 threads 2048 elements, as clipping has it (two a thread
// took 76 us instead of 74).  Bound by memory: 16384 x 4096 in bf16 with a residual
// 403 MB in 74 us, without, as the backward pass has it, 268 MB in 44.
template <class T, bool RES, bool EVEN>
__global__ __launch_bounds__(256) void k_dropout(DropoutParams P, int64_t per_row, int64_t pieces) {
  const uint64_t seed = seed_of(P.drop);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
    int64_t row = 0, k = i;
    if (P.rows > 1) {
      row = pieces <= 0xffffffffll ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row;
      k -= row * per_row;
    }
    const Piece<EVEN> p(k, P.cols);
    Raw8<T> x, r;
    x.get(static_cast<const T*>(P.x) + row * P.ldx, p);
    if constexpr (RES) r.get(static_cast<const T*>(P.residual) + row * P.ldr, p);
    const uint32_t m = keep8<EVEN>(row * P.cols + p.c, seed, P.drop.site, P.drop.threshold);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // (a dropped infinity or NaN leaves nothing)
      y[e] = (m >> e) & 1 ? x[e] * P.drop.factor : 0.0f;
      if constexpr (RES) y[e] += r[e];
    }
    put8(static_cast<T*>(P.y) + row * P.cols, p, y);
  }
}

template <class T>
static hipError_t dropout_go(const DropoutParams& P, hipStream_t s) {
  const int64_t per_row = pieces_of(P.cols), pieces = per_row * P.rows;
  // (a launch has fewer than 2^32 threads; past them a thread takes several pieces)
  const unsigned groups = (unsigned)std::min<int64_t>((pieces + 255) / 256, 1 << 23);
  auto go = [&](auto residual, auto even) {
    hipLaunchKernelGGL((k_dropout<T, decltype(residual)::value, decltype(even)::value>), dim3(groups), dim3(256), 0, s, P, per_row, pieces);
  };
  const bool even = P.cols % 8 == 0;
  if (P.residual) even ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
  else even ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
  return hipGetLastError();
}
hipError_t launch_dropout(const DropoutParams& P, int dtype, hipStream_t s) {
  switch (dtype) {
    case DT_BF16: return dropout_go<bf16>(P, s);
    case DT_F16: return dropout_go<f16>(P, s);
    default: return dropout_go<float>(P, s);
  }
}

// ------------------------------------------------------------- row sums
// v of all lanes of the row's LPR added up, in every lane; `red`: N floats per
// wave, others for every call between two barriers.
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, false));   // lane ^ 1
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, false));   // lane ^ 2
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, false));  // the other quad of 8
  if constexpr (LPR > 8) {
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, false));  // the other 8 of 16
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return v;
}
template <int LPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<LPR>(v[i]);
  if constexpr (LPR > 64) {
    constexpr int kWaves = LPR / 64;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[i * kWaves + w] = v[i];
    tile_barrier();  // (no wait for loads and stores in flight)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) t += red[i * kWaves + k];
      v[i] = t;
    }
  }
}

constexpr int group_threads(int lpr) { return lpr > 256 ? lpr : 256; }

// s of one piece: residual + keep(x) factor
template <bool EVEN, class T>
__device__ __forceinline__ void stream_piece(float (&s)[8], const Raw8<T>& x, const Raw8<T>& r, bool residual, int64_t index, const DropParams& d, uint64_t seed) {
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = x[e];
  if (d.threshold) {
    const uint32_t m = keep8<EVEN>(index, seed, d.site, d.threshold);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = (m >> e) & 1 ? s[e] * d.factor : 0.0f;
  }
  if (residual)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += r[e];
}

// ------------------------------------------------------------- forward
// The next row is loaded while this one is worked on.  Bound by memory: 16384 x
// 4096 in bf16 with dropout and residual 537 MB in 97 us.
template <class T, class W, int LPR, int NP, bool EVEN>
__global__ __launch_bounds__(group_threads(LPR)) void k_layer_norm(LayerNormParams P) {
  constexpr int kRows = group_threads(LPR) / LPR, kWaves = group_threads(LPR) / 64;
  __shared__ float red[2][2][kWaves];
  const int lane = threadIdx.x % LPR;
  const uint64_t seed = P.drop.threshold ? seed_of(P.drop) : 0;
  const float n_cols = (float)P.cols;
  Piece<EVEN> at[NP];
  Raw8<W> w[NP], b[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    at[k] = Piece<EVEN>(lane + k * LPR, P.cols);
    w[k].get(static_cast<const W*>(P.weight), at[k]);
    if (P.bias) b[k].get(static_cast<const W*>(P.bias), at[k]);
  }
  const bool residual = P.residual != nullptr;
  struct Loaded {
    Raw8<T> x[NP], r[NP];
  };
  const int64_t steps = (P.rows + kRows - 1) / kRows, own = threadIdx.x / LPR;
  // (behind the last row: the last row again, not stored)
  auto load = [&](int64_t step, Loaded& q) {
    const int64_t row = lmin(step * kRows + own, P.rows - 1);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      q.x[k].get(static_cast<const T*>(P.x) + row * P.ldx, at[k]);
      if (residual) q.r[k].get(static_cast<const T*>(P.residual) + row * P.ldr, at[k]);
    }
  };
  int turn = 0;
  Loaded next;
  load(blockIdx.x, next);
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x, turn ^= 1) {
    const Loaded q = next;
    if (step + gridDim.x < steps) load(step + gridDim.x, next);
    const int64_t row = step * kRows + own;
    float v[NP][8], sum[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      stream_piece<EVEN>(v[k], q.x[k], q.r[k], residual, row * P.cols + at[k].c, P.drop, seed);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0] += at[k].own(e) ? v[k][e] : 0.0f;
    }
    row_sums<LPR>(sum, red[turn][0]);
    const float mean = sum[0] / n_cols;
    sum[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = at[k].own(e) ? v[k][e] - mean : 0.0f;
        sum[0] = fmaf(d, d, sum[0]);
      }
    row_sums<LPR>(sum, red[turn][1]);
    const float rstd = 1.0f / sqrtf(sum[0] / n_cols + P.eps);
    if (row >= P.rows) continue;
    if (P.stats && lane == 0) *reinterpret_cast<float2*>(P.stats + 2 * row) = make_float2(mean, rstd);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      if (P.s) put8(static_cast<T*>(P.s) + row * P.cols, at[k], v[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float h = (v[k][e] - mean) * rstd;
        v[k][e] = P.bias ? fmaf(h, w[k][e], b[k][e]) : h * w[k][e];
      }
      put8(static_cast<T*>(P.y) + row * P.cols, at[k], v[k]);
    }
  }
}

// Rows longer than a workgroup's registers hold: 1024 threads read the row three
// times (the second and third time from the caches).
template <class T, class W, bool EVEN>
__global__ __launch_bounds__(1024) void k_layer_norm_long(LayerNormParams P) {
  __shared__ float red[2][2][16];
  const uint64_t seed = P.drop.threshold ? seed_of(P.drop) : 0;
  const float n_cols = (float)P.cols;
  const int64_t pieces = pieces_of(P.cols);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x, turn ^= 1) {
    auto piece = [&](const Piece<EVEN>& at, float (&v)[8]) {
      Raw8<T> x, r;
      x.get(static_cast<const T*>(P.x) + row * P.ldx, at);
      if (P.residual) r.get(static_cast<const T*>(P.residual) + row * P.ldr, at);
      stream_piece<EVEN>(v, x, r, P.residual != nullptr, row * P.cols + at.c, P.drop, seed);
    };
    float sum[1] = {0.0f}, v[8];
    for (int64_t i = threadIdx.x; i < pieces; i += 1024) {
      const Piece<EVEN> at(i, P.cols);
      piece(at, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0] += at.own(e) ? v[e] : 0.0f;
      if (P.s) put8(static_cast<T*>(P.s) + row * P.cols, at, v);
    }
    row_sums<1024>(sum, red[turn][0]);
    const float mean = sum[0] / n_cols;
    sum[0] = 0.0f;
    for (int64_t i = threadIdx.x; i < pieces; i += 1024) {
      const Piece<EVEN> at(i, P.cols);
      piece(at, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = at.own(e) ? v[e] - mean : 0.0f;
        sum[0] = fmaf(d, d, sum[0]);
      }
    }
    row_sums<1024>(sum, red[turn][1]);
    const float rstd = 1.0f / sqrtf(sum[0] / n_cols + P.eps);
    if (P.stats && threadIdx.x == 0) *reinterpret_cast<float2*>(P.stats + 2 * row) = make_float2(mean, rstd);
    for (int64_t i = threadIdx.x; i < pieces; i += 1024) {
      const Piece<EVEN> at(i, P.cols);
      Raw8<W> w, b;
      piece(at, v);
      w.get(static_cast<const W*>(P.weight), at);
      if (P.bias) b.get(static_cast<const W*>(P.bias), at);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float h = (v[e] - mean) * rstd;
        v[e] = P.bias ? fmaf(h, w[e], b[e]) : h * w[e];
      }
      put8(static_cast<T*>(P.y) + row * P.cols, at, v);
    }
  }
}

// ------------------------------------------------------------- backward
// ds' of one piece to dr, and what dropout leaves of it to dx.
template <class T, bool EVEN>
__device__ __forceinline__ void grad_piece(const LayerNormGradParams& P, float (&t)[8], int64_t row, const Piece<EVEN>& at, uint32_t kept) {
  if (P.dr) put8(static_cast<T*>(P.dr) + row * P.cols, at, t);
  if (!P.dx) return;
  if (P.drop.threshold)
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (kept >> e) & 1 ? t[e] * P.drop.factor : 0.0f;
  put8(static_cast<T*>(P.dx) + row * P.cols, at, t);
}

// AGAIN: s is computed again from x and the residual, in fp32.  fp32 parameters
// beside 16-bit tensors get gradients of fp32's precision so, for 2 more bytes
// read of 16 to 20; from s as it was rounded dw is off by half a step of the
// 16-bit type (2e-4 of its norm in fp16, 2.4e-3 in bf16, where 1.7e-3 come from
// its own rounding).  Bound by memory: 16384 x 4096 in bf16 with dropout and
// residual 671 MB in 134 us.
template <class T, class W, int LPR, int NP, bool EVEN, bool AGAIN>
__global__ __launch_bounds__(group_threads(LPR)) void k_layer_norm_grad(LayerNormGradParams P) {
  constexpr int kRows = group_threads(LPR) / LPR, kWaves = group_threads(LPR) / 64;
  __shared__ float red[2][2 * kWaves];
  const int lane = threadIdx.x % LPR;
  const uint64_t seed = P.drop.threshold ? seed_of(P.drop) : 0;
  const float n_cols = (float)P.cols;
  Piece<EVEN> at[NP];
  Raw8<W> w[NP];
  float dw[NP][8], db[NP][8];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    at[k] = Piece<EVEN>(lane + k * LPR, P.cols);
    w[k].get(static_cast<const W*>(P.weight), at[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[k][e] = db[k][e] = 0.0f;
  }
  struct Loaded {
    Raw8<T> s[NP], dy[NP], ds[NP], r[AGAIN ? NP : 1];
    float2 st;
  };
  const int64_t steps = (P.rows + kRows - 1) / kRows, own = threadIdx.x / LPR;
  auto load = [&](int64_t step, Loaded& q) {
    const int64_t row = lmin(step * kRows + own, P.rows - 1);
    q.st = *reinterpret_cast<const float2*>(P.stats + 2 * row);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      q.s[k].get(static_cast<const T*>(P.s) + row * P.ld_s, at[k]);
      if constexpr (AGAIN) q.r[k].get(static_cast<const T*>(P.residual) + row * P.ldr, at[k]);
      q.dy[k].get(static_cast<const T*>(P.dy) + row * P.ldy, at[k]);
      if (P.ds) q.ds[k].get(static_cast<const T*>(P.ds) + row * P.ldd, at[k]);
    }
  };
  int turn = 0;
  Loaded next;
  load(blockIdx.x, next);
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x, turn ^= 1) {
    const Loaded q = next;
    if (step + gridDim.x < steps) load(step + gridDim.x, next);
    const int64_t row = step * kRows + own;
    const bool live = row < P.rows;
    float h[NP][8], sum[2] = {0.0f, 0.0f};
    uint32_t kept[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      kept[k] = 0xff;
      if (P.drop.threshold) kept[k] = keep8<EVEN>(row * P.cols + at[k].c, seed, P.drop.site, P.drop.threshold);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float s = q.s[k][e];
        if constexpr (AGAIN) s = ((kept[k] >> e) & 1 ? s * P.drop.factor : 0.0f) + q.r[k][e];
        h[k][e] = (s - q.st.x) * q.st.y;
        const float g = live ? q.dy[k][e] : 0.0f, gw = at[k].own(e) ? g * w[k][e] : 0.0f;
        sum[0] += gw;
        sum[1] = fmaf(gw, h[k][e], sum[1]);
        // (a row that is read twice, behind the last, has g = 0; h may not be finite there)
        dw[k][e] = live ? fmaf(g, h[k][e], dw[k][e]) : dw[k][e];
        db[k][e] += g;
      }
    }
    if (P.dx || P.dr) {
      row_sums<LPR>(sum, red[turn]);
      const float mg = sum[0] / n_cols, mgh = sum[1] / n_cols;
      if (live)
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          float t[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            t[e] = q.st.y * (fmaf(q.dy[k][e], w[k][e], -mg) - h[k][e] * mgh);
            if (P.ds) t[e] += q.ds[k][e];
          }
          grad_piece<T, EVEN>(P, t, row, at[k], kept[k]);
        }
    }
  }
  if (!P.partial) return;
  if constexpr (kRows > 1) {  // the rows of a workgroup, in order
    __shared__ float join[(kRows - 1) * LPR * 8];
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        float(&v)[8] = part ? db[k] : dw[k];
        const int r = threadIdx.x / LPR;
        __syncthreads();
        if (r)
#pragma unroll
          for (int e = 0; e < 8; ++e) join[((r - 1) * 8 + e) * LPR + lane] = v[e];
        __syncthreads();
        if (!r)
          for (int i = 0; i < kRows - 1; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += join[(i * 8 + e) * LPR + lane];
      }
    if (threadIdx.x >= LPR) return;
  }
  float* out = P.partial + (int64_t)blockIdx.x * 2 * P.cols;
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    put8(out, at[k], dw[k]);
    put8(out + P.cols, at[k], db[k]);
  }
}

// Long rows: sums of dw and db in the workgroup's own rows of `partial`, which
// each thread reads and writes at its own columns only (of two pieces that
// overlap the second adds up its own elements).
template <class T, class W, bool EVEN>
__global__ __launch_bounds__(1024) void k_layer_norm_grad_long(LayerNormGradParams P) {
  __shared__ float red[2][32];
  const uint64_t seed = P.drop.threshold ? seed_of(P.drop) : 0;
  const float n_cols = (float)P.cols;
  const int64_t pieces = pieces_of(P.cols);
  float* part = P.partial ? P.partial + (int64_t)blockIdx.x * 2 * P.cols : nullptr;
  int turn = 0;
  bool first = true;
  for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x, turn ^= 1, first = false) {
    const float2 st = *reinterpret_cast<const float2*>(P.stats + 2 * row);
    float sum[2] = {0.0f, 0.0f}, s[8];
    Raw8<T> g;
    Raw8<W> w;
    uint32_t kept = 0xff;
    auto piece = [&](const Piece<EVEN>& at) {
      Raw8<T> x, r;
      x.get(static_cast<const T*>(P.s) + row * P.ld_s, at);
      if (P.residual) r.get(static_cast<const T*>(P.residual) + row * P.ldr, at);
      g.get(static_cast<const T*>(P.dy) + row * P.ldy, at);
      w.get(static_cast<const W*>(P.weight), at);
      if (P.drop.threshold) kept = keep8<EVEN>(row * P.cols + at.c, seed, P.drop.site, P.drop.threshold);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[e] = x[e];
        if (P.residual) s[e] = ((kept >> e) & 1 ? s[e] * P.drop.factor : 0.0f) + r[e];
      }
    };
    for (int64_t i = threadIdx.x; i < pieces; i += 1024) {
      const Piece<EVEN> at(i, P.cols);
      piece(at);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!at.own(e)) continue;
        const float h = (s[e] - st.x) * st.y, gw = g[e] * w[e];
        sum[0] += gw;
        sum[1] = fmaf(gw, h, sum[1]);
        if (part) {
          float* a = part + at.c + e;
          a[0] = fmaf(g[e], h, first ? 0.0f : a[0]);
          a[P.cols] = g[e] + (first ? 0.0f : a[P.cols]);
        }
      }
    }
    if (!P.dx && !P.dr) continue;
    row_sums<1024>(sum, red[turn]);
    const float mg = sum[0] / n_cols, mgh = sum[1] / n_cols;
    for (int64_t i = threadIdx.x; i < pieces; i += 1024) {
      const Piece<EVEN> at(i, P.cols);
      piece(at);
      float t[8];
      Raw8<T> ds;
      if (P.ds) ds.get(static_cast<const T*>(P.ds) + row * P.ldd, at);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[e] = st.y * (fmaf(g[e], w[e], -mg) - (s[e] - st.x) * st.y * mgh);
        if (P.ds) t[e] += ds[e];
      }
      grad_piece<T, EVEN>(P, t, row, at, kept);
    }
  }
}

// dw and db: 64 columns a workgroup, its 16 waves every 16th of the groups (512
// groups of 4096 columns: 17 MB in 5 us).
template <class W>
__global__ __launch_bounds__(1024) void k_layer_norm_params(const float* partial, int64_t groups, int64_t cols, W* dw, W* db) {
  __shared__ float join[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  float v = 0.0f;
  if (c < cols) {
    const float* p = partial + blockIdx.y * cols + c;
#pragma unroll 8
    for (int64_t g = wave; g < groups; g += 16) v += p[2 * g * cols];
  }
  join[wave][lane] = v;
  __syncthreads();
  if (wave || c >= cols) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v += join[i][lane];
  out[c] = from_f32<W>(v);
}

// ------------------------------------------------------------- launches
// f(LPR, NP, EVEN) of a row length; LPR 0: the long kernels.
template <class F>
static hipError_t for_width(int64_t cols, const F& f) {
  using std::integral_constant;
#define ORDA_ROW(L, N) (cols % 8 == 0 ? f(integral_constant<int, L>{}, integral_constant<int, N>{}, std::true_type{}) \
                                      : f(integral_constant<int, L>{}, integral_constant<int, N>{}, std::false_type{}))
  if (cols <= 64) return ORDA_ROW(8, 1);
  if (cols <= 512) return ORDA_ROW(64, 1);
  if (cols <= 1024) return ORDA_ROW(64, 2);
  if (cols <= 2048) return ORDA_ROW(256, 1);
  if (cols <= 4096) return ORDA_ROW(256, 2);
  if (cols <= 8192) return ORDA_ROW(1024, 1);
  return ORDA_ROW(0, 0);
#undef ORDA_ROW
}
static int64_t rows_per_group(int64_t cols) { return cols <= 64 ? 32 : cols <= 1024 ? 4 : 1; }
static int64_t threads_of(int64_t cols) { return cols <= 4096 ? 256 : 1024; }

// Workgroups of a pass: at 16384 x 4096 any number from 256 to 1024 backward and
// from 1024 to 16384 forward takes the same time (130 to 143 us, 92 to 96); fewer
// backward are fewer sums to add up.  Chosen at that width only; rows of more than
// 4096 have 1024 threads and fewer workgroups, of which 5120 columns leave 6 waves of
// 16 without a piece.  Forward and backward with dropout and residual in bf16:
// 16384 x 5120 162 to 191 and 169 to 209 us (its bytes at 6.2 TB/s: 108 and 135), 8192 x
// 8192 102 and 126 (87 and 108), 4096 x 16384, by the long kernels, 189 and 606 (87
// and 108: rows are read three times forward and twice backward, and dw and db added
// up in memory for every row, 4 bytes at a time).
constexpr int64_t kGradGroups = 512, kNormGroups = 2048;
int64_t layer_norm_groups(int64_t rows, int64_t cols) {
  const int64_t steps = (rows + rows_per_group(cols) - 1) / rows_per_group(cols);
  return std::min<int64_t>(steps, threads_of(cols) == 256 ? kGradGroups : 256);
}

template <class T, class W>
static hipError_t norm_go(const LayerNormParams& P, hipStream_t s) {
  const int64_t steps = (P.rows + rows_per_group(P.cols) - 1) / rows_per_group(P.cols);
  const unsigned groups = (unsigned)std::min<int64_t>(steps, threads_of(P.cols) == 256 ? kNormGroups : 512);
  return for_width(P.cols, [&](auto l, auto n, auto even) {
    constexpr int L = decltype(l)::value, N = decltype(n)::value;
    constexpr bool E = decltype(even)::value;
    if constexpr (L == 0) hipLaunchKernelGGL((k_layer_norm_long<T, W, E>), dim3(groups), dim3(1024), 0, s, P);
    else hipLaunchKernelGGL((k_layer_norm<T, W, L, N, E>), dim3(groups), dim3(group_threads(L)), 0, s, P);
    return hipGetLastError();
  });
}
template <class T, class W>
static hipError_t norm_grad_go(const LayerNormGradParams& P, hipStream_t s) {
  const unsigned groups = (unsigned)layer_norm_groups(P.rows, P.cols);
  return for_width(P.cols, [&](auto l, auto n, auto even) {
    constexpr int L = decltype(l)::value, N = decltype(n)::value;
    constexpr bool E = decltype(even)::value;
    auto go = [&](auto again) {
      hipLaunchKernelGGL((k_layer_norm_grad<T, W, L, N, E, decltype(again)::value>), dim3(groups), dim3(group_threads(L)), 0, s, P);
    };
    if constexpr (L == 0) {
      hipLaunchKernelGGL((k_layer_norm_grad_long<T, W, E>), dim3(groups), dim3(1024), 0, s, P);
    } else if constexpr (sizeof(T) < sizeof(W)) {
      if (P.residual) go(std::true_type{});
      else go(std::false_type{});
    } else {
      go(std::false_type{});
    }
    return hipGetLastError();
  });
}
// Parameters are fp32 or of the tensors' type.
hipError_t launch_layer_norm(const LayerNormParams& P, int dtype, int param_dtype, hipStream_t s) {
  if (dtype == DT_F32) return norm_go<float, float>(P, s);
  if (dtype == DT_F16) return param_dtype == DT_F32 ? norm_go<f16, float>(P, s) : norm_go<f16, f16>(P, s);
  return param_dtype == DT_F32 ? norm_go<bf16, float>(P, s) : norm_go<bf16, bf16>(P, s);
}
hipError_t launch_layer_norm_grad(const LayerNormGradParams& P, int dtype, int param_dtype, hipStream_t s) {
  if (dtype == DT_F32) return norm_grad_go<float, float>(P, s);
  if (dtype == DT_F16) return param_dtype == DT_F32 ? norm_grad_go<f16, float>(P, s) : norm_grad_go<f16, f16>(P, s);
  return param_dtype == DT_F32 ? norm_grad_go<bf16, float>(P, s) : norm_grad_go<bf16, bf16>(P, s);
}
hipError_t launch_layer_norm_params(const float* partial, int64_t groups, int64_t cols, void* dw, void* db, int param_dtype, hipStream_t s) {
  const dim3 grid((unsigned)((cols + 63) / 64), 2);
  switch (param_dtype) {
    case DT_BF16: hipLaunchKernelGGL((k_layer_norm_params<bf16>), grid, dim3(1024), 0, s, partial, groups, cols, (bf16*)dw, (bf16*)db); break;
    case DT_F16: hipLaunchKernelGGL((k_layer_norm_params<f16>), grid, dim3(1024), 0, s, partial, groups, cols, (f16*)dw, (f16*)db); break;
    default: hipLaunchKernelGGL((k_layer_norm_params<float>), grid, dim3(1024), 0, s, partial, groups, cols, (float*)dw, (float*)db);
  }
  return hipGetLastError();
}

}  // namespace orda
