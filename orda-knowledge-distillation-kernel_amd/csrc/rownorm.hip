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
// consecutive elements each, piece k of lane l at 8 (l + k LPR).
#include <algorithm>

#include "epilogue.hpp"
#include "step_launch.hpp"

namespace orda {

// ------------------------------------------------------------- dropout
// One piece a thread: 256 threads 2048 elements, as clipping has it.
template <class T, bool RES>
__global__ __launch_bounds__(256) void k_dropout(DropoutParams P, int64_t per_row, int64_t pieces) {
  const uint64_t seed = seed_of(P.drop);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
    int64_t row = 0, k = i;
    if (P.rows > 1) {
      row = pieces <= 0xffffffffll ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row;
      k -= row * per_row;
    }
    const int64_t c = k * 8;
    const int cnt = (int)lmin(8, P.cols - c);
    float x[8], r[8];
    ld_row<T, 8>(static_cast<const T*>(P.x) + row * P.ldx + c, x, cnt);
    if constexpr (RES) ld_row<T, 8>(static_cast<const T*>(P.residual) + row * P.ldr + c, r, cnt);
    const int64_t index = row * P.cols + c;
    const uint32_t m = keep8(index, seed, P.drop.site, P.drop.threshold);
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // (a dropped infinity or NaN leaves nothing)
      x[e] = (m >> e) & 1 ? x[e] * P.drop.factor : 0.0f;
      if constexpr (RES) x[e] += r[e];
    }
    st_row<T, 8>(static_cast<T*>(P.y) + index, x, cnt);
  }
}

template <class T>
static hipError_t dropout_go(const DropoutParams& P, hipStream_t s) {
  const int64_t per_row = (P.cols + 7) / 8, pieces = per_row * P.rows;
  // (a launch has fewer than 2^32 threads; past them a thread takes several pieces)
  const unsigned groups = (unsigned)std::min<int64_t>((pieces + 255) / 256, 1 << 23);
  if (P.residual) hipLaunchKernelGGL((k_dropout<T, true>), dim3(groups), dim3(256), 0, s, P, per_row, pieces);
  else hipLaunchKernelGGL((k_dropout<T, false>), dim3(groups), dim3(256), 0, s, P, per_row, pieces);
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
// v of all lanes of the row's LPR added up, in every lane; `red`: one float per
// wave, another one for every call between two barriers.
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, false));   // lane ^ 1
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, false));   // lane ^ 2
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, false));  // the other quad of 8
  if constexpr (LPR > 8) {
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, false));  // the other 8 of 16
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
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
    __syncthreads();
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
template <class T>
__device__ __forceinline__ void drop_piece(float (&x)[8], const float* r, int64_t index, const DropParams& d, uint64_t seed) {
  if (d.threshold) {
    const uint32_t m = keep8(index, seed, d.site, d.threshold);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (m >> e) & 1 ? x[e] * d.factor : 0.0f;
  }
  if (r)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += r[e];
}

// ------------------------------------------------------------- forward
template <class T, class W, int LPR, int NP>
__global__ __launch_bounds__(group_threads(LPR)) void k_layer_norm(LayerNormParams P) {
  constexpr int kRows = group_threads(LPR) / LPR, kWaves = group_threads(LPR) / 64;
  __shared__ float red[2][2][kWaves];
  const int lane = threadIdx.x % LPR;
  const uint64_t seed = P.drop.threshold ? seed_of(P.drop) : 0;
  const float n_cols = (float)P.cols;
  int cnt[NP];
  RawRow<W, 8> w[NP], b[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int64_t c = 8 * (int64_t)(lane + k * LPR);
    cnt[k] = (int)(P.cols - c < 0 ? 0 : lmin(8, P.cols - c));
    w[k].load(static_cast<const W*>(P.weight) + c, cnt[k]);
    if (P.bias) b[k].load(static_cast<const W*>(P.bias) + c, cnt[k]);
  }
  int turn = 0;
  const int64_t steps = (P.rows + kRows - 1) / kRows;
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x, turn ^= 1) {
    const int64_t row = step * kRows + threadIdx.x / LPR;
    const bool live = row < P.rows;
    float v[NP][8], sum[1] = {0.0f};
    RawRow<T, 8> x[NP], r[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int n = live ? cnt[k] : 0;
      const int64_t c = 8 * (int64_t)(lane + k * LPR);
      x[k].load(static_cast<const T*>(P.x) + row * P.ldx + c, n);
      if (P.residual) r[k].load(static_cast<const T*>(P.residual) + row * P.ldr + c, n);
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int64_t c = 8 * (int64_t)(lane + k * LPR);
      float add[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[k][e] = x[k][e];
        add[e] = P.residual ? r[k][e] : 0.0f;
      }
      if (live && cnt[k]) drop_piece<T>(v[k], P.residual ? add : nullptr, row * P.cols + c, P.drop, seed);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0] += e < cnt[k] ? v[k][e] : 0.0f;
    }
    row_sums<LPR>(sum, red[turn][0]);
    const float mean = sum[0] / n_cols;
    sum[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = e < cnt[k] ? v[k][e] - mean : 0.0f;
        sum[0] = fmaf(d, d, sum[0]);
      }
    row_sums<LPR>(sum, red[turn][1]);
    const float rstd = 1.0f / sqrtf(sum[0] / n_cols + P.eps);
    if (!live) continue;
    if (P.stats && lane == 0) *reinterpret_cast<float2*>(P.stats + 2 * row) = make_float2(mean, rstd);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      if (!cnt[k]) continue;
      const int64_t at = row * P.cols + 8 * (int64_t)(lane + k * LPR);
      if (P.s) st_row<T, 8>(static_cast<T*>(P.s) + at, v[k], cnt[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float h = (v[k][e] - mean) * rstd;
        v[k][e] = P.bias ? fmaf(h, w[k][e], b[k][e]) : h * w[k][e];
      }
      st_row<T, 8>(static_cast<T*>(P.y) + at, v[k], cnt[k]);
    }
  }
}

// Rows longer than a workgroup's registers hold: 1024 threads read the row three
// times (the second and third time from the caches).
template <class T, class W>
__global__ __launch_bounds__(1024) void k_layer_norm_long(LayerNormParams P) {
  __shared__ float red[2][2][16];
  const uint64_t seed = P.drop.threshold ? seed_of(P.drop) : 0;
  const float n_cols = (float)P.cols;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x, turn ^= 1) {
    auto piece = [&](int64_t c, float (&v)[8], int n) {
      float r[8];
      ld_row<T, 8>(static_cast<const T*>(P.x) + row * P.ldx + c, v, n);
      if (P.residual) ld_row<T, 8>(static_cast<const T*>(P.residual) + row * P.ldr + c, r, n);
      drop_piece<T>(v, P.residual ? r : nullptr, row * P.cols + c, P.drop, seed);
    };
    float sum[1] = {0.0f}, v[8];
    for (int64_t c = 8 * threadIdx.x; c < P.cols; c += 8192) {
      const int n = (int)lmin(8, P.cols - c);
      piece(c, v, n);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0] += e < n ? v[e] : 0.0f;
      if (P.s) st_row<T, 8>(static_cast<T*>(P.s) + row * P.cols + c, v, n);
    }
    row_sums<1024>(sum, red[turn][0]);
    const float mean = sum[0] / n_cols;
    sum[0] = 0.0f;
    for (int64_t c = 8 * threadIdx.x; c < P.cols; c += 8192) {
      const int n = (int)lmin(8, P.cols - c);
      piece(c, v, n);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = e < n ? v[e] - mean : 0.0f;
        sum[0] = fmaf(d, d, sum[0]);
      }
    }
    row_sums<1024>(sum, red[turn][1]);
    const float rstd = 1.0f / sqrtf(sum[0] / n_cols + P.eps);
    if (P.stats && threadIdx.x == 0) *reinterpret_cast<float2*>(P.stats + 2 * row) = make_float2(mean, rstd);
    for (int64_t c = 8 * threadIdx.x; c < P.cols; c += 8192) {
      const int n = (int)lmin(8, P.cols - c);
      float w[8], b[8];
      piece(c, v, n);
      ld_row<W, 8>(static_cast<const W*>(P.weight) + c, w, n);
      if (P.bias) ld_row<W, 8>(static_cast<const W*>(P.bias) + c, b, n);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float h = (v[e] - mean) * rstd;
        v[e] = P.bias ? fmaf(h, w[e], b[e]) : h * w[e];
      }
      st_row<T, 8>(static_cast<T*>(P.y) + row * P.cols + c, v, n);
    }
  }
}

// ------------------------------------------------------------- backward
// ds' of one piece to dr, and what dropout leaves of it to dx.
template <class T>
__device__ __forceinline__ void grad_piece(const LayerNormGradParams& P, float (&t)[8], int64_t at, int n, uint32_t kept) {
  if (P.dr) st_row<T, 8>(static_cast<T*>(P.dr) + at, t, n);
  if (!P.dx) return;
  if (P.drop.threshold)
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (kept >> e) & 1 ? t[e] * P.drop.factor : 0.0f;
  st_row<T, 8>(static_cast<T*>(P.dx) + at, t, n);
}

// AGAIN: s is computed again from x and the residual, in fp32.  fp32 parameters
// beside 16-bit tensors get gradients of fp32's precision so, for 2 more bytes
// read of 16 to 20; from s as it was rounded dw is off by half a step of the
// 16-bit type (2e-4 of its norm in fp16, 2.4e-3 in bf16, where 1.7e-3 come from
// its own rounding).
template <class T, class W, int LPR, int NP, bool AGAIN>
__global__ __launch_bounds__(group_threads(LPR)) void k_layer_norm_grad(LayerNormGradParams P) {
  constexpr int kRows = group_threads(LPR) / LPR, kWaves = group_threads(LPR) / 64;
  __shared__ float red[2][2 * kWaves];
  const int lane = threadIdx.x % LPR;
  const uint64_t seed = P.drop.threshold ? seed_of(P.drop) : 0;
  const float n_cols = (float)P.cols;
  int cnt[NP];
  RawRow<W, 8> w[NP];
  float dw[NP][8], db[NP][8];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int64_t c = 8 * (int64_t)(lane + k * LPR);
    cnt[k] = (int)(P.cols - c < 0 ? 0 : lmin(8, P.cols - c));
    w[k].load(static_cast<const W*>(P.weight) + c, cnt[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[k][e] = db[k][e] = 0.0f;
  }
  // a row's pieces are loaded while the row before is worked on
  struct Loaded {
    RawRow<T, 8> s[NP], dy[NP], ds[NP], r[AGAIN ? NP : 1];
    float2 st;
  };
  auto load = [&](int64_t row, Loaded& q) {
    const bool live = row < P.rows;
    q.st = live ? *reinterpret_cast<const float2*>(P.stats + 2 * row) : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int n = live ? cnt[k] : 0;
      const int64_t c = 8 * (int64_t)(lane + k * LPR);
      q.s[k].load(static_cast<const T*>(P.s) + row * P.ld_s + c, n);
      if constexpr (AGAIN) q.r[k].load(static_cast<const T*>(P.residual) + row * P.ldr + c, n);
      q.dy[k].load(static_cast<const T*>(P.dy) + row * P.ldy + c, n);
      if (P.ds) q.ds[k].load(static_cast<const T*>(P.ds) + row * P.ldd + c, n);
    }
  };
  const int64_t steps = (P.rows + kRows - 1) / kRows;
  int turn = 0;
  Loaded next;
  load((int64_t)blockIdx.x * kRows + threadIdx.x / LPR, next);
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x, turn ^= 1) {
    const int64_t row = step * kRows + threadIdx.x / LPR;
    const Loaded q = next;
    if (step + gridDim.x < steps) load(row + (int64_t)gridDim.x * kRows, next);
    const bool live = row < P.rows;
    float h[NP][8], sum[2] = {0.0f, 0.0f};
    uint32_t kept[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      kept[k] = 0xff;
      if (P.drop.threshold && live && cnt[k]) kept[k] = keep8(row * P.cols + 8 * (int64_t)(lane + k * LPR), seed, P.drop.site, P.drop.threshold);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float s = q.s[k][e];
        if constexpr (AGAIN) s = ((kept[k] >> e) & 1 ? s * P.drop.factor : 0.0f) + q.r[k][e];
        h[k][e] = e < cnt[k] ? (s - q.st.x) * q.st.y : 0.0f;
        const float g = q.dy[k][e], gw = g * w[k][e];
        sum[0] += gw;
        sum[1] = fmaf(gw, h[k][e], sum[1]);
        dw[k][e] = fmaf(g, h[k][e], dw[k][e]);
        db[k][e] += g;
      }
    }
    if (P.dx || P.dr) {
      row_sums<LPR>(sum, red[turn]);
      const float mg = sum[0] / n_cols, mgh = sum[1] / n_cols;
      if (live)
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          if (!cnt[k]) continue;
          float t[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            t[e] = q.st.y * (fmaf(q.dy[k][e], w[k][e], -mg) - h[k][e] * mgh);
            if (P.ds) t[e] += q.ds[k][e];
          }
          grad_piece<T>(P, t, row * P.cols + 8 * (int64_t)(lane + k * LPR), cnt[k], kept[k]);
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
    const int64_t c = 8 * (int64_t)(lane + k * LPR);
    if (!cnt[k]) continue;
    st_row<float, 8>(out + c, dw[k], cnt[k]);
    st_row<float, 8>(out + P.cols + c, db[k], cnt[k]);
  }
}

// Long rows: sums of dw and db in the workgroup's own rows of `partial`, which
// each thread reads and writes at its own columns only.
template <class T, class W>
__global__ __launch_bounds__(1024) void k_layer_norm_grad_long(LayerNormGradParams P) {
  __shared__ float red[2][32];
  const uint64_t seed = P.drop.threshold ? seed_of(P.drop) : 0;
  const float n_cols = (float)P.cols;
  float* part = P.partial ? P.partial + (int64_t)blockIdx.x * 2 * P.cols : nullptr;
  int turn = 0;
  bool first = true;
  for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x, turn ^= 1, first = false) {
    const float2 st = *reinterpret_cast<const float2*>(P.stats + 2 * row);
    float sum[2] = {0.0f, 0.0f}, s[8], g[8], w[8];
    uint32_t kept = 0xff;
    auto piece = [&](int64_t c, int n) {
      ld_row<T, 8>(static_cast<const T*>(P.s) + row * P.ld_s + c, s, n);
      if (P.drop.threshold) kept = keep8(row * P.cols + c, seed, P.drop.site, P.drop.threshold);
      if (P.residual) {
        float r[8];
        ld_row<T, 8>(static_cast<const T*>(P.residual) + row * P.ldr + c, r, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = ((kept >> e) & 1 ? s[e] * P.drop.factor : 0.0f) + r[e];
      }
      ld_row<T, 8>(static_cast<const T*>(P.dy) + row * P.ldy + c, g, n);
      ld_row<W, 8>(static_cast<const W*>(P.weight) + c, w, n);
    };
    for (int64_t c = 8 * threadIdx.x; c < P.cols; c += 8192) {
      const int n = (int)lmin(8, P.cols - c);
      piece(c, n);
      float a[8], b[8];
      if (part) {
        ld_row<float, 8>(part + c, a, first ? 0 : n);
        ld_row<float, 8>(part + P.cols + c, b, first ? 0 : n);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float h = e < n ? (s[e] - st.x) * st.y : 0.0f;
        sum[0] = fmaf(g[e], w[e], sum[0]);
        sum[1] = fmaf(g[e] * w[e], h, sum[1]);
        a[e] = fmaf(g[e], h, a[e]);
        b[e] += g[e];
      }
      if (part) {
        st_row<float, 8>(part + c, a, n);
        st_row<float, 8>(part + P.cols + c, b, n);
      }
    }
    if (!P.dx && !P.dr) continue;
    row_sums<1024>(sum, red[turn]);
    const float mg = sum[0] / n_cols, mgh = sum[1] / n_cols;
    for (int64_t c = 8 * threadIdx.x; c < P.cols; c += 8192) {
      const int n = (int)lmin(8, P.cols - c);
      piece(c, n);
      float t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = st.y * (fmaf(g[e], w[e], -mg) - (s[e] - st.x) * st.y * mgh);
      if (P.ds) {
        ld_row<T, 8>(static_cast<const T*>(P.ds) + row * P.ldd + c, s, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] += s[e];
      }
      grad_piece<T>(P, t, row * P.cols + c, n, kept);
    }
  }
}

// dw and db: 64 columns a workgroup, its 16 waves every 16th of the groups.
template <class W>
__global__ __launch_bounds__(1024) void k_layer_norm_params(const float* partial, int64_t groups, int64_t cols, W* dw, W* db) {
  __shared__ float join[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  float v = 0.0f;
  if (c < cols)
    for (int64_t g = wave; g < groups; g += 16) v += partial[(2 * g + blockIdx.y) * cols + c];
  join[wave][lane] = v;
  __syncthreads();
  if (wave || c >= cols) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v += join[i][lane];
  out[c] = from_f32<W>(v);
}

// ------------------------------------------------------------- launches
// f(LPR, NP) of a row length; (0, 0): the long kernels.
template <class F>
static hipError_t for_width(int64_t cols, const F& f) {
  using std::integral_constant;
#define ORDA_ROW(L, N) f(integral_constant<int, L>{}, integral_constant<int, N>{})
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

int64_t layer_norm_groups(int64_t rows, int64_t cols) {
  const int64_t steps = (rows + rows_per_group(cols) - 1) / rows_per_group(cols);
  return std::min<int64_t>(steps, threads_of(cols) == 256 ? 512 : 256);
}

template <class T, class W>
static hipError_t norm_go(const LayerNormParams& P, hipStream_t s) {
  const int64_t steps = (P.rows + rows_per_group(P.cols) - 1) / rows_per_group(P.cols);
  const unsigned groups = (unsigned)std::min<int64_t>(steps, threads_of(P.cols) == 256 ? 2048 : 512);
  return for_width(P.cols, [&](auto l, auto n) {
    constexpr int L = decltype(l)::value, N = decltype(n)::value;
    if constexpr (L == 0) hipLaunchKernelGGL((k_layer_norm_long<T, W>), dim3(groups), dim3(1024), 0, s, P);
    else hipLaunchKernelGGL((k_layer_norm<T, W, L, N>), dim3(groups), dim3(group_threads(L)), 0, s, P);
    return hipGetLastError();
  });
}
template <class T, class W>
static hipError_t norm_grad_go(const LayerNormGradParams& P, hipStream_t s) {
  const unsigned groups = (unsigned)layer_norm_groups(P.rows, P.cols);
  return for_width(P.cols, [&](auto l, auto n) {
    constexpr int L = decltype(l)::value, N = decltype(n)::value;
    if constexpr (L == 0) hipLaunchKernelGGL((k_layer_norm_grad_long<T, W>), dim3(groups), dim3(1024), 0, s, P);
    else if constexpr (sizeof(T) < sizeof(W)) {
      if (P.residual) hipLaunchKernelGGL((k_layer_norm_grad<T, W, L, N, true>), dim3(groups), dim3(group_threads(L)), 0, s, P);
      else hipLaunchKernelGGL((k_layer_norm_grad<T, W, L, N, false>), dim3(groups), dim3(group_threads(L)), 0, s, P);
    } else hipLaunchKernelGGL((k_layer_norm_grad<T, W, L, N, false>), dim3(groups), dim3(group_threads(L)), 0, s, P);
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
