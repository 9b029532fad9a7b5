// op_kernels.hpp -- launchers of the projection's and the feed-forward block's
// kernels, instantiated per dtype by k_op_*.hip.
#pragma once
#include "op_launch.hpp"
#include "ring_op.hpp"

namespace orda {

// The projection's backward pass in front of its products: dz = dy act'(z) and
// the column sums of dz, one pass over dy and the kept derivative.  dz is rounded
// to T, being an operand of the matrix cores next; the sums take it unrounded.  A
// wave takes 1 KiB (64 lanes x 16 bytes) of a row, the four waves of a workgroup
// alternate rows; bias gradients are summed per workgroup and added up by
// k_colsum, in a fixed order.  Bound by memory.
template <class T>
__global__ __launch_bounds__(256) void k_dz(DzParams P) {
  constexpr int W = 16 / (int)sizeof(T);
  __shared__ float red[3][64][W];
  const int w = wave_id(), lane = threadIdx.x & 63;
  const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * W;
  const int64_t r0 = (int64_t)blockIdx.y * P.rows_per_block, r1 = lmin(P.rows, r0 + P.rows_per_block);
  const int64_t left = P.cols - c;
  const int cnt = left <= 0 ? 0 : (left >= W ? W : (int)left);
  const T* dy = static_cast<const T*>(P.dy);
  T* dz = static_cast<T*>(P.dz);
  float sum[W];
#pragma unroll
  for (int e = 0; e < W; ++e) sum[e] = 0.f;
  if (c < P.ldz) {
#pragma unroll 4
    for (int64_t r = r0 + w; r < r1; r += 4) {  // (four rows' loads in flight)
      float g[W];
      ld_row<T, W>(dy + r * P.ldy + c, g, cnt);
      if (P.d.hi) {
        Kept<T, W> k;
        k.load(P.d.template from<T>(r * P.ldz + c), 0);  // (rows padded to ldz, a multiple of W)
#pragma unroll
        for (int e = 0; e < W; ++e) g[e] = e < cnt ? g[e] * k[e] : 0.f;
      }
      if (dz) st_row<T, W>(dz + r * P.ldz + c, g, W);
#pragma unroll
      for (int e = 0; e < W; ++e) sum[e] += g[e];
    }
  }
  if (!P.partial) return;
  if (w > 0)
#pragma unroll
    for (int e = 0; e < W; ++e) red[w - 1][lane][e] = sum[e];
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int e = 0; e < W; ++e)
    if (e < cnt) P.partial[(int64_t)blockIdx.y * P.cols + c + e] = ((sum[e] + red[0][lane][e]) + red[1][lane][e]) + red[2][lane][e];
}

// 64 columns per workgroup; 16 waves share the blocks, so that a thread's loads
// are few and in flight together (bound by their latency: with 4 waves the sum
// of 128 x 4096 partials took 10.7 us).
template <class T>
__global__ __launch_bounds__(1024) void k_colsum(const float* __restrict__ partial, int64_t blocks, int64_t cols, T* out) {
  __shared__ float red[15][64];
  const int w = wave_id(), lane = threadIdx.x & 63;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < cols) {
    const float* p = partial + c;
#pragma unroll 8
    for (int64_t b = w; b < blocks; b += 16) s += p[b * cols];
  }
  if (w > 0) red[w - 1][lane] = s;
  __syncthreads();
  if (w > 0 || c >= cols) return;
#pragma unroll
  for (int i = 0; i < 15; ++i) s += red[i][lane];
  out[c] = from_f32<T>(s);
}

template <class T> hipError_t dz_go(const DzParams& P, hipStream_t s) {
  constexpr int64_t per = 64 * (16 / (int64_t)sizeof(T));
  const dim3 grid((unsigned)((P.ldz + per - 1) / per), (unsigned)((P.rows + P.rows_per_block - 1) / P.rows_per_block));
  hipLaunchKernelGGL((k_dz<T>), grid, dim3(256), 0, s, P);
  return hipGetLastError();
}
template <class T> hipError_t colsum_go(const float* partial, int64_t blocks, int64_t cols, void* out, hipStream_t s) {
  hipLaunchKernelGGL((k_colsum<T>), dim3((unsigned)((cols + 63) / 64)), dim3(1024), 0, s, partial, blocks, cols, static_cast<T*>(out));
  return hipGetLastError();
}

template <class T, class Epi>
hipError_t skinny_go(const TileParams& P, const Epi& E, hipStream_t s) {
  SkinnyParams S{P.A, P.B, P.B1, P.M, P.N, P.K, P.lda, P.ldb};
  hipLaunchKernelGGL((k_skinny<T, Epi>), dim3((unsigned)((E.cols + 15) / 16)), dim3(kSkinnyWaves * 64), 0, s, S, E);
  return hipGetLastError();
}

template <class T, int LA, int LB, class Epi>
hipError_t tile_go(const OpPlan& pl, TileParams P, const Epi& E, hipStream_t s) {
  const int64_t bm = pl.tile / 1000, bn = pl.tile % 1000 / (Epi::kDual ? 2 : 1);
  P.tiles_m = (int)((P.M + bm - 1) / bm) * (P.pair > 0 ? 2 : 1);
  P.tiles_n = (int)((E.cols + bn - 1) / bn);
  P.splits = pl.splits;
  P.kps = pl.kps;
  const unsigned grid = (unsigned)((int64_t)P.tiles_m * P.tiles_n * P.splits);
  if (pl.tile == 128128) hipLaunchKernelGGL((k_tile<T, LA, LB, 128, 128, 2, Epi>), dim3(grid), dim3(256), 0, s, P, E);
  else if (pl.tile == 64128) hipLaunchKernelGGL((k_tile<T, LA, LB, 64, 128, 3, Epi>), dim3(grid), dim3(256), 0, s, P, E);
  else if (pl.tile == 64064) hipLaunchKernelGGL((k_tile<T, LA, LB, 64, 64, 3, Epi>), dim3(grid), dim3(256), 0, s, P, E);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

// One workgroup per CU of the current device (160 KiB of LDS each).
inline int ring_groups() {
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) == hipSuccess && hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0) return n;
    return 256;
  }();
  return cus;
}
template <class T, int LA, int LB, class Epi>
hipError_t ring_go(const OpPlan& pl, TileParams P, const Epi& E, hipStream_t s) {
  const int64_t bn = Epi::kDual ? 128 : 256;
  P.tiles_m = (int)((P.M + 255) / 256) * (P.pair > 0 ? 2 : 1);
  P.tiles_n = (int)((E.cols + bn - 1) / bn);
  P.splits = pl.splits;
  P.kps = pl.kps;
  const int64_t total = (int64_t)P.tiles_m * P.tiles_n * P.splits;
  const unsigned grid = (unsigned)(total < ring_groups() ? total : ring_groups());
  hipLaunchKernelGGL((k_ring<T, LA, LB, Epi>), dim3(grid), dim3(kThreads4), 0, s, P, E);
  return hipGetLastError();
}
template <class T, int LA, int LB, class Epi>
hipError_t any_go(const OpPlan& pl, const TileParams& P, const Epi& E, hipStream_t s) {
  return pl.engine == OP_RING ? ring_go<T, LA, LB>(pl, P, E, s) : tile_go<T, LA, LB>(pl, P, E, s);
}

// The product on tiles, or its K ranges into `part` and their sum.
template <class Epi, class Go>
hipError_t with_splits(const OpPlan& pl, const TileParams& P, const Epi& E, float* part, hipStream_t s, const Go& go) {
  if (pl.splits == 1) return go(E);
  const int64_t cols = (E.cols + 3) / 4 * 4, ld = Epi::kDual ? 2 * cols : cols, rows = P.M * (P.pair > 0 ? 2 : 1);
  EpiPart<Epi::kDual> Q{part, part + cols, rows * ld, ld, cols, P.M * ld};
  const hipError_t e = go(Q);
  if (e != hipSuccess) return e;
  const int64_t groups = (rows * (cols / 4) + 255) / 256, across = groups < (1 << 22) ? groups : (1 << 22);
  const dim3 grid((unsigned)across, (unsigned)((groups + across - 1) / across));
  hipLaunchKernelGGL((k_part_reduce<Epi>), grid, dim3(256), 0, s, part, pl.splits, rows * ld, ld, P.M, rows, cols, E);
  return hipGetLastError();
}

}  // namespace orda

#define ORDA_INSTANTIATE_OPS16(T)                                                                                  \
  template <> hipError_t launch_op_linear<T>(const OpPlan& pl, int la, int lb, TileParams P, const EpiLinear<T>& E, float* part, hipStream_t s) { \
    if (pl.engine == OP_SKINNY) return la == KMAJ && lb == KMAJ ? skinny_go<T>(P, E, s) : hipErrorInvalidValue;    \
    return with_splits(pl, P, E, part, s, [&](const auto& e) {                                                     \
      if (la == MNMAJ) return any_go<T, MNMAJ, MNMAJ>(pl, P, e, s);                                               \
      if (lb == MNMAJ) return any_go<T, KMAJ, MNMAJ>(pl, P, e, s);                                                \
      return any_go<T, KMAJ, KMAJ>(pl, P, e, s);                                                                  \
    });                                                                                                            \
  }                                                                                                                \
  template <> hipError_t launch_op_gate<T>(const OpPlan& pl, TileParams P, const EpiGate<T>& E, float* part, hipStream_t s) { \
    if (pl.engine == OP_SKINNY) return skinny_go<T>(P, E, s);                                                      \
    return with_splits(pl, P, E, part, s, [&](const auto& e) { return any_go<T, KMAJ, KMAJ>(pl, P, e, s); });     \
  }                                                                                                                \
  template <> hipError_t launch_op_gate_grad<T>(const OpPlan& pl, TileParams P, const EpiGateGrad<T>& E, float* part, hipStream_t s) { \
    return with_splits(pl, P, E, part, s, [&](const auto& e) { return any_go<T, KMAJ, MNMAJ>(pl, P, e, s); });    \
  }                                                                                                                \
  template <> hipError_t launch_dz<T>(const DzParams& P, hipStream_t s) { return dz_go<T>(P, s); }                 \
  template <> hipError_t launch_colsum<T>(const float* p, int64_t b, int64_t c, void* o, hipStream_t s) { return colsum_go<T>(p, b, c, o, s); }
