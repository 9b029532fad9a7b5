// tile_s3.hpp -- the fp32 products of orda_linear_* and orda_ffn_* on the
// split-operand engine (split3.hpp has the arithmetic, the tiles and what
// falls back to the native fp32 MFMA), with an epilogue functor
// (epilogue.hpp), two weights side by side (dual: the two halves of a tile's B
// rows) and K in ranges.
#pragma once
#include "epilogue.hpp"
#include "split3.hpp"
#include "tile16.hpp"

namespace orda {

// B row of a wave's block nb.  Dual: blocks of both halves, the same columns.
template <class C, bool DUAL>
__device__ __forceinline__ int s3_brow(int nb, int wn) {
  constexpr int MB = C::MB;
  if constexpr (DUAL) return (nb / (MB / 2)) * (C::kRowsB / 2) + wn * (8 * MB) + (nb % (MB / 2)) * 16;
  else return wn * 16 * MB + nb * 16;
}

template <class C, int LA, int LB, class Epi>
__global__ __launch_bounds__(C::kThreads, C::MB == 4 ? 2 : 3) void k_tile_s3(TileParams P, Epi E0) {
  constexpr bool DUAL = Epi::kDual;
  constexpr int MB = C::MB, RA = C::kRowsA, RB = C::kRowsB, NC = DUAL ? RB / 2 : RB;
  __shared__ __attribute__((aligned(16))) char lds[C::kLds];
  const int tiles = P.tiles_m * P.tiles_n, total = tiles * P.splits;
  const int b0 = xcd_order(blockIdx.x, gridDim.x), grid = gridDim.x;
  const int nt = b0 < total ? (total - 1 - b0) / grid + 1 : 0;
  struct Tile {
    int split;
    bool second;  // a pair's second product
    int64_t m0, n0;
  };
  auto tile_of = [&](int i) {
    const int t_all = b0 + i * grid;
    Tile x;
    x.split = t_all / tiles;
    const int t = t_all - x.split * tiles;
    constexpr int G = 8;
    const int band = t / (G * P.tiles_n), first_m = band * G;
    const int gm = min(P.tiles_m - first_m, G), rem = t % (G * P.tiles_n);
    int tm = first_m + rem % gm;
    x.second = LA == MNMAJ && P.pair > 0 && tm >= P.tiles_m / 2;
    if (x.second) tm -= P.tiles_m / 2;
    x.m0 = (int64_t)tm * RA;
    x.n0 = (int64_t)(rem / gm) * NC;
    return x;
  };
  const float* A = static_cast<const float*>(P.A);
  const float* B = static_cast<const float*>(P.B);
  const float* B1 = static_cast<const float*>(P.B1);
  // (every split takes the steps of a whole one: a short last one reads zeros)
  const int steps = (int)((P.kps + kS3Step - 1) / kS3Step);
  typename std::conditional<LA == KMAJ, S3K<RA, C::kThreads>, S3M<RA>>::type la;
  typename std::conditional<LB == KMAJ, S3K<RB, C::kThreads>, S3M<RB>>::type lb;
  int fi = 0, fs = 0;  // tile and step of the next fetch
  Tile f = tile_of(0);
  auto fetch = [&](int) __attribute__((always_inline)) {
    const int64_t kb = (int64_t)f.split * P.kps, k0 = kb + (int64_t)fs * kS3Step;
    const int64_t left = lmin(P.K, kb + P.kps) - k0;
    if constexpr (LA == KMAJ) la.template load<0, RA * 8 / C::kThreads>(A + f.m0 * P.lda + k0, P.lda, P.M - f.m0, left);
    else la.load(A + (f.second ? P.pair : 0) + k0 * P.lda + f.m0, P.lda, P.M - f.m0, left);
    if constexpr (DUAL) {
      lb.template load<0, 1>(B + f.n0 * P.ldb + k0, P.ldb, P.N - f.n0, left);
      lb.template load<1, 2>(B1 + f.n0 * P.ldb + k0, P.ldb, P.N - f.n0, left);
    } else if constexpr (LB == KMAJ) {
      lb.template load<0, RB * 8 / C::kThreads>(B + f.n0 * P.ldb + k0, P.ldb, P.N - f.n0, left);
    } else {
      const bool second = k0 >= P.kseg;
      const int64_t kk = second ? k0 - P.kseg : k0;
      lb.load((second ? B1 : B) + kk * P.ldb + f.n0, P.ldb, P.N - f.n0, lmin(P.kval - kk, left));
    }
    if (++fs == steps) {
      fs = 0;
      if (++fi < nt) f = tile_of(fi);
    }
  };
  S3Marks marks(lds + 2 * C::kStage);
  int pi = 0, ps = 0;  // tile and step being split
  auto put = [&](char* st) __attribute__((always_inline)) {
    la.store(st);
    lb.store(st + RA * 192);
    marks.big = lb.largest(la.largest(marks.big));
    if (++ps == steps) {
      ps = 0;
      marks.last_put(pi++);
    }
  };
  const int w = wave_id(), wm = w >> 1, wn = w & 1;
  S3Acc<MB> acc;
  s3_zero<MB>(acc);
  auto mul = [&](int, const char* st) __attribute__((always_inline)) {
    s3_mul<C, 0, MB, true>(acc, st + wm * (16 * MB * 64), st + RA * 192, [&](int nb) { return s3_brow<C, DUAL>(nb, wn); });
  };
  int mi = 0, ms = 0;  // tile and step being multiplied
  auto done = [&](int) __attribute__((always_inline)) {
    if (++ms < steps) return;
    ms = 0;
    const Tile x = tile_of(mi++);
    const int ol = opaque_lane();
    const int64_t ml = x.m0 + wm * 16 * MB + (ol & 15);
    if (P.K <= kS3Short || marks.met(mi - 1)) {
      s3_zero<MB>(acc);
      const auto* q = s3_args<TileParams>();
      const float* a = static_cast<const float*>(q->A) + (x.second ? q->pair : 0);
      const float* b = static_cast<const float*>(q->B);
      const float* b1 = static_cast<const float*>(q->B1);
      const int64_t kb = (int64_t)x.split * q->kps;
      auto av = [&](int mb, int64_t k) {
        const int64_t r = ml + mb * 16;
        return r < q->M ? a[LA == KMAJ ? r * q->lda + k : k * q->lda + r] : 0.f;
      };
      auto bv = [&](int nb, int64_t k) {
        int row = s3_brow<C, DUAL>(nb, wn);
        const float* p = b;
        if (DUAL && row >= NC) {
          row -= NC;
          p = b1;
        }
        const int64_t c = x.n0 + row + (ol & 15);
        if (c >= q->N) return 0.f;
        if (LB == KMAJ) return p[c * q->ldb + k];
        const bool second = k >= q->kseg;
        const int64_t kk = second ? k - q->kseg : k;
        return kk < q->kval ? (second ? b1 : b)[kk * q->ldb + c] : 0.f;
      };
      s3_native<C, 0, MB, true>(acc, kb, lmin(q->K, kb + q->kps), av, bv);
    }
    Epi E = E0.at(x.split);
    if constexpr (LA == MNMAJ) {
      if (x.second) E = E.second();
    }
    E = E.tile(x.m0, x.n0);
    const int rows = (int)lmin(P.M - x.m0, RA);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int m = wm * 16 * MB + mb * 16 + (ol & 15);
#pragma unroll
      for (int nb = 0; nb < (DUAL ? MB / 2 : MB); ++nb) {
        const int n = s3_brow<C, DUAL>(nb, wn) + 4 * (ol >> 4);
        const int64_t left = E.cols - n;
        const int cnt = left >= 4 ? 4 : (int)left;
        if (m < rows && cnt > 0) {
          float v[4] = {acc[mb][nb][0], acc[mb][nb][1], acc[mb][nb][2], acc[mb][nb][3]};
          if constexpr (DUAL) {
            float u[4] = {acc[mb][nb + MB / 2][0], acc[mb][nb + MB / 2][1], acc[mb][nb + MB / 2][2], acc[mb][nb + MB / 2][3]};
            epi_apply(E, m, n, v, u, cnt);
          } else {
            epi_apply(E, m, n, v, cnt);
          }
        }
      }
    }
    s3_zero<MB>(acc);
  };
  s3_loop<C>(lds, nt * steps, fetch, put, mul, done);
}

}  // namespace orda
