// ring_op.hpp -- the large 16-bit products of orda_linear_* and orda_ffn_* on
// the four-wave ring engine (ring16.hpp: 256 x 256 tiles, one persistent
// workgroup per CU), with an epilogue functor (epilogue.hpp).
//
// The engine leaves 256 accumulators per lane in AGPRs.  An epilogue is much
// code per element (an activation and its branch), so the accumulators go
// through LDS: 16 rows x 128 columns of a wave at a time into the ring slot
// that is free at a tile's end, from where a lane takes 8 consecutive columns
// of one row in a loop that is not unrolled: the code is there 8 times instead
// of 32, and memory sees 128 contiguous bytes of a row (8 lanes x 16 bytes).
// 16-byte chunk c of row r lies at c ^ r: neither the writes (16 rows of a
// chunk) nor the reads (16 chunks of a row) meet on a bank.
#pragma once
#include "ring16.hpp"
#include "tile16.hpp"

namespace orda {

template <class T, int LA, int LB, class Epi>
__global__ __launch_bounds__(kThreads4, 1) void k_ring(TileParams P, Epi E0) {
  constexpr bool DUAL = Epi::kDual;
  static_assert(LA == LB || (LA == KMAJ && LB == MNMAJ), "K/K, K/MN or MN/MN");
  static_assert(!DUAL || (LB == KMAJ && !Epi::kLight), "two weights are K-major, and nothing is loaded for them");
  __shared__ __attribute__((aligned(16))) char lds[kLds4Bytes];
  Acc16 acc;
  zero_acc16(acc);
  const int tiles = P.tiles_m * P.tiles_n;
  const int total = tiles * P.splits;
  const int grid = gridDim.x;
  const int b = xcd_order(blockIdx.x, grid);
  const int ntiles = b < total ? (total - 1 - b) / grid + 1 : 0;
  const T* A = static_cast<const T*>(P.A);
  const T* B = static_cast<const T*>(P.B);
  const T* B1 = static_cast<const T*>(P.B1);
  struct TI {
    int64_t m0, n0;
    int split, second, kb;
    KOp4 a, b, b1;
  };
  auto tile_info = [&](int i) {
    const int t_all = b + (i < ntiles ? i : 0) * grid;
    TI x;
    x.split = t_all / tiles;
    const int t = t_all - x.split * tiles;
    constexpr int G = 8;
    const int band = t / (G * P.tiles_n);
    const int first_m = band * G;
    const int gm = min(P.tiles_m - first_m, G);
    const int rem = t % (G * P.tiles_n);
    int tm = first_m + rem % gm;
    x.second = 0;
    if constexpr (LA == MNMAJ) {
      if (P.pair > 0 && tm >= P.tiles_m / 2) {
        x.second = 1;
        tm -= P.tiles_m / 2;
      }
    }
    x.m0 = (int64_t)tm * 256;
    x.n0 = (int64_t)(rem / gm) * (DUAL ? 128 : 256);
    const int64_t kb = (int64_t)x.split * P.kps;
    x.kb = (int)kb;
    if constexpr (LA == KMAJ) {
      x.a = kop4(A + x.m0 * P.lda + kb, P.lda, P.M - x.m0);
    } else {
      const int64_t klen = lmin(P.K - kb, P.kps);
      x.a = kop4_mn(A + kb * P.lda + x.m0 + (x.second ? P.pair : 0), P.lda, klen, P.M - x.m0);
      x.b = kop4_mn(B + kb * P.ldb + x.n0, P.ldb, klen, P.N - x.n0);
    }
    if constexpr (DUAL) {
      x.b = kop4_split(B + x.n0 * P.ldb + kb, P.N - x.n0, B1 + x.n0 * P.ldb + kb, P.N - x.n0, P.ldb);
    } else if constexpr (LB == KMAJ) {
      x.b = kop4(B + x.n0 * P.ldb + kb, P.ldb, P.N - x.n0);
    } else if constexpr (LA == KMAJ) {
      // K rows [0, kseg) from B and the rest from B1, both addressed by the K
      // row within the split (the second base lies kseg rows before B1)
      const int64_t klen = lmin(P.K - kb, P.kps);
      x.b = kop4_mn(B + kb * P.ldb + x.n0, P.ldb, lmin(P.kval - kb, klen), P.N - x.n0);
      x.b1 = x.b;
      if (B1) x.b1 = kop4_mn(B1 + (kb - P.kseg) * P.ldb + x.n0, P.ldb, lmin(P.kseg + P.kval - kb, klen), P.N - x.n0);
    }
    return x;
  };
  auto opnd = [&](const TI& x, int op, int kd) {
    if constexpr (LA == KMAJ && LB == MNMAJ) return op == 0 ? x.a : (x.kb + kd * 64 < P.kseg ? x.b : x.b1);
    else return op == 0 ? x.a : x.b;
  };
  auto epilogue = [&](int, const TI& x, Acc16& c, char* slot) __attribute__((always_inline)) {
    const int lane = opaque_lane();
    const int wm = w4_m(), wn = w4_n();
    Epi E = E0.at(x.split);
    if constexpr (LA == MNMAJ) {
      if (x.second) E = E.second();
    }
    E = E.tile(x.m0, x.n0);
    char* buf = slot + wave_id() * 8192;
    const int rows = (int)lmin(P.M - x.m0, 256), cols = (int)lmin(E.cols, 256);
    const int mw = wm * 128;
    constexpr int kIt = DUAL ? 2 : 4;
    struct Item {
      int m, row, g, col, cnt;
      bool live;
    };
    auto item = [&](int mb, int it) __attribute__((always_inline)) {
      const int i = it * 64 + lane;
      Item q;
      q.row = DUAL ? i >> 3 : i >> 4;
      q.g = DUAL ? i & 7 : i & 15;
      q.col = (q.g >> 3) * 128 + wn * 64 + (q.g & 7) * 8;
      q.m = mw + mb * 16 + q.row;
      q.cnt = min(cols - q.col, 8);
      q.live = q.m < rows && q.cnt > 0;
      return q;
    };
    auto dump = [&](int mb) __attribute__((always_inline)) {
      const int r = lane & 15;
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) {
        const int ch = nb * 4 + (lane >> 4);
        float4 v;
        v.x = acc16_get(c[mb][nb], 0);
        v.y = acc16_get(c[mb][nb], 1);
        v.z = acc16_get(c[mb][nb], 2);
        v.w = acc16_get(c[mb][nb], 3);
        *reinterpret_cast<float4*>(buf + r * 512 + ((ch ^ r) << 4)) = v;
      }
    };
    auto take = [&](int row, int g, float (&v)[8]) __attribute__((always_inline)) {
      const float4 a = *reinterpret_cast<const float4*>(buf + row * 512 + (((2 * g) ^ row) << 4));
      const float4 d = *reinterpret_cast<const float4*>(buf + row * 512 + (((2 * g + 1) ^ row) << 4));
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = d.x; v[5] = d.y; v[6] = d.z; v[7] = d.w;
    };
    typedef typename Epi::template Pre<8> Pre;
    if constexpr (Epi::kLight) {
      // little code per element: all unrolled, each item's loads two row blocks
      // (eight items) ahead of their use.  dh and its epilogue (8192 tokens,
      // 4096 x 14336: the product alone 650 us) take 910 us, with the loads one
      // block ahead 1033, where they are used 1070.
      constexpr int kAhead = 2;
      Pre p[kAhead][kIt];
      // (items outside the tile's valid part load from its last row or columns)
      auto fetch = [&](int mb, int it) __attribute__((always_inline)) {
        const Item q = item(mb, it);
        p[mb % kAhead][it] = E.template pre<8>(min(q.m, rows - 1), min(q.col, cols - 8), 8);
      };
#pragma unroll
      for (int mb = 0; mb < kAhead; ++mb)
#pragma unroll
        for (int it = 0; it < kIt; ++it) fetch(mb, it);
#pragma unroll
      for (int mb = 0; mb < 8; ++mb) {
        dump(mb);
#pragma unroll
        for (int it = 0; it < kIt; ++it) {
          const Item q = item(mb, it);
          float v[8];
          take(q.row, q.g, v);
          const Pre now = p[mb % kAhead][it];
          if (mb + kAhead < 8) fetch(mb + kAhead, it);
          if (q.live) E(q.m, q.col, v, q.cnt, now, {});
        }
      }
    } else {
      // much code per element: a loop over a row block's items, with the loads
      // of the next block's items in flight; a lane has the same columns in all
      Pre p[2][kIt];
      auto fetch = [&](int mb) __attribute__((always_inline)) {
#pragma unroll
        for (int it = 0; it < kIt; ++it) {
          const Item q = item(mb, it);
          if (q.live) p[mb & 1][it] = E.template pre<8>(q.m, q.col, q.cnt);
        }
      };
      const Item first = item(0, 0);
      const auto col = E.template col<8>(first.col, first.cnt);
      fetch(0);
#pragma unroll
      for (int mb = 0; mb < 8; ++mb) {
        if (mb < 7) fetch(mb + 1);
        dump(mb);
#pragma unroll 1
        for (int it = 0; it < kIt; ++it) {
          const Item q = item(mb, it);
          float v[8];
          take(q.row, q.g, v);
          if constexpr (DUAL) {
            float u[8];
            take(q.row, q.g + 8, u);
            if (q.live) E(q.m, q.col, v, u, q.cnt, p[mb & 1][0], col);
          } else {
            Pre now = p[mb & 1][0];
            if (it == 1) now = p[mb & 1][1];
            if (it == 2) now = p[mb & 1][2];
            if (it == 3) now = p[mb & 1][3];
            if (q.live) E(q.m, q.col, v, q.cnt, now, col);
          }
        }
      }
    }
    tile_barrier();  // (the slot's next DMA may start once every wave has read its part)
  };
  pipeline16<T, LA, LB, true, true, true>(acc, lds, ntiles, P.kps, P.lda, P.ldb, tile_info, opnd, epilogue);
}

}  // namespace orda
