// tile16.hpp -- products of bf16 / fp16 operands on tiles smaller than the
// ring engine's 256 x 256, for calls whose large tiles would leave most of
// the 256 CUs idle: C = A B^T with A and B each K-major or MN-major, fp32
// accumulators, an epilogue functor (epilogue.hpp), and K split over
// workgroups.
//
// Workgroup: 4 waves (2 x 2), tile BM x BN, K steps of 64 in a ring of NS
// stages that the DMA fills NS - 1 steps ahead (buffer loads into LDS; chunks
// out of range land as zeros).  One barrier per step: after it every wave has
// read the stage that the next DMA overwrites.
//
// LDS, per operand of R rows: K-major R x 128 bytes, chunk c (16 bytes) of row
// r at c ^ ((r / 2) % 8) as in the other engines; MN-major 64 K rows x 2 R
// bytes, chunk c of K row k at c ^ 2 f(k): a transposed read (8 bytes per
// lane) takes K rows 8 g + 0..3 of g = 0, 1 (then 2, 3) at one 32-byte column
// segment, and f(k) = k % 4 + 4 (k / 8 % 2) (R = 128, one K row per 256-byte
// bank line) or k / 2 % 2 + 2 (k / 8 % 2) (R = 64, two) puts the eight on
// different banks.
//
// The MFMAs run swapped (B x A^T): lane l holds row l % 16 of a block and
// columns 4 (l / 16) .. + 3.
#pragma once
#include "epilogue.hpp"

namespace orda {

struct TileParams {
  const void* A;
  const void* B;
  const void* B1;        // dual: the second weight; K-major x MN-major: B's K rows from kseg on
  int64_t M, N, K;       // N: rows of B (of each half when dual)
  int64_t lda, ldb;
  int64_t kseg;          // A's columns [0, kseg) meet B, the rest B1 (a multiple of 64; = K without B1)
  int64_t kval;          // valid K rows of an MN-major B (of each segment)
  int tiles_m, tiles_n, splits;
  int64_t kps;           // K of one split (a multiple of 64)
  int64_t pair;          // > 0: two products side by side, the second with A's columns from here on (MN/MN, one split)
};

template <int R>
__device__ __forceinline__ int mn_f(int k) {
  return R == 128 ? (k & 3) | (((k >> 3) & 1) << 2) : ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
}

// Fragment (8 K values of row row0 + lane % 16, K 32 hf + 8 (lane / 16) ..).
template <class T, int L, int R>
__device__ __forceinline__ typename Traits<T>::Frag tile_frag(const char* t, int row0, int hf, int lane) {
  if constexpr (L == KMAJ) {
    const int r = row0 + (lane & 15);
    return *reinterpret_cast<const typename Traits<T>::Frag*>(t + r * 128 + (((hf * 4 + (lane >> 4)) ^ kswz(r)) << 4));
  } else {
    typedef short s4 __attribute__((ext_vector_type(4)));
    const int k = hf * 32 + 8 * (lane >> 4) + ((lane & 15) >> 2);
    const int m = row0 + 4 * (lane & 3);
    const char* p = t + k * (2 * R) + (((m >> 3) ^ (mn_f<R>(k) << 1)) << 4) + (m & 7) * 2;
    auto rd = [](const char* q) {
      return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)q);
    };
    const s4 lo = rd(p), hi = rd(p + 4 * (2 * R));  // (f(k + 4) = f(k))
    typedef short s8 __attribute__((ext_vector_type(8)));
    const s8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Traits<T>::Frag, both);
  }
}

typedef float f4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f4v mma16(bf16x8 a, bf16x8 b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4v mma16(f16x8 a, f16x8 b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* p, int64_t bytes) {
  const uint64_t u = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  const uint32_t n = __builtin_amdgcn_readfirstlane((uint32_t)(bytes < 0 ? 0 : bytes));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((uint64_t)hi << 32) | lo), (short)0, (int)n, 0x00020000);
}

// One operand's DMA: R rows, NQ = R / 32 chunks per thread and step.
template <class T, int L, int R>
struct TileDma {
  static constexpr int NQ = R / 32;
  uint32_t row, chunk;  // K-major: row of chunk 0; MN-major: K row.  Logical 16-byte chunk
  __device__ __forceinline__ TileDma() {
    const int w = wave_id(), lane = threadIdx.x & 63;
    if constexpr (L == KMAJ) {
      row = (uint32_t)(w * 8 + (lane >> 3));
      chunk = (uint32_t)((lane & 7) ^ kswz((int)row));
    } else if constexpr (R == 128) {
      row = (uint32_t)(w * 4 + (lane >> 4));
      chunk = (uint32_t)((lane & 15) ^ (mn_f<R>((int)row) << 1));
    } else {
      row = (uint32_t)(w * 8 + (lane >> 3));
      chunk = (uint32_t)((lane & 7) ^ (mn_f<R>((int)row) << 1));
    }
  }
  static constexpr int kRowStep = L == KMAJ ? 32 : (R == 128 ? 16 : 32);
  // chunk q of the step at byte k0b of K (K-major; kb the K extent in bytes)
  // or at the resource's first K row (MN-major; cols valid columns)
  __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t r, uint32_t ldb, uint32_t k0b, uint32_t kb, int64_t cols,
                                        int q, char* tile) const {
    uint32_t off;
    if constexpr (L == KMAJ) off = k0b + chunk * 16 < kb ? row * ldb + chunk * 16 + k0b : kOob;
    else off = (int64_t)chunk * 8 < cols ? row * ldb + chunk * 16 : kOob;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(tile + (q * 4 + wave_id()) * 1024),
                                             16, off, (uint32_t)q * kRowStep * ldb, 0, 0);
  }
};

template <class T, int LA, int LB, int BM, int BN, int NS, class Epi>
__global__ __launch_bounds__(256) void k_tile(TileParams P, Epi E0) {
  constexpr bool DUAL = Epi::kDual;
  static_assert(!DUAL || LB == KMAJ, "two weights are K-major");
  constexpr int kA = BM * 128, kB = BN * 128, kStage = kA + kB;
  constexpr int MB = BM / 32, NB = BN / 32;
  using Frag = typename Traits<T>::Frag;
  __shared__ __attribute__((aligned(16))) char lds[NS * kStage];
  const int tiles = P.tiles_m * P.tiles_n;
  const int t_all = xcd_order(blockIdx.x, gridDim.x);
  const int split = t_all / tiles, t = t_all - split * tiles;
  constexpr int G = 8;
  const int band = t / (G * P.tiles_n), first_m = band * G;
  const int gm = min(P.tiles_m - first_m, G), rem = t % (G * P.tiles_n);
  const int64_t m0 = (int64_t)(first_m + rem % gm) * BM;
  const int64_t n0 = (int64_t)(rem / gm) * (DUAL ? BN / 2 : BN);
  const int64_t kb0 = (int64_t)split * P.kps, ke = lmin(P.K, kb0 + P.kps);
  const int nk = (int)((ke - kb0 + 63) / 64);
  const uint32_t ldab = (uint32_t)(P.lda * 2), ldbb = (uint32_t)(P.ldb * 2);
  const char* A = static_cast<const char*>(P.A);
  const char* B = static_cast<const char*>(P.B);
  const char* B1 = static_cast<const char*>(P.B1);
  const TileDma<T, LA, BM> da;
  const TileDma<T, LB, BN> db;

  // K-major resources are fixed: rows from the tile's first one at K = 0
  // (a K extent below 2^30 bytes, checked on the host)
  __amdgpu_buffer_rsrc_t ra = tile_rsrc(A, 0), rb0 = ra, rb1 = ra;
  if constexpr (LA == KMAJ) ra = tile_rsrc(A + m0 * ldab, lmin(P.M - m0, BM) * ldab);
  if constexpr (LB == KMAJ) {
    if constexpr (DUAL) {
      rb0 = tile_rsrc(B + n0 * ldbb, lmin(P.N - n0, BN / 2) * ldbb);
      // (rows BN / 2 .. of the tile are B1's first ones: the base is moved back)
      rb1 = tile_rsrc(B1 + n0 * ldbb, lmin(P.N - n0, BN / 2) * ldbb);
    } else {
      rb0 = tile_rsrc(B + n0 * ldbb, lmin(P.N - n0, BN) * ldbb);
    }
  }
  auto issue = [&](int kt) __attribute__((always_inline)) {
    char* st = lds + (kt % NS) * kStage;
    const bool live = kt < nk;
    const int64_t k0 = kb0 + (int64_t)kt * 64;
    const uint32_t kend = live ? (uint32_t)(ke * 2) : 0u;
    if constexpr (LA == MNMAJ) ra = tile_rsrc(A + k0 * ldab + m0 * 2, live ? lmin(ke - k0, 64) * ldab - m0 * 2 : 0);
    if constexpr (LB == MNMAJ) {
      const bool second = k0 >= P.kseg;
      const int64_t kk = second ? k0 - P.kseg : k0;
      rb0 = tile_rsrc((second ? B1 : B) + kk * ldbb + n0 * 2, live ? lmin(P.kval - kk, 64) * ldbb - n0 * 2 : 0);
    }
#pragma unroll
    for (int q = 0; q < TileDma<T, LA, BM>::NQ; ++q) da.issue(ra, ldab, (uint32_t)(k0 * 2), kend, P.M - m0, q, st);
#pragma unroll
    for (int q = 0; q < TileDma<T, LB, BN>::NQ; ++q) {
      if constexpr (DUAL) {
        constexpr int H = TileDma<T, LB, BN>::NQ / 2;
        const auto r = q < H ? rb0 : rb1;
        uint32_t off = (uint32_t)(k0 * 2) + db.chunk * 16 < kend ? db.row * ldbb + db.chunk * 16 + (uint32_t)(k0 * 2) : kOob;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (__attribute__((address_space(3))) void*)(st + kA + (q * 4 + wave_id()) * 1024), 16, off,
            (uint32_t)(q < H ? q : q - H) * 32u * ldbb, 0, 0);
      } else {
        db.issue(rb0, ldbb, (uint32_t)(k0 * 2), kend, P.N - n0, q, st + kA);
      }
    }
  };
  const int w = wave_id(), wm = w >> 1, wn = w & 1;
  const int lane = threadIdx.x & 63;
  auto brow = [&](int nb) { return (nb / (NB / 2)) * (BN / 2) + wn * (BN / 4) + (nb % (NB / 2)) * 16; };
  f4v acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f4v{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue(s);
  constexpr int kDma = BM / 32 + BN / 32;
  for (int kt = 0; kt < nk; ++kt) {
    wait_vmem<(NS - 2) * kDma>();  // step kt has landed
    tile_barrier();
    issue(kt + NS - 1);  // (the slot of step kt - 1; past the end: zeros, so that the count above holds)
    const char* sa = lds + (kt % NS) * kStage;
    const char* sb = sa + kA;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      Frag a[MB], b[NB];
#pragma unroll
      for (int i = 0; i < MB; ++i) a[i] = tile_frag<T, LA, BM>(sa, wm * (BM / 2) + i * 16, hf, lane);
#pragma unroll
      for (int j = 0; j < NB; ++j) b[j] = tile_frag<T, LB, BN>(sb, brow(j), hf, lane);
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mma16(b[j], a[i], acc[i][j]);
    }
  }
  wait_vmem<0>();  // nothing may land after the waves end

  const Epi E = E0.at(split);
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t m = m0 + wm * (BM / 2) + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < (DUAL ? NB / 2 : NB); ++j) {
      const int64_t n = n0 + brow(j) + 4 * (lane >> 4);
      const int64_t left = E.cols - n;
      const int cnt = left >= 4 ? 4 : (int)left;
      if (m < P.M && cnt > 0) {
        float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        if constexpr (DUAL) {
          const f4v c = acc[i][j + NB / 2];
          float u[4] = {c[0], c[1], c[2], c[3]};
          E(m, n, v, u, cnt);
        } else {
          E(m, n, v, cnt);
        }
      }
    }
  }
}

}  // namespace orda
