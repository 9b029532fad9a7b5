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
// columns 4 (l / 16) .. + 3, until the epilogue.
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
  int64_t pair;          // > 0: two products side by side, the second with A's columns from here on (MN-major A; tiles_m counts both)
};

template <int R>
__device__ __forceinline__ int mn_f(int k) {
  return R >= 128 ? (k & 3) | (((k >> 3) & 1) << 2) : ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
}

// Where a lane reads its fragments of one operand: 8 K values of row
// row0 + lane % 16 at K 32 hf + 8 (lane / 16).., for blocks of 16 rows row0 =
// r0, r0 + 16, .. .  K-major: one address per half, the block's offset an
// immediate.  MN-major: two transposed reads four K rows apart; the block
// enters an exclusive or with the lane's swizzle, so one address per block,
// the half an immediate.
template <class T, int L, int R, int NBLK>
struct TileFrags {
  static constexpr int kHalf = 32 * 2 * R, kFour = 4 * 2 * R;  // MN-major: 32 and 4 K rows on
  uint32_t at[L == KMAJ ? 2 : NBLK];
  template <class Row>
  __device__ __forceinline__ void init(const Row& row0) {
    const int lane = threadIdx.x & 63;
    if constexpr (L == KMAJ) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = lane & 15;
        at[h] = (uint32_t)((row0(0) + r) * 128 + (((h * 4 + (lane >> 4)) ^ kswz(r)) << 4));
      }
    } else {
      const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
      for (int i = 0; i < NBLK; ++i) {
        const int m = row0(i) + 4 * (lane & 3);
        at[i] = (uint32_t)(k * (2 * R) + (((m >> 3) ^ (mn_f<R>(k) << 1)) << 4) + (m & 7) * 2);
      }
    }
  }
  // K-major; off: the block's rows past row0(0)
  __device__ __forceinline__ typename Traits<T>::Frag read(const char* tile, int off, int hf) const {
    static_assert(L == KMAJ, "transposed reads go through tr_read");
    return *reinterpret_cast<const typename Traits<T>::Frag*>(tile + at[hf] + off * 128);
  }
};

// Transposed reads of NB blocks (2 or 4) at LDS addresses a[] + OFF and a[] +
// OFF + FOUR, waited for in the same block.  Assembly, because the compiler
// waits for every DMA in flight before its own transposed read (it cannot tell
// the stages apart): 4096 x 1024 x 4096, K-major x MN-major, took 103 us so.
typedef short tr_s4 __attribute__((ext_vector_type(4)));
typedef short tr_s8 __attribute__((ext_vector_type(8)));
template <int OFF, int FOUR, int NB>
__device__ __forceinline__ void tr_read(const uint32_t (&a)[NB], uint32_t tile, tr_s8 (&o)[NB]) {
  static_assert(NB == 2 || NB == 4, "blocks");
  static_assert(OFF + FOUR < 65536, "ds offset field");
  tr_s4 x[NB][2];
  if constexpr (NB == 2) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
        "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1])
        : "v"(a[0] + tile), "v"(a[1] + tile), "n"(OFF), "n"(OFF + FOUR)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(x[2][0]), "=&v"(x[2][1]),
          "=&v"(x[3][0]), "=&v"(x[3][1])
        : "v"(a[0] + tile), "v"(a[1] + tile), "v"(a[2] + tile), "v"(a[3] + tile), "n"(OFF), "n"(OFF + FOUR)
        : "memory");
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) o[i] = __builtin_shufflevector(x[i][0], x[i][1], 0, 1, 2, 3, 4, 5, 6, 7);
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
  static constexpr int kPer = L == KMAJ ? 8 : R / 8;  // 16-byte chunks of a tile row
  uint32_t row, chunk;  // K-major: row of chunk 0; MN-major: K row.  Logical 16-byte chunk
  __device__ __forceinline__ TileDma() {
    const int i = wave_id() * 64 + (threadIdx.x & 63);
    row = (uint32_t)(i / kPer);
    chunk = (uint32_t)((i % kPer) ^ (L == KMAJ ? kswz((int)row) : mn_f<R>((int)row) << 1));
  }
  static constexpr int kRowStep = 256 / kPer;
  // The thread's offset (chunk q lies q kRowStep rows on, the caller adds them), or
  // past every resource.  K-major: left = bytes of K from the step on;
  // MN-major: left = valid columns.
  __device__ __forceinline__ uint32_t off(uint32_t ldb, int left) const {
    return (int)(chunk * (L == KMAJ ? 16 : 8)) < left ? row * ldb + chunk * 16 : kOob;
  }
  static __device__ __forceinline__ void go(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff, int q, char* tile) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(tile + (q * 4 + wave_id()) * 1024),
                                             16, off, soff, 0, 0);
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
  int tm = first_m + rem % gm;
  const bool second = LA == MNMAJ && P.pair > 0 && tm >= P.tiles_m / 2;
  if (second) tm -= P.tiles_m / 2;
  const int64_t m0 = (int64_t)tm * BM;
  const int64_t n0 = (int64_t)(rem / gm) * (DUAL ? BN / 2 : BN);
  const int64_t kb0 = (int64_t)split * P.kps, ke = lmin(P.K, kb0 + P.kps);
  const int nk = (int)((ke - kb0 + 63) / 64);
  const uint32_t ldab = (uint32_t)(P.lda * 2), ldbb = (uint32_t)(P.ldb * 2);
  const char* A = static_cast<const char*>(P.A) + (second ? P.pair * 2 : 0);
  const char* B = static_cast<const char*>(P.B);
  const char* B1 = static_cast<const char*>(P.B1);
  const TileDma<T, LA, BM> da;
  const TileDma<T, LB, BN> db;

  // Resources of the tile's rows (K-major) or of the split's K rows from the
  // tile's first column on (MN-major), ending where the data does; a step adds
  // a scalar offset.  A split's MN-major K rows span less than 2^30 bytes and
  // a K-major row at most 2^23 (host), so that kOob and a step's offset together
  // stay below 2^32.
  const int64_t klen = ke - kb0;
  __amdgpu_buffer_rsrc_t ra, rb0, rb1;
  if constexpr (LA == KMAJ) ra = tile_rsrc(A + m0 * ldab + kb0 * 2, lmin(P.M - m0, BM) * ldab);
  else ra = tile_rsrc(A + kb0 * ldab + m0 * 2, klen * ldab - m0 * 2);
  rb1 = ra;
  if constexpr (DUAL) {
    rb0 = tile_rsrc(B + n0 * ldbb + kb0 * 2, lmin(P.N - n0, BN / 2) * ldbb);
    rb1 = tile_rsrc(B1 + n0 * ldbb + kb0 * 2, lmin(P.N - n0, BN / 2) * ldbb);
  } else if constexpr (LB == KMAJ) {
    rb0 = tile_rsrc(B + n0 * ldbb + kb0 * 2, lmin(P.N - n0, BN) * ldbb);
  } else {
    // (B1's base lies kseg rows before it: both are addressed by the K row
    // within the split)
    rb0 = tile_rsrc(B + kb0 * ldbb + n0 * 2, lmin(P.kval - kb0, klen) * ldbb - n0 * 2);
    if (B1) rb1 = tile_rsrc(B1 + (kb0 - P.kseg) * (int64_t)ldbb + n0 * 2, lmin(P.kseg + P.kval - kb0, klen) * ldbb - n0 * 2);
  }
  const int seg = (int)lmin((P.kseg - kb0 + 63) / 64, 0x7fffffff);  // B1's first step
  const int kbytes = (int)(klen * 2);
  const int mleft = (int)lmin(P.M - m0, BM), nleft = (int)lmin(P.N - n0, BN);
  const uint32_t offa = da.off(ldab, mleft), offb = db.off(ldbb, nleft);  // (MN-major)
  auto issue = [&](int kt, char* st) __attribute__((always_inline)) {
    const int left = kbytes - kt * 128;  // (past the end: <= 0, zeros; the count of DMAs stays the same)
    {
      const uint32_t o = LA == KMAJ ? da.off(ldab, left) : left > 0 ? offa : kOob;
      const uint32_t so = LA == KMAJ ? (uint32_t)kt * 128u : left > 0 ? (uint32_t)kt * 64u * ldab : 0u;
#pragma unroll
      for (int q = 0; q < TileDma<T, LA, BM>::NQ; ++q)
        da.go(ra, o, so + (uint32_t)(q * TileDma<T, LA, BM>::kRowStep) * ldab, q, st);
    }
    {
      const uint32_t o = LB == KMAJ ? db.off(ldbb, left) : left > 0 ? offb : kOob;
      const uint32_t so = LB == KMAJ ? (uint32_t)kt * 128u : left > 0 ? (uint32_t)kt * 64u * ldbb : 0u;
      constexpr int H = TileDma<T, LB, BN>::NQ / 2;
#pragma unroll
      for (int q = 0; q < TileDma<T, LB, BN>::NQ; ++q) {
        const bool two = DUAL ? q >= H : (LB == MNMAJ && LA == KMAJ && kt >= seg);
        db.go(two ? rb1 : rb0, o,
              so + (uint32_t)((DUAL && q >= H ? q - H : q) * TileDma<T, LB, BN>::kRowStep) * ldbb, q, st + kA);
      }
    }
  };
  const int w = wave_id(), wm = w >> 1, wn = w & 1;
  const int lane = threadIdx.x & 63;
  // B rows (output columns) of a wave's block nb: BN / 2 in a row, dual the same
  // BN / 4 of each half
  auto bofs = [](int nb) { return DUAL ? (nb / (NB / 2)) * (BN / 2) + (nb % (NB / 2)) * 16 : nb * 16; };
  const int wcol = wn * (DUAL ? BN / 4 : BN / 2);
  auto brow = [&](int nb) { return wcol + bofs(nb); };
  TileFrags<T, LA, BM, MB> fa;
  TileFrags<T, LB, BN, NB> fb;
  fa.init([&](int i) { return wm * (BM / 2) + i * 16; });
  fb.init(brow);
  f4v acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f4v{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue(s, lds + s * kStage);
  constexpr int kDma = BM / 32 + BN / 32;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
  int rd = 0, wr = (NS - 1) * kStage;  // the stages of step kt and of step kt + NS - 1
#pragma unroll 1
  for (int kt = 0; kt < nk; ++kt) {
    wait_vmem<(NS - 2) * kDma>();  // step kt has landed
    tile_barrier();
    issue(kt + NS - 1, lds + wr);  // (the stage of step kt - 1)
    const char* sa = lds + rd;
    const char* sb = sa + kA;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      Frag a[MB], b[NB];
      if constexpr (LA == KMAJ) {
#pragma unroll
        for (int i = 0; i < MB; ++i) a[i] = fa.read(sa, i * 16, hf);
      }
      if constexpr (LB == KMAJ) {
#pragma unroll
        for (int j = 0; j < NB; ++j) b[j] = fb.read(sb, bofs(j), hf);
      }
      auto transposed = [&](const auto& f, uint32_t tile, auto& frags, auto half) __attribute__((always_inline)) {
        using FR = std::remove_reference_t<decltype(f)>;
        constexpr int N = sizeof(frags) / sizeof(frags[0]);
        tr_s8 o[N];
        tr_read<decltype(half)::value * FR::kHalf, FR::kFour, N>(f.at, tile, o);
#pragma unroll
        for (int i = 0; i < N; ++i) frags[i] = __builtin_bit_cast(Frag, o[i]);
      };
      auto both = [&](auto half) __attribute__((always_inline)) {
        if constexpr (LB == MNMAJ) transposed(fb, lds0 + rd + kA, b, half);
        if constexpr (LA == MNMAJ) transposed(fa, lds0 + rd, a, half);
      };
      if (hf == 0) both(std::integral_constant<int, 0>{});
      else both(std::integral_constant<int, 1>{});
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mma16(b[j], a[i], acc[i][j]);
    }
    wr = rd;
    rd = rd + kStage == NS * kStage ? 0 : rd + kStage;
  }
  wait_vmem<0>();  // nothing may land after the waves end

  Epi E = E0.at(split);
  if constexpr (LA == MNMAJ) {
    if (second) E = E.second();
  }
  E = E.tile(m0, n0);
  // The accumulators through LDS (each wave its own part of the stages), so that
  // a lane takes 8 consecutive columns of a row and 8 or 4 lanes a row's
  // contiguous bytes, and the epilogue's code is there once: 8192 x 2048 x 4096
  // with gelu and its kept derivative takes 174 us, from the accumulators' own
  // layout (4 columns of 16 rows) it took 219; 48 x 4096 x 11008 gated 32.
  __syncthreads();
  constexpr int kC = BN / 8;  // 16-byte chunks of a wave's row
  char* buf = lds + w * (BM / 2) * (BN / 2) * 4;
  static_assert(4 * (BM / 2) * (BN / 2) * 4 <= NS * kStage, "the accumulators fit the stages");
  auto at = [](int row, int c) {
    return kC == 16 ? row * 256 + ((c ^ (row & 15)) << 4) : row * 128 + ((c ^ ((row >> 1) & 7)) << 4);
  };
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      *reinterpret_cast<f4v*>(buf + at(i * 16 + (lane & 15), j * 4 + (lane >> 4))) = acc[i][j];
  // (the same wave reads them: LDS serves a wave in order)
  constexpr int kG = (DUAL ? kC / 2 : kC) / 2;  // groups of 8 columns in a row (of one half)
  const int g = lane % kG;
  const int n = wcol + g * 8;
  const int64_t left = E.cols - n;
  const int cnt = left >= 8 ? 8 : (int)left;
  if (cnt <= 0) return;
  const auto col = E.template col<8>(n, cnt);
  auto take = [&](int row, int c, float (&v)[8]) __attribute__((always_inline)) {
    const f4v x = *reinterpret_cast<const f4v*>(buf + at(row, c)), y = *reinterpret_cast<const f4v*>(buf + at(row, c + 1));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = x[e];
      v[4 + e] = y[e];
    }
  };
  const int mw = wm * (BM / 2), rows = (int)lmin(P.M - m0, BM);
#pragma unroll 2
  for (int row = lane / kG; row < BM / 2; row += 64 / kG) {
    const int m = mw + row;
    if (m >= rows) break;
    const auto pre = E.template pre<8>(m, n, cnt);
    float v[8];
    take(row, 2 * g, v);
    if constexpr (DUAL) {
      float u[8];
      take(row, kC / 2 + 2 * g, u);
      E(m, n, v, u, cnt, pre, col);
    } else {
      E(m, n, v, cnt, pre, col);
    }
  }
}

}  // namespace orda
