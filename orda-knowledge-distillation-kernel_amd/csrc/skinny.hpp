// skinny.hpp -- products of at most 16 rows (the tokens of a decoding step)
// with a weight: y[M x N] = x[M x K] W[N x K]^T.  Streaming W once is all the
// work, so nothing is staged: W goes from memory into the matrix cores'
// operand registers, 128 contiguous bytes of a row by 4 lanes.
//
// Workgroup: 16 rows of W (of both weights when dual), K split over its waves
// in blocks of 128 bytes a row, the waves' sums added through LDS in wave
// order.  A lane holds row l % 16 of W and of x (rows past M are zero) and the
// same two 16-byte pieces of K in both (any order of K serves when both
// operands use it), so that 4 lanes read 64 contiguous bytes at a time.
// The result has row (token) l % 16 and columns 4 (l / 16) .. + 3 per lane.
#pragma once
#include "tile16.hpp"

namespace orda {

struct SkinnyParams {
  const void* x;
  const void* w;
  const void* w1;
  int64_t M, N, K, ldx, ldw;
};

// 16 waves of 2 blocks in flight each: 1 token, 2 x 14336 x 4096 and 4096 x
// 14336 weights in bf16: 43.0 and 22.2 us (5.5, 5.3 TB/s); 8 waves of 4 blocks
// 46.2 and 22.7, 4 of 8 46.5 and 25.6.
constexpr int kSkinnyWaves = 16;

// A lane's two pieces of a block, 64 bytes apart; those past K (`left` bytes
// from the first on, a multiple of 16) are zero.
struct Raw32 {
  uint4 v[2];
};
__device__ __forceinline__ Raw32 skinny_load(const char* p) {
  Raw32 r;
  r.v[0] = *reinterpret_cast<const uint4*>(p);
  r.v[1] = *reinterpret_cast<const uint4*>(p + 64);
  return r;
}
__device__ __forceinline__ Raw32 skinny_load(const char* p, int64_t left) {
  Raw32 r;
  r.v[0] = r.v[1] = make_uint4(0, 0, 0, 0);
  if (left > 0) r.v[0] = *reinterpret_cast<const uint4*>(p);
  if (left > 64) r.v[1] = *reinterpret_cast<const uint4*>(p + 64);
  return r;
}
template <class T>
__device__ __forceinline__ void skinny_mma(f4v& c, const Raw32& w, const Raw32& x) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      c = mma16(__builtin_bit_cast(typename Traits<T>::Frag, w.v[i]), __builtin_bit_cast(typename Traits<T>::Frag, x.v[i]), c);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t a[4] = {w.v[i].x, w.v[i].y, w.v[i].z, w.v[i].w}, b[4] = {x.v[i].x, x.v[i].y, x.v[i].z, x.v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    }
  }
}

template <class T, class Epi>
__global__ __launch_bounds__(kSkinnyWaves * 64) void k_skinny(SkinnyParams P, Epi E) {
  constexpr bool DUAL = Epi::kDual;
  constexpr int U = 2;  // blocks in flight per wave and turn
  __shared__ __attribute__((aligned(16))) f4v part[kSkinnyWaves][DUAL ? 2 : 1][64];
  const int w = wave_id(), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t row = n0 + r < P.N ? n0 + r : P.N - 1;  // (a row past N repeats the last one and is not written)
  const int64_t kb = P.K * (int64_t)sizeof(T);          // bytes of a row
  const char* pw = static_cast<const char*>(P.w) + row * P.ldw * (int64_t)sizeof(T) + g * 16;
  const char* pw1 = DUAL ? static_cast<const char*>(P.w1) + row * P.ldw * (int64_t)sizeof(T) + g * 16 : nullptr;
  const bool live = r < P.M;
  const char* px = static_cast<const char*>(P.x) + (live ? r : 0) * P.ldx * (int64_t)sizeof(T) + g * 16;
  f4v c = {0.f, 0.f, 0.f, 0.f}, c1 = {0.f, 0.f, 0.f, 0.f};
  const int64_t full = kb / 128;  // whole blocks
  int64_t b = w;
  for (; b + (U - 1) * kSkinnyWaves < full; b += U * kSkinnyWaves) {
    Raw32 a[U], a1[U], x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t o = (b + u * kSkinnyWaves) * 128;
      a[u] = skinny_load(pw + o);
      if constexpr (DUAL) a1[u] = skinny_load(pw1 + o);
      x[u] = skinny_load(px + o, live ? 128 : 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      skinny_mma<T>(c, a[u], x[u]);
      if constexpr (DUAL) skinny_mma<T>(c1, a1[u], x[u]);
    }
  }
  for (; b * 128 < kb; b += kSkinnyWaves) {  // the rest, and the last block's part inside K
    const int64_t o = b * 128, left = kb - o - g * 16;
    const Raw32 x = skinny_load(px + o, live ? left : 0);
    skinny_mma<T>(c, skinny_load(pw + o, left), x);
    if constexpr (DUAL) skinny_mma<T>(c1, skinny_load(pw1 + o, left), x);
  }
  part[w][0][lane] = c;
  if constexpr (DUAL) part[w][1][lane] = c1;
  __syncthreads();
  if (threadIdx.x >= 64 || !live) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int kSum = DUAL ? 4 : kSkinnyWaves;  // (both products' sums in one go need more registers than the K loop)
#pragma unroll kSum
  for (int i = 0; i < kSkinnyWaves; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] += part[i][0][lane][e];
      if constexpr (DUAL) u[e] += part[i][1][lane][e];
    }
  E = E.tile(0, n0);
  const int n = 4 * g;
  const int64_t left = E.cols - n;
  const int cnt = left >= 4 ? 4 : (int)left;
  if (cnt <= 0) return;
  if constexpr (DUAL) epi_apply(E, r, n, v, u, cnt);
  else epi_apply(E, r, n, v, cnt);
}

}  // namespace orda
