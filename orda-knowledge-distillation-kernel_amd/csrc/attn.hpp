// attn.hpp -- masked self-attention of 16-bit tensors, forward and backward, on
// the matrix cores (gfx950).
//
//   z = scale q.k, cap tanh(z / cap) with a cap, less slope |i - j| with slopes
//   P = softmax of z over the keys that a query sees, o = P v
//   dv = P^T do,  dz = P (do v^T - delta), delta = sum(do o), times 1 - tanh^2
//   dq = scale dz k,  dk = scale dz^T q
//
// Nothing of size S x S reaches memory: the forward pass keeps a running maximum
// and sum per query and leaves L = max + log2(sum) for the backward pass, which
// makes P again from z and L.
//
// One kernel's wave holds 32 queries (forward, dq) or 32 keys (dk and dv) and
// walks tiles of 64 rows of the other side, which the DMA brings into LDS one
// tile ahead.  Products are arranged so that a lane holds one of the wave's 32
// rows throughout: z^T = K q^T has queries in its columns, so that a query's
// maximum, sum, L and delta are one lane's own (and that of lane ^ 32, which
// holds the other half of the keys), and what the lane holds of P^T is, rounded
// to 16 bits, already an operand of the next product, o^T = V^T P^T: an MFMA
// adds up over its K index in any order, so V's rows are read in the order in
// which the lane holds P's (4 h + 0..3 and 8 + 4 h + 0..3 of 16, h = lane / 32).
//
// Two kernels for the backward pass, seven products of S x S x D instead of the
// five that one kernel would need, whose gradients of q would have to be added
// up by atomics in an order that changes from run to run.
//
// LDS: a tile's rows of HD elements (64 or 128; a head of D < HD is zero-padded
// on the way in), chunk c (16 bytes) of row r at c ^ swz(r), so that neither 16
// rows at one chunk (row reads) nor 4 rows at 64 bytes (transposed reads) meet
// in a bank.
//
// Which tiles are walked: 64 tiles at a time, lane t looks at tile t (causal
// bound, prefix, the ranges of document numbers on both sides) and a ballot
// tells which are seen at all and which need a look at each element.
#pragma once
#include "step_launch.hpp"
#include "tile16.hpp"

namespace orda {

constexpr int kAttnRows = 128;  // queries (forward, dq) or keys (dk, dv) of a workgroup: 4 waves of 32
constexpr int kAttnTile = 64;   // rows of the other side that one step takes

template <int HD>
__device__ __forceinline__ int attn_swz(int r) {
  return HD == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// A tile of 64 rows to LDS, 16 bytes a lane.  Rows from `rows` on and columns
// from D on arrive as zeros.
template <int HD>
struct AttnDma {
  static constexpr int kChunks = HD / 8, kIssues = 64 * kChunks / 256, kStep = 256 / kChunks;
  uint32_t off, step;
  int row;
  bool in;
  __device__ __forceinline__ void init(int64_t ss, int D) {
    const int p = wave_id() * 64 + (threadIdx.x & 63);
    row = p / kChunks;
    const int c = (p % kChunks) ^ attn_swz<HD>(row);  // (rows kStep apart have one swizzle)
    in = c * 8 < D;
    off = (uint32_t)row * (uint32_t)(ss * 2) + (uint32_t)c * 16;
    step = (uint32_t)kStep * (uint32_t)(ss * 2);
  }
  __device__ __forceinline__ void issue(const void* p, int64_t rows, char* tile) const {
    const auto rs = rsrc_of(p);
    const int w = wave_id();
#pragma unroll
    for (int i = 0; i < kIssues; ++i)
      dma16(rs, in && row + i * kStep < rows ? off + i * step : kOob, tile + (i * 4 + w) * 1024);
  }
};

// Fragments of a tile in LDS.
template <class T, int HD>
struct AttnFrags {
  static constexpr int kRow = HD * 2, kBlocks = HD / 32;
  uint32_t row_at, lo, hi;  // byte offsets in a tile
  __device__ __forceinline__ void init() {
    const int lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31;
    row_at = (uint32_t)(r * kRow + ((h ^ attn_swz<HD>(r)) << 4));
    const int s = lane & 15, k = 4 * h + (s >> 2), m = 16 * ((lane >> 4) & 1) + 4 * (s & 3);
    lo = (uint32_t)(k * kRow + (((m >> 3) ^ attn_swz<HD>(k)) << 4) + (m & 7) * 2);
    hi = (uint32_t)((k + 8) * kRow + (((m >> 3) ^ attn_swz<HD>(k + 8)) << 4) + (m & 7) * 2);
  }
  // rows 32 block + lane % 32, columns 16 ks + 8 (lane / 32)..
  __device__ __forceinline__ typename Traits<T>::Frag rows(const char* tile, int block, int ks) const {
    return *reinterpret_cast<const typename Traits<T>::Frag*>(tile + block * 32 * kRow + (row_at ^ (uint32_t)(ks << 5)));
  }
  // column 32 d + lane % 32 for all d, rows 16 KS + the permuted 8 of lane / 32
  template <int KS>
  __device__ __forceinline__ void cols(uint32_t tile, typename Traits<T>::Frag (&out)[kBlocks]) const {
    constexpr int kOff = KS * 16 * kRow;
    tr_s4 x[kBlocks][2];
    if constexpr (kBlocks == 4) {
      asm volatile(
          "ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
          "ds_read_b64_tr_b16 %2, %10 offset:%16\n\tds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
          "ds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
          "ds_read_b64_tr_b16 %6, %14 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%16\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(x[2][0]), "=&v"(x[2][1]),
            "=&v"(x[3][0]), "=&v"(x[3][1])
          : "v"(tile + lo), "v"(tile + hi), "v"(tile + (lo ^ 64u)), "v"(tile + (hi ^ 64u)), "v"(tile + (lo ^ 128u)),
            "v"(tile + (hi ^ 128u)), "v"(tile + (lo ^ 192u)), "v"(tile + (hi ^ 192u)), "n"(kOff)
          : "memory");
    } else {
      asm volatile(
          "ds_read_b64_tr_b16 %0, %4 offset:%8\n\tds_read_b64_tr_b16 %1, %5 offset:%8\n\t"
          "ds_read_b64_tr_b16 %2, %6 offset:%8\n\tds_read_b64_tr_b16 %3, %7 offset:%8\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1])
          : "v"(tile + lo), "v"(tile + hi), "v"(tile + (lo ^ 64u)), "v"(tile + (hi ^ 64u)), "n"(kOff)
          : "memory");
    }
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
      out[d] = __builtin_bit_cast(typename Traits<T>::Frag, __builtin_shufflevector(x[d][0], x[d][1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// The wave's own 32 rows as operands: row lane % 32, columns 16 ks + 8 h.. .
template <class T, int HD>
__device__ __forceinline__ void own_rows(const T* p, int64_t ss, int64_t row0, int64_t rows, int D, typename Traits<T>::Frag (&f)[HD / 16]) {
  const int lane = threadIdx.x & 63;
  const int64_t r = row0 + (lane & 31);
  const T* at = p + r * ss + 8 * (lane >> 5);
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    const bool in = r < rows && ks * 16 + 8 * (lane >> 5) < D;
    const s16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    f[ks] = in ? *reinterpret_cast<const typename Traits<T>::Frag*>(at + ks * 16) : __builtin_bit_cast(typename Traits<T>::Frag, zero);
  }
}

// v of this lane and of lane ^ 32.
__device__ __forceinline__ void both_halves(float v, float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
__device__ __forceinline__ float halves_sum(float v) {
  float a, b;
  both_halves(v, a, b);
  return a + b;
}
__device__ __forceinline__ float halves_max(float v) {
  float a, b;
  both_halves(v, a, b);
  return fmaxf(a, b);
}

// x (16 rows of the 32 that the MFMA's block has) as two operands of 16 rows.
template <class T>
__device__ __forceinline__ void as_operand(const float (&x)[16], typename Traits<T>::Frag (&f)[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint4 u;
    u.x = pack2<T>(x[8 * k], x[8 * k + 1]);
    u.y = pack2<T>(x[8 * k + 2], x[8 * k + 3]);
    u.z = pack2<T>(x[8 * k + 4], x[8 * k + 5]);
    u.w = pack2<T>(x[8 * k + 6], x[8 * k + 7]);
    f[k] = __builtin_bit_cast(typename Traits<T>::Frag, u);
  }
}

// acc^T (columns d, the lane's row) times `mul` to the lane's row at p: lanes l
// and l + 32 exchange groups of 4 columns, so that each stores 8 in a row.  LOW:
// what the rounding left instead, itself rounded.
template <class T, int HD, bool LOW = false>
__device__ __forceinline__ void store_own(const f32x16 (&acc)[HD / 32], float mul, T* p, int D, bool live) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = acc[d][8 * g + 2 * e] * mul, y = acc[d][8 * g + 2 * e + 1] * mul;
        u[e] = pack2<T>(x, y);
        if constexpr (LOW) u[e] = pack2<T>(x - lo16<T>(u[e]), y - hi16<T>(u[e]));
      }
      const auto a = __builtin_amdgcn_permlane32_swap(u[0], u[2], false, false);
      const auto b = __builtin_amdgcn_permlane32_swap(u[1], u[3], false, false);
      const int at = d * 32 + 16 * g + 8 * h;
      if (live && at < D) *reinterpret_cast<uint4*>(p + at) = make_uint4(a[0], b[0], a[1], b[1]);
    }
}

// ------------------------------------------------------------- masks
// The tiles [base, base + 64) of one side against the rows [r0, r0 + 128) of the
// other: seen by any, with elements that are not seen, with padding rows.
struct AttnTiles {
  uint64_t seen, part, pad;
};
// What the workgroup's rows have of documents: the smallest and largest number
// and whether there is padding.
struct DocRange {
  int lo, hi, pad;
  __device__ __forceinline__ void join(const int4& o) {
    lo = min(lo, o.x);
    hi = max(hi, o.y);
    pad |= o.z;
  }
};
template <bool KEYS>  // the tiles are keys (else queries)
__device__ __forceinline__ AttnTiles attn_tiles(const AttnParams& P, int base, int64_t r0, int64_t prefix, const int4* ranges, const DocRange& own) {
  const int t = base + (threadIdx.x & 63);
  const int64_t a = (int64_t)t * kAttnTile, b = lmin(a + kAttnTile, P.S), r1 = lmin(r0 + kAttnRows, P.S);  // [a, b) against [r0, r1)
  bool seen = a < P.S, part = KEYS && a + kAttnTile > P.S, pad = false;
  if (P.causal) {
    const int64_t q0 = KEYS ? r0 : a, q1 = KEYS ? r1 : b, k0 = KEYS ? a : r0, k1 = KEYS ? b : r1;
    if (k0 >= q1 && k0 >= prefix) seen = false;
    if (k1 - 1 > q0 && k1 > prefix) part = true;
  }
  if (ranges && seen) {
    const int4 d = ranges[t];
    if (d.x > own.hi || d.y < own.lo) seen = false;
    if (d.x != d.y || own.lo != own.hi || d.x != own.lo || d.z || own.pad) part = true;
    pad = d.z != 0;
  }
  return {__ballot(seen), __ballot(seen && part), __ballot(seen && pad)};
}

// Rows without a document: zeros in LDS, so that whatever they hold (nothing, for
// what lies behind a batch's sequences) is not multiplied by a probability of 0.
template <int HD>
__device__ __forceinline__ void clear_padding(const int* docs, char* one, char* two) {
  constexpr int kChunks = HD / 8;
  for (int p = threadIdx.x; p < kAttnTile * kChunks; p += 256)
    if (docs[p / kChunks] < 0) {
      reinterpret_cast<uint4*>(one)[p] = make_uint4(0, 0, 0, 0);
      if (two) reinterpret_cast<uint4*>(two)[p] = make_uint4(0, 0, 0, 0);
    }
  __syncthreads();
}

// Document numbers of the tile's rows that the lane's 16 elements of block
// `block` belong to.
__device__ __forceinline__ void tile_docs(const int* docs, int block, int (&d)[16]) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int4 v = *reinterpret_cast<const int4*>(docs + 32 * block + 8 * g + 4 * h);
    d[4 * g] = v.x;
    d[4 * g + 1] = v.y;
    d[4 * g + 2] = v.z;
    d[4 * g + 3] = v.w;
  }
}
// The tile's row, relative to the tile, of element r of block `block`.
__device__ __forceinline__ int tile_row(int block, int r) {
  return 32 * block + (r >> 2) * 8 + ((threadIdx.x & 63) >> 5) * 4 + (r & 3);
}

// Scores in units of log2 from products: z[r] = log2(e) (cap tanh(scale s / cap)
// - slope |i - j|), and with CAP the tanh.  dist: the lane's row less the tile's
// first.  tanh u = 1 - 2 / (1 + e^2u) on the hardware's exp2 and reciprocal, off
// by 2e-7, a cap of 50 by 1e-5, below half a step of a 16-bit probability.
template <bool CAP, bool BIAS>
__device__ __forceinline__ void scores(const f32x16& s, float (&z)[16], float (&th)[16], const AttnParams& P, float slope, int dist, int block) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    if constexpr (CAP) {
      const float e = __builtin_amdgcn_exp2f(s[r] * P.cap_in);
      th[r] = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + e);
      z[r] = th[r] * P.cap_out;
    } else {
      z[r] = s[r] * P.scale_log2;
    }
    if constexpr (BIAS) z[r] = fmaf(-slope, fabsf((float)(dist - tile_row(block, r))), z[r]);
  }
}

// ------------------------------------------------------------- forward
template <class T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void k_attn(AttnParams P) {
  using Frag = typename Traits<T>::Frag;
  constexpr int kTile = kAttnTile * HD * 2, kBlocks = HD / 32;
  __shared__ __attribute__((aligned(16))) char lds[2][2][kTile];
  const int t = xcd_order(blockIdx.x, gridDim.x);
  const int bh = t / P.tiles, q0 = (P.tiles - 1 - t % P.tiles) * kAttnRows;  // (long rows first)
  const int b = bh / P.H, head = bh - b * P.H, kv = head / P.group;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int64_t row0 = q0 + w * 32, i = row0 + (lane & 31);
  const T* K = static_cast<const T*>(P.k) + b * P.kb + kv * P.kh;
  const T* V = static_cast<const T*>(P.v) + b * P.vb + kv * P.vh;
  Frag q[HD / 16];
  own_rows<T, HD>(static_cast<const T*>(P.q) + b * P.qb + head * P.qh, P.qs, row0, P.S, P.D, q);
  const int64_t prefix = P.prefix ? P.prefix[b] : 0;
  const float slope = BIAS ? P.slopes[head] * kLog2e : 0.0f;
  const int* docs = P.docs ? P.docs + (int64_t)b * P.padded : nullptr;
  const int4* ranges = P.docs ? P.ranges + (int64_t)b * (P.padded / kAttnTile) : nullptr;
  DocRange own{0x7fffffff, -1, 0};
  int doc = 0;
  if (docs) {
    own.join(ranges[q0 / kAttnTile]);
    own.join(ranges[q0 / kAttnTile + 1]);
    doc = docs[i];
  }
  AttnDma<HD> kd, vd;
  kd.init(P.ks, P.D);
  vd.init(P.vs, P.D);
  AttnFrags<T, HD> fr;
  fr.init();
  const uint32_t base_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0][0];

  f32x16 o[kBlocks];
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  float m = -kInf, l = 0.0f;
  int stage = 0;
  auto issue = [&](int tile, int st) {
    const int64_t k0 = (int64_t)tile * kAttnTile;
    kd.issue(K + k0 * P.ks, P.S - k0, lds[st][0]);
    vd.issue(V + k0 * P.vs, P.S - k0, lds[st][1]);
  };
  const int all = (int)((P.S + kAttnTile - 1) / kAttnTile);
  for (int base = 0; base < all; base += 64) {
    AttnTiles tiles = attn_tiles<true>(P, base, q0, prefix, ranges, own);
    if (!tiles.seen) continue;
    int j = __builtin_ctzll(tiles.seen);
    issue(base + j, stage);
    while (true) {
      const uint64_t rest = tiles.seen & (tiles.seen - 1);
      const int next = rest ? __builtin_ctzll(rest) : -1;
      wait_vmem<0>();
      tile_barrier();
      if (next >= 0) issue(base + next, stage ^ 1);
      const int64_t k0 = (int64_t)(base + j) * kAttnTile;
      const bool part = (tiles.part >> j) & 1;
      if ((tiles.pad >> j) & 1) clear_padding<HD>(docs + k0, lds[stage][1], nullptr);
      const bool hidden = P.causal && k0 > row0 + 31 && k0 >= prefix;  // (for this wave's rows)
      if (!hidden) {
        const char* kt = lds[stage][0];
        const uint32_t vt = base_lds + (uint32_t)(stage * 2 + 1) * kTile;
        float p[2][16], top = -kInf;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          f32x16 s;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) s = Traits<T>::mma(fr.rows(kt, n, ks), q[ks], s);
          float th[16];
          scores<CAP, BIAS>(s, p[n], th, P, slope, (int)(i - k0), n);
          if (part) {
            int dk[16];
            if (docs) tile_docs(docs + k0, n, dk);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int64_t key = k0 + tile_row(n, r);
              bool see = key < P.S && (!P.causal || key <= i || key < prefix);
              if (docs) see = see && dk[r] == doc && doc >= 0;
              p[n][r] = see ? p[n][r] : -kInf;
            }
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, p[n][r]);
        }
        top = halves_max(top);
        // The maximum follows only where it grows by more than 2^8: sums and
        // products of probabilities up to 2^8 lose nothing in fp32.
        if (__any(top > m + 8.0f)) {
          const float to = fmaxf(m, top), by = to == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - to);
          m = to;
          l *= by;
#pragma unroll
          for (int d = 0; d < kBlocks; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] *= by;
        }
        const float at = m == -kInf ? 0.0f : m;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            p[n][r] = __builtin_amdgcn_exp2f(p[n][r] - at);
            l += p[n][r];
          }
          // P is rounded to 16 bits as an operand of the product, its sum is not
          Frag pf[2], vf[kBlocks];
          as_operand<T>(p[n], pf);
          static_for<0, 2>([&](auto k) {
            constexpr int KS = decltype(k)::value;
            if (n == 0) fr.template cols<KS>(vt, vf);
            else fr.template cols<2 + KS>(vt, vf);
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) o[d] = Traits<T>::mma(vf[d], pf[KS], o[d]);
          });
        }
      }
      stage ^= 1;
      if (next < 0) break;
      tiles.seen = rest;
      j = next;
    }
  }
  l = halves_sum(l);
  const bool empty = !(l > 0.0f) && l == l;
  if (P.lse && lane < 32)
    P.lse[(int64_t)bh * P.padded + i] = i >= P.S || empty ? kInf : m + __builtin_amdgcn_logf(l);
  const int64_t at = ((b * P.S + i) * P.H + head) * P.D;
  const float inv = empty ? 0.0f : 1.0f / l;
  store_own<T, HD>(o, inv, static_cast<T*>(P.o) + at, P.D, i < P.S);
  // dz = P (dP - delta) cancels where P is near 1, and delta = sum(do o) would be
  // as far off as o's rounding: for the backward pass o is kept in both halves
  // (8 short rows: dq and dk off by 2.4e-3 of their norm instead of 3.4e-3 in bf16).
  if (P.o_low) store_own<T, HD, true>(o, inv, static_cast<T*>(P.o_low) + at, P.D, i < P.S);
}

// ------------------------------------------------------------- dq
// Also delta = sum(do o) of each query, which the next kernel reads.
template <class T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void k_attn_dq(AttnParams P) {
  using Frag = typename Traits<T>::Frag;
  constexpr int kTile = kAttnTile * HD * 2, kBlocks = HD / 32;
  __shared__ __attribute__((aligned(16))) char lds[2][2][kTile];
  const int t = xcd_order(blockIdx.x, gridDim.x);
  const int bh = t / P.tiles, q0 = (P.tiles - 1 - t % P.tiles) * kAttnRows;
  const int b = bh / P.H, head = bh - b * P.H, kv = head / P.group;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int64_t row0 = q0 + w * 32, i = row0 + (lane & 31);
  const T* K = static_cast<const T*>(P.k) + b * P.kb + kv * P.kh;
  const T* V = static_cast<const T*>(P.v) + b * P.vb + kv * P.vh;
  const int64_t prefix = P.prefix ? P.prefix[b] : 0;
  const float slope = BIAS ? P.slopes[head] * kLog2e : 0.0f;
  const int* docs = P.docs ? P.docs + (int64_t)b * P.padded : nullptr;
  const int4* ranges = P.docs ? P.ranges + (int64_t)b * (P.padded / kAttnTile) : nullptr;
  DocRange own{0x7fffffff, -1, 0};
  int doc = 0;
  if (docs) {
    own.join(ranges[q0 / kAttnTile]);
    own.join(ranges[q0 / kAttnTile + 1]);
    doc = docs[i];
  }
  Frag q[HD / 16], g[HD / 16];
  own_rows<T, HD>(static_cast<const T*>(P.q) + b * P.qb + head * P.qh, P.qs, row0, P.S, P.D, q);
  own_rows<T, HD>(static_cast<const T*>(P.dout) + b * P.gb + head * P.gh, P.gs, row0, P.S, P.D, g);
  float delta = 0.0f;
  {
    Frag o[HD / 16], low[HD / 16];
    const int64_t at = (b * P.S * P.H + head) * P.D;
    own_rows<T, HD>(static_cast<const T*>(P.o) + at, P.H * P.D, row0, P.S, P.D, o);
    own_rows<T, HD>(static_cast<const T*>(P.o_low) + at, P.H * P.D, row0, P.S, P.D, low);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf(to_f32(g[ks][e]), to_f32(o[ks][e]) + to_f32(low[ks][e]), delta);
    delta = halves_sum(delta);
    if (doc < 0) delta = 0.0f;
    if (lane < 32) P.delta[(int64_t)bh * P.padded + i] = delta;
  }
  if (!P.dq) return;
  const float lse = P.lse[(int64_t)bh * P.padded + i];
  AttnDma<HD> kd, vd;
  kd.init(P.ks, P.D);
  vd.init(P.vs, P.D);
  AttnFrags<T, HD> fr;
  fr.init();
  const uint32_t base_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0][0];
  f32x16 dq[kBlocks];
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.0f;
  int stage = 0;
  auto issue = [&](int tile, int st) {
    const int64_t k0 = (int64_t)tile * kAttnTile;
    kd.issue(K + k0 * P.ks, P.S - k0, lds[st][0]);
    vd.issue(V + k0 * P.vs, P.S - k0, lds[st][1]);
  };
  const int all = (int)((P.S + kAttnTile - 1) / kAttnTile);
  for (int base = 0; base < all; base += 64) {
    AttnTiles tiles = attn_tiles<true>(P, base, q0, prefix, ranges, own);
    if (!tiles.seen) continue;
    int j = __builtin_ctzll(tiles.seen);
    issue(base + j, stage);
    while (true) {
      const uint64_t rest = tiles.seen & (tiles.seen - 1);
      const int next = rest ? __builtin_ctzll(rest) : -1;
      wait_vmem<0>();
      tile_barrier();
      if (next >= 0) issue(base + next, stage ^ 1);
      const int64_t k0 = (int64_t)(base + j) * kAttnTile;
      const bool part = (tiles.part >> j) & 1;
      if ((tiles.pad >> j) & 1) clear_padding<HD>(docs + k0, lds[stage][0], lds[stage][1]);
      const bool hidden = P.causal && k0 > row0 + 31 && k0 >= prefix;
      if (!hidden) {
        const char *kt = lds[stage][0], *vt = lds[stage][1];
        const uint32_t ktr = base_lds + (uint32_t)(stage * 2) * kTile;
        static_for<0, 2>([&](auto nn) {
          constexpr int n = decltype(nn)::value;
          f32x16 s, dp;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            s = Traits<T>::mma(fr.rows(kt, n, ks), q[ks], s);
            dp = Traits<T>::mma(fr.rows(vt, n, ks), g[ks], dp);
          }
          float z[16], th[16];
          scores<CAP, BIAS>(s, z, th, P, slope, (int)(i - k0), n);
          if (part) {
            int dk[16];
            if (docs) tile_docs(docs + k0, n, dk);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int64_t key = k0 + tile_row(n, r);
              bool see = key < P.S && (!P.causal || key <= i || key < prefix);
              if (docs) see = see && dk[r] == doc && doc >= 0;
              z[r] = see ? z[r] : -kInf;
            }
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            z[r] = __builtin_amdgcn_exp2f(z[r] - lse) * (dp[r] - delta);
            if constexpr (CAP) z[r] *= 1.0f - th[r] * th[r];
          }
          Frag zf[2], kf[kBlocks];
          as_operand<T>(z, zf);  // (dz in 16 bits, as an operand of the product)
          static_for<0, 2>([&](auto k) {
            constexpr int KS = decltype(k)::value;
            fr.template cols<2 * n + KS>(ktr, kf);
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) dq[d] = Traits<T>::mma(kf[d], zf[KS], dq[d]);
          });
        });
      }
      stage ^= 1;
      if (next < 0) break;
      tiles.seen = rest;
      j = next;
    }
  }
  if (doc < 0)  // (what a padding row holds may not be finite)
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[d][r] = 0.0f;
  T* out = static_cast<T*>(P.dq) + ((b * P.S + i) * P.H + head) * P.D;
  store_own<T, HD>(dq, P.scale, out, P.D, i < P.S);
}

// ------------------------------------------------------------- dk and dv
// A workgroup's 128 keys against the queries of all heads that share them.
template <class T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 1) void k_attn_dkv(AttnParams P) {
  using Frag = typename Traits<T>::Frag;
  constexpr int kTile = kAttnTile * HD * 2, kBlocks = HD / 32;
  __shared__ __attribute__((aligned(16))) char lds[2][2][kTile];
  __shared__ __attribute__((aligned(16))) float stats[2][2][kAttnTile];  // L and delta of the tile's queries
  const int t = xcd_order(blockIdx.x, gridDim.x);
  const int bk = t / P.tiles, r0 = (t % P.tiles) * kAttnRows;  // (with a causal mask the first keys have the most queries)
  const int b = bk / P.KV, kv = bk - b * P.KV;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int64_t row0 = r0 + w * 32, key = row0 + (lane & 31);
  const int64_t prefix = P.prefix ? P.prefix[b] : 0;
  const int* docs = P.docs ? P.docs + (int64_t)b * P.padded : nullptr;
  const int4* ranges = P.docs ? P.ranges + (int64_t)b * (P.padded / kAttnTile) : nullptr;
  DocRange own{0x7fffffff, -1, 0};
  int doc = 0;
  if (docs) {
    own.join(ranges[r0 / kAttnTile]);
    own.join(ranges[r0 / kAttnTile + 1]);
    doc = docs[key];
  }
  Frag kf[HD / 16], vf[HD / 16];
  own_rows<T, HD>(static_cast<const T*>(P.k) + b * P.kb + kv * P.kh, P.ks, row0, P.S, P.D, kf);
  own_rows<T, HD>(static_cast<const T*>(P.v) + b * P.vb + kv * P.vh, P.vs, row0, P.S, P.D, vf);
  AttnDma<HD> qd, gd;
  qd.init(P.qs, P.D);
  gd.init(P.gs, P.D);
  AttnFrags<T, HD> fr;
  fr.init();
  const uint32_t base_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0][0];
  f32x16 dk[kBlocks], dv[kBlocks];
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.0f;
  int stage = 0;
  const int all = (int)((P.S + kAttnTile - 1) / kAttnTile);
  for (int head = kv * P.group; head < (kv + 1) * P.group; ++head) {
    const T* Q = static_cast<const T*>(P.q) + b * P.qb + head * P.qh;
    const T* G = static_cast<const T*>(P.dout) + b * P.gb + head * P.gh;
    const float* lse = P.lse + ((int64_t)b * P.H + head) * P.padded;
    const float* delta = P.delta + ((int64_t)b * P.H + head) * P.padded;
    const float slope = BIAS ? P.slopes[head] * kLog2e : 0.0f;
    auto issue = [&](int tile, int st) {
      const int64_t a = (int64_t)tile * kAttnTile;
      qd.issue(Q + a * P.qs, P.S - a, lds[st][0]);
      gd.issue(G + a * P.gs, P.S - a, lds[st][1]);
      if (w < 2)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of((w ? delta : lse) + a), (__attribute__((address_space(3))) void*)stats[st][w], 4,
                                                 lane * 4, 0, 0, 0);
    };
    for (int base = 0; base < all; base += 64) {
      AttnTiles tiles = attn_tiles<false>(P, base, r0, prefix, ranges, own);
      if (!tiles.seen) continue;
      int j = __builtin_ctzll(tiles.seen);
      issue(base + j, stage);
      while (true) {
        const uint64_t rest = tiles.seen & (tiles.seen - 1);
        const int next = rest ? __builtin_ctzll(rest) : -1;
        wait_vmem<0>();
        tile_barrier();
        if (next >= 0) issue(base + next, stage ^ 1);
        const int64_t a = (int64_t)(base + j) * kAttnTile;
        const bool part = (tiles.part >> j) & 1;
        if ((tiles.pad >> j) & 1) clear_padding<HD>(docs + a, lds[stage][0], lds[stage][1]);
        const bool hidden = P.causal && row0 > a + kAttnTile - 1 && row0 >= prefix;
        if (!hidden) {
          const char *qt = lds[stage][0], *gt = lds[stage][1];
          const uint32_t qtr = base_lds + (uint32_t)(stage * 2) * kTile, gtr = qtr + kTile;
          static_for<0, 2>([&](auto nn) {
            constexpr int n = decltype(nn)::value;
            f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
              s = Traits<T>::mma(fr.rows(qt, n, ks), kf[ks], s);
              dp = Traits<T>::mma(fr.rows(gt, n, ks), vf[ks], dp);
            }
            float z[16], th[16], p[16];
            scores<CAP, BIAS>(s, z, th, P, slope, (int)(key - a), n);
            if (part) {
              int dq[16];
              if (docs) tile_docs(docs + a, n, dq);
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int64_t i = a + tile_row(n, r);
                bool see = !P.causal || key <= i || key < prefix;
                if (docs) see = see && dq[r] == doc && doc >= 0;
                z[r] = see ? z[r] : -kInf;
              }
            }
            // queries behind the last, or that see nothing, have L = inf
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
              const int at = tile_row(n, 4 * gq);
              const float4 L = *reinterpret_cast<const float4*>(&stats[stage][0][at]);
              const float4 dl = *reinterpret_cast<const float4*>(&stats[stage][1][at]);
              const float Lr[4] = {L.x, L.y, L.z, L.w}, dr[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int r = 4 * gq + e;
                p[r] = __builtin_amdgcn_exp2f(z[r] - Lr[e]);
                z[r] = p[r] * (dp[r] - dr[e]);
                if constexpr (CAP) z[r] *= 1.0f - th[r] * th[r];
              }
            }
            Frag pf[2], zf[2], cf[kBlocks];
            as_operand<T>(p, pf);
            as_operand<T>(z, zf);
            static_for<0, 2>([&](auto k) {
              constexpr int KS = decltype(k)::value;
              fr.template cols<2 * n + KS>(gtr, cf);
#pragma unroll
              for (int d = 0; d < kBlocks; ++d) dv[d] = Traits<T>::mma(cf[d], pf[KS], dv[d]);
              fr.template cols<2 * n + KS>(qtr, cf);
#pragma unroll
              for (int d = 0; d < kBlocks; ++d) dk[d] = Traits<T>::mma(cf[d], zf[KS], dk[d]);
            });
          });
        }
        stage ^= 1;
        if (next < 0) break;
        tiles.seen = rest;
        j = next;
      }
    }
  }
  if (doc < 0)
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.0f;
  const int64_t at = ((b * P.S + key) * P.KV + kv) * P.D;
  if (P.dk) store_own<T, HD>(dk, P.scale, static_cast<T*>(P.dk) + at, P.D, key < P.S);
  if (P.dv) store_own<T, HD>(dv, 1.0f, static_cast<T*>(P.dv) + at, P.D, key < P.S);
}

// ------------------------------------------------------------- launches
template <class T, int HD, bool CAP, bool BIAS>
static hipError_t attn_go(AttnParams P, AttnPass pass, hipStream_t s) {
  P.tiles = (int)((P.S + kAttnRows - 1) / kAttnRows);
  const dim3 grid((unsigned)(P.tiles * P.B * (pass == ATTN_DKV ? P.KV : P.H)));
  switch (pass) {
    case ATTN_FORWARD: hipLaunchKernelGGL((k_attn<T, HD, CAP, BIAS>), grid, dim3(256), 0, s, P); break;
    case ATTN_DQ: hipLaunchKernelGGL((k_attn_dq<T, HD, CAP, BIAS>), grid, dim3(256), 0, s, P); break;
    default: hipLaunchKernelGGL((k_attn_dkv<T, HD, CAP, BIAS>), grid, dim3(256), 0, s, P);
  }
  return hipGetLastError();
}
template <class T, int HD>
hipError_t launch_attn(const AttnParams& P, AttnPass pass, hipStream_t s) {
  const bool bias = P.slopes != nullptr;
  if (P.cap_out > 0.0f) return bias ? attn_go<T, HD, true, true>(P, pass, s) : attn_go<T, HD, true, false>(P, pass, s);
  return bias ? attn_go<T, HD, false, true>(P, pass, s) : attn_go<T, HD, false, false>(P, pass, s);
}

}  // namespace orda
