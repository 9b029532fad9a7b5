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
// LDS: a tile's rows of 64 or 128 elements, of which HD (64, 96, 128) go through
// the products (a head of D < HD is zero-padded on the way in), chunk c (16 bytes)
// of row r at c ^ swz(r), so that neither 16 rows at one chunk (row reads) nor 4
// rows at 64 bytes (transposed reads) meet in a bank.
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
constexpr int kAttnLd = HD <= 64 ? 64 : 128;  // elements of a row in LDS

template <int LD>
__device__ __forceinline__ int attn_swz(int r) {
  return LD == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// Workgroup -> (head of the batch, tile of its rows).  An XCD takes whole heads,
// so that its L2 holds their keys and values.  With a causal mask a tile's work
// grows (or falls) with its number: of 8 heads of an XCD together the longest
// tiles come first, so that the last to end are short ones.
__device__ __forceinline__ void attn_place(const AttnParams& P, int id, int heads, bool last_first, int& head, int& tile) {
  constexpr int kTogether = 8;
  if (P.causal && heads % 8 == 0) {
    const int per = heads / 8, local = id / 8;
    const int g = local / (kTogether * P.tiles) * kTogether, n = min(kTogether, per - g), in = local - g * P.tiles;
    head = id % 8 * per + g + in % n;
    tile = in / n;
  } else {
    const int t = xcd_order(id, gridDim.x);
    head = t / P.tiles;
    tile = t - head * P.tiles;
  }
  if (last_first) tile = P.tiles - 1 - tile;
}

// A tile of 64 rows to LDS, 16 bytes a lane.  Rows from `rows` on and columns
// from D on arrive as zeros.
template <int LD>
struct AttnDma {
  static constexpr int WAVES = 4;
  static constexpr int kChunks = LD / 8, kIssues = kChunks / WAVES, kStep = 64 * WAVES / kChunks;
  static_assert(kIssues > 0 && kStep % 16 == 0, "rows kStep apart have one swizzle");
  uint32_t off[kIssues];
  int row;
  __device__ __forceinline__ void init(int64_t ss, int D) {
    const int p = threadIdx.x & 255;
    row = p / kChunks;
    const int c = (p % kChunks) ^ attn_swz<LD>(row);
#pragma unroll
    for (int i = 0; i < kIssues; ++i) off[i] = c * 8 < D ? (uint32_t)(row + i * kStep) * (uint32_t)(ss * 2) + (uint32_t)c * 16 : kOob;
  }
  __device__ __forceinline__ void issue(const void* p, int rows, char* tile) const {
    const auto rs = rsrc_of(p);
    const int w = wave_id() & 3;
    if (rows >= kAttnTile) {
#pragma unroll
      for (int i = 0; i < kIssues; ++i) dma16(rs, off[i], tile + (i * WAVES + w) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kIssues; ++i) dma16(rs, row + i * kStep < rows ? off[i] : kOob, tile + (i * WAVES + w) * 1024);
    }
  }
};

// Fragments of a tile in LDS.
template <class T, int HD>
struct AttnFrags {
  static constexpr int kRow = kAttnLd<HD> * 2, kBlocks = HD / 32;
  uint32_t row_at, lo, hi;  // byte offsets in a tile
  __device__ __forceinline__ void init() {
    const int lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31;
    row_at = (uint32_t)(r * kRow + ((h ^ attn_swz<kAttnLd<HD>>(r)) << 4));
    const int s = lane & 15, k = 4 * h + (s >> 2), m = 16 * ((lane >> 4) & 1) + 4 * (s & 3);
    lo = (uint32_t)(k * kRow + (((m >> 3) ^ attn_swz<kAttnLd<HD>>(k)) << 4) + (m & 7) * 2);
    hi = (uint32_t)((k + 8) * kRow + (((m >> 3) ^ attn_swz<kAttnLd<HD>>(k + 8)) << 4) + (m & 7) * 2);
  }
  // rows lane % 32 of the 32 at `block`, columns 16 ks + 8 (lane / 32)..
  __device__ __forceinline__ typename Traits<T>::Frag rows(const char* block, int ks) const {
    return *reinterpret_cast<const typename Traits<T>::Frag*>(block + (row_at ^ (uint32_t)(ks << 5)));
  }
  // column 32 d + lane % 32 for all d, the 32 rows at LDS address `block` in two
  // operands of 16 (of each the permuted 8 of lane / 32).  Assembly that waits
  // for its own reads: the compiler's transposed read waits for the DMA too.
  __device__ __forceinline__ void cols(uint32_t block, typename Traits<T>::Frag (&out)[2][kBlocks]) const {
    constexpr int kOff = 16 * kRow;
    const uint32_t a = block + lo, b = block + hi;  // (blocks are aligned: the exclusive or below stays in the row)
    tr_s4 x[2][kBlocks][2];
    if constexpr (kBlocks == 4) {
      asm volatile(
          "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %17\n\t"
          "ds_read_b64_tr_b16 %2, %18\n\tds_read_b64_tr_b16 %3, %19\n\t"
          "ds_read_b64_tr_b16 %4, %20\n\tds_read_b64_tr_b16 %5, %21\n\t"
          "ds_read_b64_tr_b16 %6, %22\n\tds_read_b64_tr_b16 %7, %23\n\t"
          "ds_read_b64_tr_b16 %8, %16 offset:%24\n\tds_read_b64_tr_b16 %9, %17 offset:%24\n\t"
          "ds_read_b64_tr_b16 %10, %18 offset:%24\n\tds_read_b64_tr_b16 %11, %19 offset:%24\n\t"
          "ds_read_b64_tr_b16 %12, %20 offset:%24\n\tds_read_b64_tr_b16 %13, %21 offset:%24\n\t"
          "ds_read_b64_tr_b16 %14, %22 offset:%24\n\tds_read_b64_tr_b16 %15, %23 offset:%24\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(x[0][0][0]), "=&v"(x[0][0][1]), "=&v"(x[0][1][0]), "=&v"(x[0][1][1]), "=&v"(x[0][2][0]), "=&v"(x[0][2][1]),
            "=&v"(x[0][3][0]), "=&v"(x[0][3][1]), "=&v"(x[1][0][0]), "=&v"(x[1][0][1]), "=&v"(x[1][1][0]), "=&v"(x[1][1][1]),
            "=&v"(x[1][2][0]), "=&v"(x[1][2][1]), "=&v"(x[1][3][0]), "=&v"(x[1][3][1])
          : "v"(a), "v"(b), "v"(a ^ 64u), "v"(b ^ 64u), "v"(a ^ 128u), "v"(b ^ 128u), "v"(a ^ 192u), "v"(b ^ 192u), "n"(kOff)
          : "memory");
    } else if constexpr (kBlocks == 3) {
      asm volatile(
          "ds_read_b64_tr_b16 %0, %12\n\tds_read_b64_tr_b16 %1, %13\n\t"
          "ds_read_b64_tr_b16 %2, %14\n\tds_read_b64_tr_b16 %3, %15\n\t"
          "ds_read_b64_tr_b16 %4, %16\n\tds_read_b64_tr_b16 %5, %17\n\t"
          "ds_read_b64_tr_b16 %6, %12 offset:%18\n\tds_read_b64_tr_b16 %7, %13 offset:%18\n\t"
          "ds_read_b64_tr_b16 %8, %14 offset:%18\n\tds_read_b64_tr_b16 %9, %15 offset:%18\n\t"
          "ds_read_b64_tr_b16 %10, %16 offset:%18\n\tds_read_b64_tr_b16 %11, %17 offset:%18\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(x[0][0][0]), "=&v"(x[0][0][1]), "=&v"(x[0][1][0]), "=&v"(x[0][1][1]), "=&v"(x[0][2][0]), "=&v"(x[0][2][1]),
            "=&v"(x[1][0][0]), "=&v"(x[1][0][1]), "=&v"(x[1][1][0]), "=&v"(x[1][1][1]), "=&v"(x[1][2][0]), "=&v"(x[1][2][1])
          : "v"(a), "v"(b), "v"(a ^ 64u), "v"(b ^ 64u), "v"(a ^ 128u), "v"(b ^ 128u), "n"(kOff)
          : "memory");
    } else {
      asm volatile(
          "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9\n\t"
          "ds_read_b64_tr_b16 %2, %10\n\tds_read_b64_tr_b16 %3, %11\n\t"
          "ds_read_b64_tr_b16 %4, %8 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
          "ds_read_b64_tr_b16 %6, %10 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(x[0][0][0]), "=&v"(x[0][0][1]), "=&v"(x[0][1][0]), "=&v"(x[0][1][1]), "=&v"(x[1][0][0]), "=&v"(x[1][0][1]),
            "=&v"(x[1][1][0]), "=&v"(x[1][1][1])
          : "v"(a), "v"(b), "v"(a ^ 64u), "v"(b ^ 64u), "n"(kOff)
          : "memory");
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
        out[k][d] = __builtin_bit_cast(typename Traits<T>::Frag, __builtin_shufflevector(x[k][d][0], x[k][d][1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// acc^T times `mul`, to a row of fp32.
template <int HD>
__device__ __forceinline__ void store_part(const f32x16 (&acc)[HD / 32], float mul, float* p, int D, bool live) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * d + 8 * g + 4 * h;
      if (live && col < D) *reinterpret_cast<f4v*>(p + col) = f4v{acc[d][4 * g] * mul, acc[d][4 * g + 1] * mul, acc[d][4 * g + 2] * mul, acc[d][4 * g + 3] * mul};
    }
}

// The wave's own 32 rows as operands: row lane % 32, columns 16 ks + 8 h.. .
// negate: with their signs turned.
template <class T, int HD>
__device__ __forceinline__ void own_rows(const T* p, int64_t ss, int row0, int rows, int D, typename Traits<T>::Frag (&f)[HD / 16], bool negate = false) {
  const int lane = threadIdx.x & 63, r = row0 + (lane & 31);
  const T* at = p + r * ss + 8 * (lane >> 5);
  const uint32_t turn = negate ? 0x80008000u : 0u;
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (r < rows && ks * 16 + 8 * (lane >> 5) < D) u = *reinterpret_cast<const uint4*>(at + ks * 16);
    u.x ^= turn;
    u.y ^= turn;
    u.z ^= turn;
    u.w ^= turn;
    f[ks] = __builtin_bit_cast(typename Traits<T>::Frag, u);
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

// What x's rounding to f left, as operands of their own: FINE, for short sequences
// (step_abi.hip, where `fine` is set, has both sides measured).
template <class T>
__device__ __forceinline__ void rest_operand(const float (&x)[16], const typename Traits<T>::Frag (&f)[2], typename Traits<T>::Frag (&rest)[2]) {
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = x[i] - to_f32(f[i >> 3][i & 7]);
  as_operand<T>(y, rest);
}

// fp16 operands.  Below 2^-14 fp16 has steps of 2^-24, and probabilities of long
// rows and what small gradients from above make of them lie there: dz of 4096
// keys with gradients of 1e-4 put dq off by 5 % of its norm.  Operands are lifted
// by powers of two, which the results take out in fp32.  (bf16 has fp32's range.)
// Forward: P, up to 2^8 of the running maximum's, by 2^7.  Backward: P, up to 1
// (by the rounding of L at scores of 1e5 a little more), by 2^10, within L.  dz
// has no bound that is known beforehand: it starts at another 2^30, and where the
// lane's row (a query of dq, a key of dk) passes 2^15 goes down to 2^8, with its sum
// so far.  (dq and dk in fp16 take up to 8 % longer for it: 3 x 1777 rows of 12 heads
// of 80 with a cap 81 -> 85 and 120 -> 126 us, 2 x 4096 of 32 heads of 128 436 and 688
// -> 718.)
template <class T>
constexpr bool kNarrow = std::is_same_v<T, f16>;
template <class T>
constexpr float kLiftForward = kNarrow<T> ? 7.0f : 0.0f;
template <class T>
constexpr float kLiftBackward = kNarrow<T> ? 10.0f : 0.0f;
template <class T>
constexpr float kLiftScores = kNarrow<T> ? 30.0f : 0.0f;
// The exponent that dz of the lane's row goes down by, 0 nearly always.
template <int N>
__device__ __forceinline__ int keep_in_range(float (&z)[16], f32x16 (&acc)[N]) {
  constexpr float kTop = 32768.0f;
  float top = fabsf(z[0]);
#pragma unroll
  for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(z[r]));
  if (!__any(top > kTop)) return 0;
  top = halves_max(top);
  const int down = top > kTop && top < kInf ? __builtin_amdgcn_frexp_expf(top) - 8 : 0;
  const float by = __builtin_amdgcn_ldexpf(1.0f, -down);
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] *= by;
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] *= by;
  return down;
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
// What the workgroup's 128 rows have of documents: the smallest and largest
// number and whether there is padding.
struct DocRange {
  int lo, hi, pad;
  __device__ __forceinline__ DocRange(const int4& a) : lo(a.x), hi(a.y), pad(a.z) {}
  __device__ __forceinline__ void join(const DocRange& o) {
    lo = min(lo, o.lo);
    hi = max(hi, o.hi);
    pad |= o.pad;
  }
  __device__ __forceinline__ bool meets(const DocRange& o) const { return lo <= o.hi && hi >= o.lo; }
  __device__ __forceinline__ bool one(const DocRange& o) const { return lo == hi && o.lo == o.hi && lo == o.lo && !pad && !o.pad; }
};
// A tile of the other side that a workgroup's rows meet, and for the wave's 32
// rows and either block of 32 of the tile: whether they meet, and whether each
// element has to be looked at.
struct AttnTile {
  int first;  // its first row, -1 behind the last tile
  int flags;
  int head;   // (queries: of the heads that share the keys)
  __device__ __forceinline__ bool sees(int block) const { return (flags >> block) & 1; }
  __device__ __forceinline__ bool part(int block) const { return (flags >> (2 + block)) & 1; }
  __device__ __forceinline__ bool pad() const { return (flags >> 4) & 1; }  // (some of its rows are padding)
  __device__ __forceinline__ bool done(int block) const { return (flags >> (5 + block)) & 1; }  // (the wave meets neither it nor any behind)
};
template <bool KEYS>  // the tiles are keys (else queries)
struct AttnWalk {
  int S, r0, prefix, causal, base;
  int head, heads;  // the walk's turn, and how many
  const int4* ranges;
  uint64_t seen;  // tiles from `base` on that the workgroup meets
  int flags;      // of tile base + lane
  // rows [r, r1) of the workgroup and [a, b) of the other side
  __device__ __forceinline__ bool meets(int a, int b, int r, int r1) const {
    const int k0 = KEYS ? a : r, q1 = min(KEYS ? r1 : b, S);
    return a < S && r < S && !(causal && k0 >= q1 && k0 >= prefix);
  }
  __device__ __forceinline__ bool in_part(int a, int b, int r, int r1) const {
    const int q0 = KEYS ? r : a, k1 = min(KEYS ? b : r1, S);
    return (KEYS && b > S) || (causal && k1 - 1 > q0 && k1 > prefix);
  }
  __device__ __forceinline__ void look() {
    const int t = base + (threadIdx.x & 63), a = t * kAttnTile, w = wave_id() & 3, r = r0 + 32 * w;
    bool any = meets(a, a + kAttnTile, r0, r0 + kAttnRows), s[2], p[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      s[k] = meets(a + 32 * k, a + 32 * k + 32, r, r + 32);
      p[k] = in_part(a + 32 * k, a + 32 * k + 32, r, r + 32);
    }
    bool pad = false;
    if (ranges && any) {
      DocRange all(ranges[r0 / 32]), both(ranges[2 * t]);
      const DocRange own(ranges[r0 / 32 + w]), tile[2] = {both, ranges[2 * t + 1]};
#pragma unroll
      for (int k = 1; k < 4; ++k) all.join(ranges[r0 / 32 + k]);
      both.join(tile[1]);
      any = all.meets(both);
      pad = both.pad;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        s[k] = s[k] && own.meets(tile[k]);
        p[k] = p[k] || !own.one(tile[k]);
      }
    }
    seen = __ballot(any);
    const bool last = (base + 64) * kAttnTile >= S;
    const uint64_t from = __ballot(s[0] || s[1]) >> (threadIdx.x & 63);  // (the wave's, from this tile on)
    flags = s[0] | s[1] << 1 | p[0] << 2 | p[1] << 3 | pad << 4 | (last && !from) << 5 | (last && !s[1] && !(from >> 1)) << 6;
  }
  __device__ __forceinline__ void init(const AttnParams& P, int b, int row0, int turns = 1) {
    head = 0;
    heads = turns;
    S = (int)P.S;
    r0 = row0;
    causal = P.causal;
    prefix = P.prefix ? P.prefix[b] : 0;
    ranges = P.docs ? P.ranges + (int64_t)b * (P.padded / 32) : nullptr;
    base = -64;
    seen = 0;
  }
  __device__ __forceinline__ AttnTile next() {
    while (!seen) {
      base += 64;
      if (base * kAttnTile >= S) {
        if (++head >= heads) {
          head = heads;  // (stays behind the last)
          base -= 64;
          return {-1, 0, 0};
        }
        base = 0;
      }
      look();
    }
    const int j = __builtin_ctzll(seen);
    seen &= seen - 1;
    return {(base + j) * kAttnTile, __builtin_amdgcn_readlane(flags, j), head};
  }
};

// Rows without a document: zeros in LDS, so that whatever they hold (nothing, for
// what lies behind a batch's sequences) is not multiplied by a probability of 0.
template <int LD>
__device__ __forceinline__ void clear_padding(const int* docs, char* one, char* two) {
  constexpr int kChunks = LD / 8;
  for (int p = threadIdx.x; p < kAttnTile * kChunks; p += (int)blockDim.x)
    if (docs[p / kChunks] < 0) {
      reinterpret_cast<uint4*>(one)[p] = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(two)[p] = make_uint4(0, 0, 0, 0);
    }
  __syncthreads();
}

// The row, relative to a block of 32, of element r of the lane's 16.
__device__ __forceinline__ int block_row(int r) { return (r >> 2) * 8 + ((threadIdx.x & 63) >> 5) * 4 + (r & 3); }

// z = -inf for what is not seen.  Keys in the rows: those below `bound` (behind
// the query and its prefix, the sequence's end) are seen; queries in the rows:
// those from `bound` on.  Relative to the block of 32 at row `at`; docs, ranges:
// the numbers and their ranges, or null, read by scalar loads (a vector load would
// wait for the DMA in flight).  A block within one document takes one comparison
// a lane; of others the lower half of a wave compares four rows and the upper half
// the next four (12 heads of 80, 3 rows of one document of 1777: forward 49 us
// instead of 76).
template <bool KEYS>
__device__ __forceinline__ void hide(f32x16& z, int bound, const int* docs, const int4* ranges, int at, int doc) {
  const int own = doc < 0 ? -2 : doc;  // (padding sees nothing, padding neither)
  bound -= at;
  bool mixed = false;
  if (docs) {
    const auto* range = (const __attribute__((address_space(4))) int*)(uintptr_t)(ranges + at / 32);
    mixed = range[0] != range[1] || range[2];
    if (!mixed && own != range[0]) bound = KEYS ? -1 : 32;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = block_row(r);
    z[r] = (KEYS ? row < bound : row >= bound) ? z[r] : -kInf;
  }
  if (mixed) {
    const auto* d = (const __attribute__((address_space(4))) int*)(uintptr_t)(docs + at);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = (r >> 2) * 8 + (r & 3);
      const uint64_t low = __ballot(own == d[i]), high = __ballot(own == d[i + 4]);
      const uint64_t seen = (low & 0xffffffffull) | (high & 0xffffffff00000000ull);
      z[r] = __builtin_amdgcn_inverse_ballot_w64(seen) ? z[r] : -kInf;
    }
  }
}

// Scores from products s = q.k.  Without a cap in units of the products, s - slope
// / |scale| |i - j|, and what uses them multiplies by mul = |scale| log2(e); with
// one in units of log2 (mul = 1), log2(e) (cap tanh(scale s / cap) - slope |i - j|),
// and also the tanh.  slope: slope_of's.  dist: the lane's row less the block's
// first.  (A negative scale is turned over to one of the operands.)
//
// tanh u = 1 - 2 / (1 + e^2u) on the hardware's exp2 and reciprocal is off by 2e-7
// whatever u is, and cap tanh u by 2e-7 cap.  CAP_SMALL takes that (128: 2e-5, a
// 25th of half a step of an fp16 probability).  CAP_ANY has below |u| = 1/4 the
// series u (1 - u^2/3 + 2 u^4/15 - 17 u^6/315 + 62 u^8/2835), whose next term is 9e-9
// of it, so that the capped score is off by at most 2^-18 of itself at any cap.
// (3 x 1777 rows of 12 heads of 80, forward, dq, dk and dv: 67, 82 and 122 us with
// CAP_SMALL, 100, 119 and 171 with CAP_ANY.)
// A slope is taken for what keeps a whole sequence's distance from it below 2^30 in
// log2 (2^24 positions: 64 each), so that no exponent passes fp32's range, and a
// negative one, whose far keys have the largest scores, below 2^22, where fp32 holds
// a score to a quarter.
__device__ __forceinline__ float slope_of(const AttnParams& P, float given) {
  const float s = given * P.slope_mul;
  return s > P.slope_high ? P.slope_high : s < P.slope_low ? P.slope_low : s;
}
template <int CAP, bool BIAS>
__device__ __forceinline__ void scores(f32x16& z, float (&th)[16], const AttnParams& P, float slope, int dist) {
  if constexpr (CAP || BIAS) {
    const float from = (float)(dist - block_row(0));  // (exact: lengths are below 2^24)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (CAP) {
        const float s = z[r], twice = s * P.cap_in, part = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(twice));
        th[r] = fmaf(-2.0f, part, 1.0f);
        z[r] = fmaf(-2.0f * P.cap_out, part, P.cap_out);
        if constexpr (CAP == CAP_ANY) {
          const float u = twice * 0.34657359f, w = u * u;  // (ln(2) / 2)
          const float poly = fmaf(w, fmaf(w, fmaf(w, fmaf(w, 0.021869489f, -0.053968254f), 0.13333333f), -0.33333333f), 1.0f);
          if (w < 0.0625f) {
            th[r] = u * poly;
            z[r] = s * P.scale_log2 * poly;
          }
        }
      }
      if constexpr (BIAS) z[r] = fmaf(-slope, fabsf(from - (float)((r >> 2) * 8 + (r & 3))), z[r]);
    }
  }
}

__device__ __forceinline__ uint32_t lds_at(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p; }

// ------------------------------------------------------------- the pipeline
// The walk over a workgroup's tiles, block by block of 32 rows, with the products
// of the next block (`ahead`) in the same straight piece of code as the softmax
// of this one, so that the matrix cores run under it.
//
// Operands that only `ahead` reads have two slots in LDS, those that the products
// behind the softmax read too three.  Half way through a tile the workgroup
// meets: then the next tile has arrived (it was sent for a tile earlier), and
// nobody reads the tile before this one any more, nor this one's `ahead`
// operands, so that the tile after the next goes there.
//
// f.issue(tile, two, three), f.ready(tile, two, three): the tile sent for, in that
// slot of the two and of the three; arrived.  f.ahead<BLOCK>(two): products of that
// block of the tile, into the BLOCK-th set of registers.  f.work<BLOCK>(tile,
// three, two): the block's softmax and what follows, beside `ahead` of the next
// block, which is in slot `two` (behind the last tile: of what lies in LDS,
// unused).
template <class F>
__device__ __forceinline__ void attn_walk(AttnWalk<true>& walk, F& f) {
  AttnTile t0 = walk.next();
  if (t0.first < 0) return;
  AttnTile t1 = walk.next();
  int two = 0, three = 0, after = 1, behind = 2;
  f.issue(t0, 0, 0);
  if (t1.first >= 0) f.issue(t1, 1, 1);
  wait_vmem<0>();
  tile_barrier();
  f.ready(t0, 0, 0);
  if (t1.first >= 0) f.ready(t1, 1, 1);
  f.template ahead<0>(0);
  for (bool sent = true;; sent = false) {  // (sent: the first two tiles have arrived)
    if (!t0.done(0)) f.template work<0>(t0, three, two);
    AttnTile t2{-1, 0, 0};
    if (t1.first >= 0) {
      t2 = walk.next();
      wait_vmem<0>();
      tile_barrier();
      if (t2.first >= 0) f.issue(t2, two, behind);
      if (!sent) f.ready(t1, two ^ 1, after);
    }
    if (!t0.done(1)) f.template work<1>(t0, three, two ^ 1);
    if (t1.first < 0) return;
    t0 = t1;
    t1 = t2;
    two ^= 1;
    const int free = three;
    three = after;
    after = behind;
    behind = free;
  }
}

// The same without products ahead, where the registers do not hold them and two
// waves of a SIMD run beside each other: two slots, f.work<BLOCK>(tile, slot).
template <bool KEYS, class F>
__device__ __forceinline__ void attn_walk_plain(AttnWalk<KEYS>& walk, F& f) {
  AttnTile t = walk.next();
  if (t.first < 0) return;
  f.issue(t, 0);
  for (int slot = 0;; slot ^= 1) {
    const AttnTile then = walk.next();
    wait_vmem<0>();
    tile_barrier();
    if (then.first >= 0) f.issue(then, slot ^ 1);
    f.ready(t, slot);
    if (t.sees(0)) f.template work<0>(t, slot);
    if (t.sees(1)) f.template work<1>(t, slot);
    if (then.first < 0) return;
    t = then;
  }
}

// ------------------------------------------------------------- forward
// 2 x 4096 rows of 32 heads (8) of 128 in bf16, causal: 275 GFLOP in 322 us, 854
// TFLOP/s; the matrix cores are busy for 47 % of it, at 1.9 GHz (16 heads without
// others, no mask: 157 us, 875 TFLOP/s; 8 heads, a workgroup to a CU: 104 us, what
// a workgroup's 128 blocks take one after the other).
template <class T, int HD, int CAP, bool BIAS>
struct AttnForward {
  using Frag = typename Traits<T>::Frag;
  static constexpr int kTile = kAttnTile * kAttnLd<HD> * 2, kBlocks = HD / 32, kHalf = kTile / 2;
  const AttnParams& P;
  char *klds, *vlds;  // two slots of K, three of V
  const T *K, *V;
  const int* docs;
  const int4* ranges;
  AttnDma<kAttnLd<HD>> kd, vd;
  AttnFrags<T, HD> fr;
  Frag q[HD / 16], rows[HD / 16];
  f32x16 o[kBlocks];
  f32x16 s[2];
  float m, l, slope;
  float bar;  // (the score from which the maximum follows)
  int row0, i, bound, doc;
  __device__ __forceinline__ AttnForward(const AttnParams& p) : P(p) {}
  __device__ __forceinline__ void issue(const AttnTile& t, int two, int three) {
    kd.issue(K + t.first * P.ks, (int)P.S - t.first, klds + two * kTile);
    vd.issue(V + t.first * P.vs, (int)P.S - t.first, vlds + three * kTile);
  }
  __device__ __forceinline__ void ready(const AttnTile& t, int two, int three) {
    if (t.pad()) clear_padding<kAttnLd<HD>>(docs + t.first, klds + two * kTile, vlds + three * kTile);
  }
  template <int BLOCK>
  __device__ __forceinline__ void fetch(int two) {
    const char* kt = klds + two * kTile + BLOCK * kHalf;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) rows[ks] = fr.rows(kt, ks);
  }
  template <int BLOCK>
  __device__ __forceinline__ void products() {
    f32x16& z = s[BLOCK];
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) z = Traits<T>::mma(rows[ks], q[ks], z);
  }
  template <int BLOCK>
  __device__ __forceinline__ void ahead(int two) {
    fetch<BLOCK>(two);
    products<BLOCK>();
  }
  // what the exponents of 2 have beside x mul
  __device__ __forceinline__ float offset(float mul) const { return kNarrow<T> ? fmaf(-m, mul, kLiftForward<T>) : -m * mul; }
  template <int BLOCK>
  __device__ __forceinline__ void work(const AttnTile& t, int three, int two) {
    const int at = t.first + 32 * BLOCK;
    f32x16& x = s[BLOCK];
    fetch<1 - BLOCK>(two);
    Frag vf[2][kBlocks];
    fr.cols(lds_at(vlds) + (uint32_t)(three * kTile + BLOCK * kHalf), vf);  // (one wait for both)
    float th[16];
    scores<CAP, BIAS>(x, th, P, slope, i - at);
    if (!t.sees(BLOCK)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = -kInf;
    } else if (t.part(BLOCK)) {
      hide<true>(x, bound, docs, ranges, at, doc);
    }
    float top = fmaxf(x[0], x[1]);
#pragma unroll
    for (int r = 2; r < 16; ++r) top = fmaxf(top, x[r]);
    top = halves_max(top);
    const float mul = CAP ? 1.0f : P.scale_log2;
    // The wave's maxima follow only where one grows by more than 2^8: sums and products of
    // probabilities up to 2^8 lose nothing in fp32.  Past 2^20 (far keys behind a steep
    // slope) fp32 holds no eighth of a score, and the maximum's own exponent is the
    // rounding of m mul: in fp16 it follows there wherever it grows, and is taken for 2
    // to 4 steps more, so that no probability passes the type's largest value.
    if (__any(top > bar)) {
      const bool more = top > m, far = kNarrow<T> && fabsf(top * mul) > 0x1p20f;
      const float to = more ? (far ? fmaf(fabsf(top), 0x1p-22f, top) : top) : m;
      const float by = more ? __builtin_amdgcn_exp2f((m - to) * mul) : 1.0f;
      bar = more ? (far ? top : fmaf(8.0f, __builtin_amdgcn_rcpf(mul), top)) : bar;
      m = to;
      l *= by;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= by;
    }
    const float off = m == -kInf ? 0.0f : offset(mul);
    products<1 - BLOCK>();
    float p[16], sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = __builtin_amdgcn_exp2f(fmaf(x[r], mul, off));
      sum[r & 1] += p[r];
    }
    l += sum[0] + sum[1];
    // P is rounded to 16 bits as an operand of the product, its sum is not
    Frag pf[2];
    as_operand<T>(p, pf);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) o[d] = Traits<T>::mma(vf[k][d], pf[k], o[d]);
    // S of the next block beside the exponentials of this one, where the compiler
    // does not see to it (1.5 % of the kernel)
    if constexpr (HD == 128) {
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, 6, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, HD / 16, 0);
    }
  }
};

template <class T, int HD, int CAP, bool BIAS>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void k_attn(AttnParams P) {
  constexpr int kTile = kAttnTile * kAttnLd<HD> * 2, kBlocks = HD / 32;
  __shared__ __attribute__((aligned(1024))) char lds[5 * kTile];
  int bh, q0;
  attn_place(P, blockIdx.x, P.B * P.H, true, bh, q0);
  q0 *= kAttnRows;
  const int b = bh / P.H, head = bh - b * P.H, kv = head / P.group;
  const int lane = threadIdx.x & 63, S = (int)P.S;
  AttnForward<T, HD, CAP, BIAS> f(P);
  f.klds = lds;
  f.vlds = lds + 2 * kTile;
  f.row0 = q0 + wave_id() * 32;
  f.i = f.row0 + (lane & 31);
  f.K = static_cast<const T*>(P.k) + b * P.kb + kv * P.kh;
  f.V = static_cast<const T*>(P.v) + b * P.vb + kv * P.vh;
  f.slope = BIAS ? slope_of(P, P.slopes[head]) : 0.0f;
  f.docs = P.docs ? P.docs + (int64_t)b * P.padded : nullptr;
  f.ranges = P.docs ? P.ranges + (int64_t)b * (P.padded / 32) : nullptr;
  f.doc = P.docs ? f.docs[f.i] : 0;
  AttnWalk<true> walk;
  walk.init(P, b, q0);
  f.bound = P.causal ? min(S, max(f.i + 1, walk.prefix)) : S;
  own_rows<T, HD>(static_cast<const T*>(P.q) + b * P.qb + head * P.qh, P.qs, f.row0, S, P.D, f.q, P.scale < 0.0f);
  f.kd.init(P.ks, P.D);
  f.vd.init(P.vs, P.D);
  f.fr.init();
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) f.o[d][r] = 0.0f;
  f.m = f.bar = -kInf;
  f.l = 0.0f;
  attn_walk(walk, f);
  const float mul = CAP ? 1.0f : P.scale_log2;
  const float l = halves_sum(f.l);
  // (one key alone: its 2^(m mul - m mul) is 1 but for the rounding of one of the
  // two products; o is divided by what it was multiplied by, so that it is v.  The
  // smaller of m and bar is the maximum itself)
  const float off = f.offset(mul), one = __builtin_amdgcn_exp2f(fmaf(fminf(f.m, f.bar), mul, off)), sum = l == one ? to_f32(from_f32<T>(one)) : l;
  const bool empty = !(l > 0.0f) && l == l;
  if (P.lse && lane < 32) P.lse[(int64_t)bh * P.padded + f.i] = f.i >= S || empty ? kInf : __builtin_amdgcn_logf(l) - kLiftBackward<T> - off;
  const int64_t at = (((int64_t)b * S + f.i) * P.H + head) * P.D;
  const float inv = empty ? 0.0f : 1.0f / sum;
  store_own<T, HD>(f.o, inv, static_cast<T*>(P.o) + at, P.D, f.i < S);
  // dz = P (dP - delta) cancels where P is near 1, and delta = sum(do o) would be
  // as far off as o's rounding: for the backward pass o is kept in both halves, at
  // the price of a second tensor of its size, written here and read with dq (67 MB
  // each for 2 x 4096 rows of 32 heads of 128).  dq in bf16 is off by, of its norm,
  //   4096 rows, scores of order 1, 4, 16: 2.4e-3, 2.9e-3, 3.5e-3; without the lower
  //   half 2.5e-3, 3.6e-3, 6.3e-3;  8 rows: 1.7e-3, 1.8e-3, 2.0e-3 for 2.1e-3, 5.4e-3,
  //   3.8e-3  (fp16 alike: 4096 rows 3.0e-4, 3.5e-4, 4.4e-4 for 3.2e-4, 4.4e-4, 8.2e-4)
  if (P.o_low) store_own<T, HD, true>(f.o, inv, static_cast<T*>(P.o_low) + at, P.D, f.i < S);
}

// ------------------------------------------------------------- dq
// Also delta = sum(do o) of each query, which the next kernel reads.  2 x 4096 rows
// of 32 heads (8) of 128 in bf16, causal: 412 GFLOP in 408 us, 1010 TFLOP/s,
// the matrix cores busy for 56 % of it at 1.8 GHz.
template <class T, int HD, int CAP, bool BIAS, bool FINE>
struct AttnGradQ {
  using Frag = typename Traits<T>::Frag;
  static constexpr int kTile = kAttnTile * kAttnLd<HD> * 2, kBlocks = HD / 32, kHalf = kTile / 2;
  const AttnParams& P;
  char *klds, *vlds;  // two slots each
  const T *K, *V;
  const int* docs;
  const int4* ranges;
  AttnDma<kAttnLd<HD>> kd, vd;
  AttnFrags<T, HD> fr;
  Frag q[HD / 16], g[HD / 16];
  f32x16 dq[kBlocks];
  float lse, delta, slope;
  float lift;  // exponent, of dz beside P's
  int row0, i, bound, doc;
  __device__ __forceinline__ AttnGradQ(const AttnParams& p) : P(p) {}
  __device__ __forceinline__ void issue(const AttnTile& t, int slot) {
    kd.issue(K + t.first * P.ks, (int)P.S - t.first, klds + slot * kTile);
    vd.issue(V + t.first * P.vs, (int)P.S - t.first, vlds + slot * kTile);
  }
  __device__ __forceinline__ void ready(const AttnTile& t, int slot) {
    if (t.pad()) clear_padding<kAttnLd<HD>>(docs + t.first, klds + slot * kTile, vlds + slot * kTile);
  }
  template <int BLOCK>
  __device__ __forceinline__ void work(const AttnTile& t, int slot) {
    const int at = t.first + 32 * BLOCK;
    const char *kt = klds + slot * kTile + BLOCK * kHalf, *vt = vlds + slot * kTile + BLOCK * kHalf;
    f32x16 x, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = dp[r] = 0.0f;
    Frag krows[HD / 16], vrows[HD / 16];
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) krows[ks] = fr.rows(kt, ks);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      x = Traits<T>::mma(krows[ks], q[ks], x);
      vrows[ks] = fr.rows(vt, ks);
    }
    auto second = [&] {
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) dp = Traits<T>::mma(vrows[ks], g[ks], dp);
    };
    // Reads go four ahead of the products: by itself the compiler may wait for each
    // (8 heads of 128, 4096: 139 us instead of 124).  Where registers are left the
    // second product comes beside the exponentials (heads of 64: 3 % less).
    constexpr bool kBeside = HD == 64;
    if constexpr (!kBeside) second();
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < HD / 16 * (kBeside ? 1 : 2) - (kBeside ? 0 : 4); ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    if constexpr (!kBeside) __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    float th[16];
    scores<CAP, BIAS>(x, th, P, slope, i - at);
    if (t.part(BLOCK)) hide<true>(x, bound, docs, ranges, at, doc);
    if constexpr (kBeside) second();
    const float mul = CAP ? 1.0f : P.scale_log2;
    float z[16];
    const float off = kNarrow<T> ? lift - lse : -lse;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = __builtin_amdgcn_exp2f(fmaf(x[r], mul, off));
    if constexpr (kBeside)
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x402, 8, 1);
      }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      z[r] *= dp[r] - delta;
      if constexpr (CAP) z[r] *= 1.0f - th[r] * th[r];
    }
    if constexpr (kNarrow<T>) lift -= (float)keep_in_range(z, dq);
    Frag zf[2], kf[2][kBlocks];
    as_operand<T>(z, zf);  // (dz in 16 bits, as an operand of the product)
    fr.cols(lds_at(klds) + (uint32_t)(slot * kTile + BLOCK * kHalf), kf);
    if constexpr (FINE) {
      Frag rest[2];
      rest_operand<T>(z, zf, rest);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) dq[d] = Traits<T>::mma(kf[k][d], rest[k], dq[d]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) dq[d] = Traits<T>::mma(kf[k][d], zf[k], dq[d]);
  }
};

template <class T, int HD, int CAP, bool BIAS, bool FINE>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void k_attn_dq(AttnParams P) {
  constexpr int kTile = kAttnTile * kAttnLd<HD> * 2, kBlocks = HD / 32;
  __shared__ __attribute__((aligned(1024))) char lds[4 * kTile];
  int bh, q0;
  attn_place(P, blockIdx.x, P.B * P.H, true, bh, q0);
  q0 *= kAttnRows;
  const int b = bh / P.H, head = bh - b * P.H, kv = head / P.group;
  const int lane = threadIdx.x & 63, S = (int)P.S;
  AttnGradQ<T, HD, CAP, BIAS, FINE> f(P);
  f.klds = lds;
  f.vlds = lds + 2 * kTile;
  f.row0 = q0 + wave_id() * 32;
  f.i = f.row0 + (lane & 31);
  f.K = static_cast<const T*>(P.k) + b * P.kb + kv * P.kh;
  f.V = static_cast<const T*>(P.v) + b * P.vb + kv * P.vh;
  f.slope = BIAS ? slope_of(P, P.slopes[head]) : 0.0f;
  f.docs = P.docs ? P.docs + (int64_t)b * P.padded : nullptr;
  f.ranges = P.docs ? P.ranges + (int64_t)b * (P.padded / 32) : nullptr;
  f.doc = P.docs ? f.docs[f.i] : 0;
  own_rows<T, HD>(static_cast<const T*>(P.dout) + b * P.gb + head * P.gh, P.gs, f.row0, S, P.D, f.g);
  {
    // The diagonal of o do^T, by the products that make dP: a query that sees one key
    // has o = v, and dP - delta is 0 to the bit.
    typename Traits<T>::Frag o[HD / 16];
    const int64_t at = ((int64_t)b * S * P.H + head) * P.D;
    f32x16 x;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = 0.0f;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      own_rows<T, HD>(static_cast<const T*>(part ? P.o : P.o_low) + at, P.H * P.D, f.row0, S, P.D, o);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) x = Traits<T>::mma(o[ks], f.g[ks], x);
    }
    f.delta = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) f.delta = block_row(r) == (lane & 31) ? x[r] : f.delta;
    f.delta = f.doc < 0 ? 0.0f : halves_sum(f.delta);
    if (lane < 32) P.delta[(int64_t)bh * P.padded + f.i] = f.delta;
  }
  if (!P.dq) return;
  f.lse = P.lse[(int64_t)bh * P.padded + f.i];
  f.lift = kLiftScores<T>;
  AttnWalk<true> walk;
  walk.init(P, b, q0);
  f.bound = P.causal ? min(S, max(f.i + 1, walk.prefix)) : S;
  own_rows<T, HD>(static_cast<const T*>(P.q) + b * P.qb + head * P.qh, P.qs, f.row0, S, P.D, f.q, P.scale < 0.0f);
  f.kd.init(P.ks, P.D);
  f.vd.init(P.vs, P.D);
  f.fr.init();
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) f.dq[d][r] = 0.0f;
  attn_walk_plain(walk, f);
  if (f.doc < 0)  // (what a padding row holds may not be finite)
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) f.dq[d][r] = 0.0f;
  T* out = static_cast<T*>(P.dq) + (((int64_t)b * S + f.i) * P.H + head) * P.D;
  const float unlift = kNarrow<T> ? __builtin_amdgcn_exp2f(-f.lift - kLiftBackward<T>) : 1.0f;
  store_own<T, HD>(f.dq, P.scale * unlift, out, P.D, f.i < S);
}

// ------------------------------------------------------------- dk and dv
struct AttnKeys {  // of a workgroup: batch, key head, first row, the heads it takes (of all that share these keys, or one part)
  int b, kv, part, r0, head, heads;
  __device__ __forceinline__ AttnKeys(const AttnParams& P, int id) {
    int at;
    attn_place(P, id, P.B * P.KV * P.parts, false, at, r0);
    r0 *= kAttnRows;
    part = at % P.parts;
    b = at / P.parts / P.KV;
    kv = at / P.parts - b * P.KV;
    head = kv * P.group + part * P.share;
    heads = min(P.share, P.group - part * P.share);
  }
  __device__ __forceinline__ int64_t row(const AttnParams& P, int key) const { return ((b * P.S + key) * P.KV + kv) * P.D; }
  __device__ __forceinline__ float* partial(const AttnParams& P, int which) const { return P.partial + (which * P.parts + part) * (P.B * P.S * P.KV * P.D); }
};

// A workgroup's 128 keys against the queries of all heads that share them: two
// waves for every 32 keys, on one SIMD.  The first makes P from S = Q k^T and adds
// up dv = P^T do; the second makes dz from P, which it gets through LDS in fp32,
// and dP = do v^T, and adds up dk = dz^T Q.  Each has half of the matrix products
// and half of the registers (dk and dv of 32 keys are 128 of 256).
//
// A phase takes 32 queries, and the workgroup meets behind it.  In phase p the
// first wave starts with the softmax of block p and goes on with the products
// dv of p and S of p + 1; the second starts with the products dk of p - 2 and dP of
// p - 1, whose operands it read in the phase before, and goes on with dz of p - 1:
// while one has the matrix cores the other has the vector unit.  (Either wave's
// product beside its own vector work instead took 158 us against 136: 8 heads of
// 80, 4096.)
//
// 2 x 4096 rows of 32 heads (8) of 128 in bf16, causal: 550 GFLOP in 640 us, 860
// TFLOP/s; the matrix cores are busy for 46 % of it, at 1.9 GHz, LDS for 37 %, and a
// phase waits for its two halves in turn.
template <class T, int HD, int CAP, bool BIAS>
struct AttnGradKV {
  using Frag = typename Traits<T>::Frag;
  static constexpr int kTile = kAttnTile * kAttnLd<HD> * 2, kBlocks = HD / 32, kHalf = kTile / 2;
  static constexpr int kStats = 2 * kAttnTile * 4, kProbs = 4 * 4096;
  static constexpr int kLds = 6 * kTile + 2 * kProbs + 3 * kStats;
  const AttnParams& P;
  // (one object: between two the compiler waits for the DMA into either before it reads the other)
  char *qlds, *glds;  // three slots of Q and of do
  char *probs;        // two blocks of P
  char *stats;        // three of (L, delta) of the queries
  const T *Q, *G;     // of the first head
  const float *lse, *delta, *slopes;
  const int* docs;
  const int4* ranges;
  AttnDma<kAttnLd<HD>> qd, gd;  // of the second waves, which have the matrix cores while they send for a tile
  AttnFrags<T, HD> fr;
  Frag own[HD / 16];  // the wave's keys, or their values
  f32x16 acc[kBlocks];
  f32x16 x;                              // first: S of the next phase's block
  Frag rows[HD / 16], cf[2][kBlocks];    // second: operands of the next phase
  Frag zf[2];                            // second: dz of the last phase's block
  float lift;                            // second: of dz beside P's
  int row0, key, bound, doc;
  __device__ __forceinline__ AttnGradKV(const AttnParams& p) : P(p) {}
  __device__ __forceinline__ void issue(const AttnTile& t, int slot) {
    qd.issue(Q + t.head * P.qh + t.first * P.qs, (int)P.S - t.first, qlds + slot * kTile);
    gd.issue(G + t.head * P.gh + t.first * P.gs, (int)P.S - t.first, glds + slot * kTile);
    const int w = wave_id() & 3;
    if (w < 2)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of((w ? delta : lse) + t.head * P.padded + t.first),
                                               (__attribute__((address_space(3))) void*)(stats + slot * kStats + w * (kStats / 2)), 4,
                                               (threadIdx.x & 63) * 4, 0, 0, 0);
  }
  __device__ __forceinline__ void ready(const AttnTile& t, int slot) {
    if (t.pad()) clear_padding<kAttnLd<HD>>(docs + t.first, qlds + slot * kTile, glds + slot * kTile);
  }
  __device__ __forceinline__ char* qrows(int slot, int block) const { return qlds + slot * kTile + block * kHalf; }
  __device__ __forceinline__ char* grows(int slot, int block) const { return glds + slot * kTile + block * kHalf; }
  __device__ __forceinline__ void fetch(const char* at) {
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) rows[ks] = fr.rows(at, ks);
  }
  __device__ __forceinline__ void product(f32x16& z) {
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) z = Traits<T>::mma(rows[ks], own[ks], z);
  }
  __device__ __forceinline__ void add_up(const Frag (&f)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) acc[d] = Traits<T>::mma(cf[j][d], f[j], acc[d]);
  }
  // four consecutive queries of the lane's rows at a time
  __device__ __forceinline__ const char* stat(int slot, int block, int which) const {
    return stats + slot * kStats + which * (kStats / 2) + 128 * block + ((threadIdx.x & 63) >> 5) * 16;
  }
  __device__ __forceinline__ char* prob(int buffer) const { return probs + buffer * kProbs + (wave_id() & 3) * 4096 + (threadIdx.x & 63) * 16; }
  // The first wave's phase: block BLOCK of tile t in `slot`; `then`: S of the block
  // behind it, block 1 - BLOCK of the tile in slot `to`.
  template <int BLOCK>
  __device__ __forceinline__ void lead(const AttnTile& t, int slot, bool then, int to) {
    const int at = t.first + 32 * BLOCK;
    if (then) fetch(qrows(to, 1 - BLOCK));
    if (t.sees(BLOCK)) {
      f4v L[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) L[g] = *reinterpret_cast<const f4v*>(stat(slot, BLOCK, 0) + 32 * g);
      fr.cols(lds_at(grows(slot, BLOCK)), cf);
      float th[16], p[16];
      scores<CAP, BIAS>(x, th, P, BIAS ? slope_of(P, slopes[t.head]) : 0.0f, key - at);
      if (t.part(BLOCK)) hide<false>(x, bound, docs, ranges, at, doc);
      const float mul = CAP ? 1.0f : P.scale_log2;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f4v out;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          p[r] = __builtin_amdgcn_exp2f(fmaf(x[r], mul, -L[g][e]));  // (queries behind the last, or that see nothing: L = inf)
          out[e] = CAP ? p[r] * (1.0f - th[r] * th[r]) : p[r];
        }
        *reinterpret_cast<f4v*>(prob(BLOCK) + g * 1024) = out;
      }
      Frag pf[2];
      as_operand<T>(p, pf);
      add_up(pf);
    }
    if (then) product(x);
  }
  // The second wave's: dk of block BLOCK of tile u (has: there is one), dz of
  // block 1 - BLOCK of tile t in `slot` (here: there is one), and the operands of
  // the next phase, dP of block BLOCK of the tile in slot `to` (more: there is
  // one) and dk of the block whose dz this is.
  template <int BLOCK>
  __device__ __forceinline__ void follow(const AttnTile& u, bool has, const AttnTile& t, int slot, bool here, int to, bool more) {
    constexpr int kOther = 1 - BLOCK;
    float z[16];
    const bool made = here && t.sees(kOther);
    if (has && u.sees(BLOCK)) add_up(zf);
    if (made) {
      f32x16 dp;
      f4v dl[4], p[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        dl[g] = *reinterpret_cast<const f4v*>(stat(slot, kOther, 1) + 32 * g);
        p[g] = *reinterpret_cast<const f4v*>(prob(kOther) + g * 1024);
      }
      product(dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        z[r] = p[r >> 2][r & 3] * (dp[r] - dl[r >> 2][r & 3]);
        if constexpr (kNarrow<T>) z[r] *= lift;
      }
      if constexpr (kNarrow<T>) lift = __builtin_amdgcn_ldexpf(lift, -keep_in_range(z, acc));
      as_operand<T>(z, zf);
    }
    if (more) fetch(grows(to, BLOCK));
    if (here) fr.cols(lds_at(qrows(slot, kOther)), cf);
    if (P.fine && made) {
      Frag rest[2];
      rest_operand<T>(z, zf, rest);
      add_up(rest);
    }
  }
  // (a loop of its own for each of the two: in one, what either holds would take
  // registers of both)
  template <bool LEADS>
  __device__ __forceinline__ void walk(AttnWalk<false>& w) {
    AttnTile t0 = w.next(), last = t0;
    if (t0.first < 0) return;
    AttnTile t1 = w.next();
    if constexpr (!LEADS) {
      issue(t0, 0);
      if (t1.first >= 0) issue(t1, 1);
      wait_vmem<0>();
    }
    tile_barrier();
    ready(t0, 0);
    if constexpr (LEADS) {
      if (t0.sees(0)) {
        fetch(qrows(0, 0));
        product(x);
      }
    }
    int slot = 0, after = 1, behind = 2;  // of t0, t1, and the tile before t0
    for (bool first = true;; first = false) {
      if constexpr (LEADS) lead<0>(t0, slot, t0.sees(1), slot);
      else follow<0>(last, !first, last, behind, !first, slot, true);
      if constexpr (!LEADS) wait_vmem<0>();  // (t1, sent for two phases ago)
      tile_barrier();
      const AttnTile t2 = w.next();
      if constexpr (!LEADS)
        if (t2.first >= 0) issue(t2, behind);  // (whose last block was read in the phase before)
      const bool more = t1.first >= 0;
      if (more) ready(t1, after);
      if constexpr (LEADS) lead<1>(t0, slot, t1.sees(0), after);
      else follow<1>(last, !first, t0, slot, true, slot, true);
      tile_barrier();
      last = t0;
      if (!more) break;
      t0 = t1;
      t1 = t2;
      const int free = behind;
      behind = slot;
      slot = after;
      after = free;
    }
    if constexpr (!LEADS) {
      follow<0>(last, true, last, slot, true, slot, false);
      if (last.sees(1)) add_up(zf);
    }
  }
};

template <class T, int HD, int CAP, bool BIAS>
__global__ __launch_bounds__(512, 2) void k_attn_dkv(AttnParams P) {
  using F = AttnGradKV<T, HD, CAP, BIAS>;
  constexpr int kBlocks = HD / 32;
  constexpr float kUnlift = kNarrow<T> ? 1.0f / 1024.0f : 1.0f;  // 2^-kLiftBackward
  __shared__ __attribute__((aligned(1024))) char lds[F::kLds];
  const AttnKeys at(P, blockIdx.x);
  const int b = at.b, kv = at.kv, r0 = at.r0, head = at.head;
  const int lane = threadIdx.x & 63, S = (int)P.S, w = wave_id();
  const bool leads = w < 4;
  F f(P);
  f.qlds = lds;
  f.glds = lds + 3 * F::kTile;
  f.probs = lds + 6 * F::kTile;
  f.stats = f.probs + 2 * F::kProbs;
  f.row0 = r0 + (w & 3) * 32;
  f.key = f.row0 + (lane & 31);
  f.docs = P.docs ? P.docs + (int64_t)b * P.padded : nullptr;
  f.ranges = P.docs ? P.ranges + (int64_t)b * (P.padded / 32) : nullptr;
  f.doc = P.docs ? f.docs[f.key] : 0;
  const int prefix = P.prefix ? P.prefix[b] : 0;
  f.bound = P.causal && f.key >= prefix ? f.key : 0;
  f.Q = static_cast<const T*>(P.q) + b * P.qb + head * P.qh;
  f.G = static_cast<const T*>(P.dout) + b * P.gb + head * P.gh;
  f.lse = P.lse + ((int64_t)b * P.H + head) * P.padded;
  f.delta = P.delta + ((int64_t)b * P.H + head) * P.padded;
  f.slopes = BIAS ? P.slopes + head : nullptr;
  f.qd.init(P.qs, P.D);
  f.gd.init(P.gs, P.D);
  f.fr.init();
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) f.acc[d][r] = 0.0f;
  f.lift = __builtin_amdgcn_exp2f(kLiftScores<T>);
  AttnWalk<false> walk;
  walk.init(P, b, r0, at.heads);
  // (zeros for a padding row: what it holds may not be finite)
  auto finish = [&](T* out, int which, float mul, float unlift) {
    if (f.doc < 0)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) f.acc[d][r] = 0.0f;
    int id = blockIdx.x;
    asm volatile("" : "+s"(id));  // (where the sums go is worked out again: the loop has no registers for it)
    const AttnKeys to(P, id);
    const int64_t row = to.row(P, f.key);
    if (P.partial) store_part<HD>(f.acc, unlift, to.partial(P, which) + row, P.D, f.key < P.S);
    else if (out) store_own<T, HD>(f.acc, mul * unlift, out + row, P.D, f.key < P.S);
  };
  if (leads) {
    own_rows<T, HD>(static_cast<const T*>(P.k) + b * P.kb + kv * P.kh, P.ks, f.row0, S, P.D, f.own, P.scale < 0.0f);
    f.template walk<true>(walk);
    finish(static_cast<T*>(P.dv), 1, 1.0f, kUnlift);
  } else {
    own_rows<T, HD>(static_cast<const T*>(P.v) + b * P.vb + kv * P.vh, P.vs, f.row0, S, P.D, f.own);
    f.template walk<false>(walk);
    finish(static_cast<T*>(P.dk), 0, P.scale, kUnlift / f.lift);
  }
}

// Heads of up to 64: both sums fit one wave's registers, no P goes through LDS, and
// two workgroups of a CU run beside each other (4096 tokens and 16 heads: 151 us
// instead of 202, 64 heads: 594 instead of 788).  96 columns would not fit: 23
// registers in scratch, and 202 us instead of 141 for 8 heads of 80, 1036 instead of
// 1072 for 64.
template <class T, int CAP, bool BIAS, bool FINE>
struct AttnGradBoth {
  static constexpr int HD = 64;
  using Frag = typename Traits<T>::Frag;
  static constexpr int kTile = kAttnTile * kAttnLd<HD> * 2, kBlocks = HD / 32, kHalf = kTile / 2;
  static constexpr int kStats = 2 * kAttnTile * 4, kLds = 4 * kTile + 2 * kStats;
  const AttnParams& P;
  char *qlds, *glds;  // two slots of Q and of do
  char *stats;        // two of (L, delta) of the queries
  const T *Q, *G;     // of the first head
  const float *lse, *delta, *slopes;
  const int* docs;
  const int4* ranges;
  AttnDma<kAttnLd<HD>> qd, gd;
  AttnFrags<T, HD> fr;
  Frag k[HD / 16], v[HD / 16];
  f32x16 dk[kBlocks], dv[kBlocks];
  float lift;  // of dz beside P's
  float slope;  // the tile's head's
  int row0, key, bound, doc;
  __device__ __forceinline__ AttnGradBoth(const AttnParams& p) : P(p) {}
  __device__ __forceinline__ void issue(const AttnTile& t, int slot) {
    qd.issue(Q + t.head * P.qh + t.first * P.qs, (int)P.S - t.first, qlds + slot * kTile);
    gd.issue(G + t.head * P.gh + t.first * P.gs, (int)P.S - t.first, glds + slot * kTile);
    const int w = wave_id();
    if (w < 2)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of((w ? delta : lse) + t.head * P.padded + t.first),
                                               (__attribute__((address_space(3))) void*)(stats + slot * kStats + w * (kStats / 2)), 4,
                                               (threadIdx.x & 63) * 4, 0, 0, 0);
  }
  __device__ __forceinline__ void ready(const AttnTile& t, int slot) {
    if constexpr (BIAS) slope = slope_of(P, slopes[t.head]);
    if (t.pad()) clear_padding<kAttnLd<HD>>(docs + t.first, qlds + slot * kTile, glds + slot * kTile);
  }
  template <int BLOCK>
  __device__ __forceinline__ void work(const AttnTile& t, int slot) {
    const int at = t.first + 32 * BLOCK;
    const char *qt = qlds + slot * kTile + BLOCK * kHalf, *gt = glds + slot * kTile + BLOCK * kHalf;
    const char* st = stats + slot * kStats + 128 * BLOCK + ((threadIdx.x & 63) >> 5) * 16;
    f32x16 x, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = dp[r] = 0.0f;
    Frag rows[HD / 16], cf[2][kBlocks];
    f4v stat[4];
    auto fetch = [&](const char* from, Frag (&to)[HD / 16]) {
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) to[ks] = fr.rows(from, ks);
    };
    auto stats_of = [&](int which) {
#pragma unroll
      for (int g = 0; g < 4; ++g) stat[g] = *reinterpret_cast<const f4v*>(st + which * (kStats / 2) + 32 * g);
    };
    fetch(qt, rows);
    stats_of(0);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) x = Traits<T>::mma(rows[ks], k[ks], x);
    fetch(gt, rows);
    fr.cols(lds_at(gt), cf);
    float th[16], p[16];
    scores<CAP, BIAS>(x, th, P, slope, key - at);
    if (t.part(BLOCK)) hide<false>(x, bound, docs, ranges, at, doc);
    const float mul = CAP ? 1.0f : P.scale_log2;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) dp = Traits<T>::mma(rows[ks], v[ks], dp);
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(fmaf(x[r], mul, -stat[r >> 2][r & 3]));  // (queries behind the last, or that see nothing: L = inf)
    Frag f[2];
    as_operand<T>(p, f);
    if constexpr (CAP)
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] *= 1.0f - th[r] * th[r];
    stats_of(1);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) dv[d] = Traits<T>::mma(cf[j][d], f[j], dv[d]);
    fr.cols(lds_at(qt), cf);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] *= dp[r] - stat[r >> 2][r & 3];
      if constexpr (kNarrow<T>) p[r] *= lift;
    }
    if constexpr (kNarrow<T>) lift = __builtin_amdgcn_ldexpf(lift, -keep_in_range(p, dk));
    as_operand<T>(p, f);
    if constexpr (FINE) {
      Frag rest[2];
      rest_operand<T>(p, f, rest);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) dk[d] = Traits<T>::mma(cf[j][d], rest[j], dk[d]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) dk[d] = Traits<T>::mma(cf[j][d], f[j], dk[d]);
  }
};

template <class T, int CAP, bool BIAS, bool FINE>
__global__ __launch_bounds__(256, 2) void k_attn_dkv_one(AttnParams P) {
  using F = AttnGradBoth<T, CAP, BIAS, FINE>;
  constexpr int HD = F::HD, kBlocks = F::kBlocks;
  constexpr float kUnlift = kNarrow<T> ? 1.0f / 1024.0f : 1.0f;  // 2^-kLiftBackward
  __shared__ __attribute__((aligned(1024))) char lds[F::kLds];
  const AttnKeys at(P, blockIdx.x);
  const int b = at.b, kv = at.kv, r0 = at.r0, head = at.head;
  const int lane = threadIdx.x & 63, S = (int)P.S;
  F f(P);
  f.qlds = lds;
  f.glds = lds + 2 * F::kTile;
  f.stats = lds + 4 * F::kTile;
  f.row0 = r0 + wave_id() * 32;
  f.key = f.row0 + (lane & 31);
  f.docs = P.docs ? P.docs + (int64_t)b * P.padded : nullptr;
  f.ranges = P.docs ? P.ranges + (int64_t)b * (P.padded / 32) : nullptr;
  f.doc = P.docs ? f.docs[f.key] : 0;
  const int prefix = P.prefix ? P.prefix[b] : 0;
  f.bound = P.causal && f.key >= prefix ? f.key : 0;
  f.Q = static_cast<const T*>(P.q) + b * P.qb + head * P.qh;
  f.G = static_cast<const T*>(P.dout) + b * P.gb + head * P.gh;
  f.lse = P.lse + ((int64_t)b * P.H + head) * P.padded;
  f.delta = P.delta + ((int64_t)b * P.H + head) * P.padded;
  f.slopes = BIAS ? P.slopes + head : nullptr;
  f.qd.init(P.qs, P.D);
  f.gd.init(P.gs, P.D);
  f.fr.init();
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) f.dk[d][r] = f.dv[d][r] = 0.0f;
  own_rows<T, HD>(static_cast<const T*>(P.k) + b * P.kb + kv * P.kh, P.ks, f.row0, S, P.D, f.k, P.scale < 0.0f);
  own_rows<T, HD>(static_cast<const T*>(P.v) + b * P.vb + kv * P.vh, P.vs, f.row0, S, P.D, f.v);
  f.lift = __builtin_amdgcn_exp2f(kLiftScores<T>);
  AttnWalk<false> walk;
  walk.init(P, b, r0, at.heads);
  attn_walk_plain(walk, f);
  const int64_t row = at.row(P, f.key);
  const bool live = f.key < S;
  if (f.doc < 0)  // (zeros for a padding row: what it holds may not be finite)
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) f.dk[d][r] = f.dv[d][r] = 0.0f;
  if (P.partial) {
    store_part<HD>(f.dk, kUnlift / f.lift, at.partial(P, 0) + row, P.D, live);
    store_part<HD>(f.dv, kUnlift, at.partial(P, 1) + row, P.D, live);
    return;
  }
  if (P.dk) store_own<T, HD>(f.dk, P.scale * (kUnlift / f.lift), static_cast<T*>(P.dk) + row, P.D, live);
  if (P.dv) store_own<T, HD>(f.dv, kUnlift, static_cast<T*>(P.dv) + row, P.D, live);
}

// ------------------------------------------------------------- launches
template <class T, int HD, int CAP, bool BIAS>
static hipError_t attn_go(AttnParams P, AttnPass pass, hipStream_t s) {
  P.tiles = (int)((P.S + kAttnRows - 1) / kAttnRows);
  const dim3 grid((unsigned)(P.tiles * P.B * (pass == ATTN_DKV ? P.KV * P.parts : P.H)));
  switch (pass) {
    case ATTN_FORWARD: hipLaunchKernelGGL((k_attn<T, HD, CAP, BIAS>), grid, dim3(256), 0, s, P); break;
    case ATTN_DQ:
      if (P.fine) hipLaunchKernelGGL((k_attn_dq<T, HD, CAP, BIAS, true>), grid, dim3(256), 0, s, P);
      else hipLaunchKernelGGL((k_attn_dq<T, HD, CAP, BIAS, false>), grid, dim3(256), 0, s, P);
      break;
    default:
      if constexpr (HD == 64) {
        if (P.fine) hipLaunchKernelGGL((k_attn_dkv_one<T, CAP, BIAS, true>), grid, dim3(256), 0, s, P);
        else hipLaunchKernelGGL((k_attn_dkv_one<T, CAP, BIAS, false>), grid, dim3(256), 0, s, P);
      } else {
        hipLaunchKernelGGL((k_attn_dkv<T, HD, CAP, BIAS>), grid, dim3(512), 0, s, P);
      }
  }
  return hipGetLastError();
}
template <class T, int HD, int CAP>
static hipError_t attn_bias(const AttnParams& P, AttnPass pass, hipStream_t s) {
  return P.slopes ? attn_go<T, HD, CAP, true>(P, pass, s) : attn_go<T, HD, CAP, false>(P, pass, s);
}
template <class T, int HD>
hipError_t launch_attn(const AttnParams& P, AttnPass pass, hipStream_t s) {
  switch (P.cap) {
    case CAP_NONE: return attn_bias<T, HD, CAP_NONE>(P, pass, s);
    case CAP_SMALL: return attn_bias<T, HD, CAP_SMALL>(P, pass, s);
    default: return attn_bias<T, HD, CAP_ANY>(P, pass, s);
  }
}

}  // namespace orda
