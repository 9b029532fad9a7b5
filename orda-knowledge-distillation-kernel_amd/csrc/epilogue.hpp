// epilogue.hpp -- what the products of the projection (orda_linear_*) and of
// the gated feed-forward block (orda_ffn_*) do with their fp32 accumulators:
// bias, activation, gate product and residual on the way out, or the
// activation's derivative on the way back.  Every engine hands an epilogue W
// consecutive columns of one row, in fp32; each output is rounded once.
#pragma once
#include <type_traits>

#include "orda_core.hpp"

namespace orda {

__host__ __device__ __forceinline__ int64_t lmin(int64_t a, int64_t b) { return a < b ? a : b; }

enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4, ACT_SIGMOID = 5, ACT_COUNT = 6 };

// 1 / (1 + exp(-x)): in fp32 with the library's exp and an exact division,
// for 16-bit outputs on the hardware's exp2 and reciprocal (errors of 1e-6,
// far below half a step of the output).
template <class T>
__device__ __forceinline__ float sigmoid_of(float x) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-x));
  else return __builtin_amdgcn_rcpf(1.0f + fexp(-x));
}

// Phi(x) = erfc(-x / sqrt 2) / 2, which keeps its relative accuracy where
// 1 + erf cancels, and e = exp(-x^2 / 2).  For 16-bit outputs erfc(u) exp(u^2),
// u = |x| / sqrt 2, is t P(t) with t = 1 / (1 + u / 2) and P of degree 6 fitted
// to least relative error on u in [0, 9.5] (iterated reweighted least squares):
// a dozen instructions, where the library's erfc made the epilogue of an 8192 x
// 2048 x 4096 product 80 us of its 186.  The polynomial errs by 1.4e-6 in fp32
// arithmetic; Phi by 1.9e-6 of its value above x = -5 and, through the rounding
// of the exponent's argument, by up to 8.2e-6 down to x = -13 (half a step of
// fp16 is 2.4e-4 or more).
template <class T>
__device__ __forceinline__ float normal_cdf(float x, float& e) {
  if constexpr (sizeof(T) == 4) {
    e = expf(-0.5f * x * x);
    return 0.5f * erfcf(x * -0.70710678118654752f);
  } else {
    e = __builtin_amdgcn_exp2f(-0.72134752f * x * x);
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(x), 0.35355339f, 1.0f));
    float p = 0.08912547f;
    p = fmaf(p, t, -0.35998616f);
    p = fmaf(p, t, 0.39377975f);
    p = fmaf(p, t, 0.03465823f);
    p = fmaf(p, t, 0.28271983f);
    p = fmaf(p, t, 0.27735361f);
    p = fmaf(p, t, 0.28234809f);
    const float q = 0.5f * p * t * e;
    return x < 0.0f ? q : 1.0f - q;
  }
}

// f = act(x), and with GRAD also df = act'(x).
//   relu: a NaN stays one.  gelu: x Phi(x).  gelu_tanh:
//   (1 + tanh u) / 2 = sigmoid(2 u), u = sqrt(2 / pi) (x + 0.044715 x^3).
// `kind` is uniform over the grid (a scalar branch).
template <class T, bool GRAD, int W>
__device__ __forceinline__ void act_eval(int kind, const float (&x)[W], float (&f)[W], float (&df)[W]) {
  switch (kind) {
    case ACT_RELU:
#pragma unroll
      for (int e = 0; e < W; ++e) {
        f[e] = x[e] < 0.0f ? 0.0f : x[e];
        if constexpr (GRAD) df[e] = x[e] <= 0.0f ? 0.0f : 1.0f;
      }
      break;
    case ACT_GELU:
#pragma unroll
      for (int e = 0; e < W; ++e) {
        float g;
        const float phi = normal_cdf<T>(x[e], g);
        f[e] = x[e] * phi;
        if constexpr (GRAD) df[e] = g == 0.0f ? phi : phi + x[e] * (0.3989422804014327f * g);
      }
      break;
    case ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float s = sigmoid_of<T>(1.5957691216057308f * (x[e] + 0.044715f * x[e] * x[e] * x[e]));
        f[e] = x[e] * s;
        if constexpr (GRAD) {
          const float q = s * (1.0f - s);
          df[e] = q == 0.0f ? s : s + x[e] * q * 1.5957691216057308f * (1.0f + 0.134145f * x[e] * x[e]);
        }
      }
      break;
    case ACT_SILU:
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float s = sigmoid_of<T>(x[e]);
        f[e] = x[e] * s;
        if constexpr (GRAD) df[e] = s + x[e] * s * (1.0f - s);
      }
      break;
    case ACT_SIGMOID:
#pragma unroll
      for (int e = 0; e < W; ++e) {
        f[e] = sigmoid_of<T>(x[e]);
        if constexpr (GRAD) df[e] = f[e] * (1.0f - f[e]);
      }
      break;
    default:
#pragma unroll
      for (int e = 0; e < W; ++e) {
        f[e] = x[e];
        if constexpr (GRAD) df[e] = 1.0f;
      }
  }
}

// W consecutive values at any address that is aligned to one of them (the
// hardware's unaligned vector accesses; rows of odd lengths), or the first cnt
// of them.
template <class T, int N>
struct AnyVec {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <class T, int W>
__device__ __forceinline__ void ld_row(const T* p, float (&v)[W], int cnt) {
  constexpr int kE = W * (int)sizeof(T) <= 16 ? W : 16 / (int)sizeof(T);
  typedef typename AnyVec<T, kE>::type vec;
  if (cnt == W) {
#pragma unroll
    for (int i = 0; i < W / kE; ++i) {
      const vec x = *reinterpret_cast<const vec*>(p + i * kE);
#pragma unroll
      for (int e = 0; e < kE; ++e) v[i * kE + e] = to_f32(x[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = e < cnt ? to_f32(p[e]) : 0.0f;
  }
}
template <class T, int W>
__device__ __forceinline__ void st_row(T* p, const float (&v)[W], int cnt) {
  constexpr int kE = W * (int)sizeof(T) <= 16 ? W : 16 / (int)sizeof(T);
  typedef typename AnyVec<T, kE>::type vec;
  if (cnt == W) {
#pragma unroll
    for (int i = 0; i < W / kE; ++i) {
      if constexpr (sizeof(T) == 2) {
        typedef uint32_t words __attribute__((ext_vector_type(kE / 2)));
        words u;
#pragma unroll
        for (int e = 0; e < kE / 2; ++e) u[e] = pack2<T>(v[i * kE + 2 * e], v[i * kE + 2 * e + 1]);
        typedef typename AnyVec<uint16_t, kE>::type half_words;
        *reinterpret_cast<half_words*>(p + i * kE) = __builtin_bit_cast(half_words, u);
      } else {
        vec x;
#pragma unroll
        for (int e = 0; e < kE; ++e) x[e] = v[i * kE + e];
        *reinterpret_cast<vec*>(p + i * kE) = x;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (e < cnt) p[e] = from_f32<T>(v[e]);
  }
}

// W consecutive values as they lie in memory: loaded early, unpacked later.
template <class T, int W>
struct RawRow {
  typedef T vec __attribute__((ext_vector_type(W)));
  vec v;
  __device__ __forceinline__ void load(const T* p, int cnt) {
    if (cnt == W) {
      v = *reinterpret_cast<const typename AnyVec<T, W>::type*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = e < cnt ? p[e] : (T)0.0f;
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return to_f32(v[e]); }
};

// Factors that the backward pass multiplies by.  For 16-bit tensors they are
// kept in 24 bits, an fp32 value's sign, exponent and first 15 bits, in a plane
// of 16-bit halves and a plane of bytes: rounded to bf16 they made the gradients
// of the feed-forward block 1.8 times as far off float64 as one rounding at the
// end, with 24 bits 1.4 times (da and db are rounded as operands).  Rounded to
// nearest, ties away from zero, so that sums over many tokens see no one-sided
// error; half a step is 2^-16 of the value.  (Adding half a step to the bits
// carries into the exponent as it should and leaves infinities; a NaN that came
// from 16-bit operands or from arithmetic has zeros in the bits it could carry
// out of.)  fp32: as is, in the first plane.
// i: index of the first of W values, a multiple of W.
template <class T>
constexpr int kKeptBytes = sizeof(T) == 4 ? 4 : 3;
struct Planes {
  char* hi;
  char* lo;
  // the planes from value i on
  template <class T>
  __device__ __forceinline__ Planes from(int64_t i) const {
    return {hi + i * (sizeof(T) == 4 ? 4 : 2), lo + i};
  }
};
template <class T>
__host__ inline Planes planes(const void* base, int64_t values) {
  char* p = static_cast<char*>(const_cast<void*>(base));
  return {p, p ? p + 2 * values : nullptr};
}
template <class T, int W>
__device__ __forceinline__ void keep(const Planes& p, uint32_t i, const float (&v)[W]) {
  if constexpr (sizeof(T) == 4) {
    st_row<float, W>(reinterpret_cast<float*>(p.hi + i * 4), v, W);
  } else {
    uint32_t r[W], h[W / 2], l[W / 4];
#pragma unroll
    for (int e = 0; e < W; ++e) r[e] = __float_as_uint(v[e]) + 0x80u;
#pragma unroll
    for (int e = 0; e < W / 2; ++e) h[e] = __builtin_amdgcn_perm(r[2 * e + 1], r[2 * e], 0x07060302u);
#pragma unroll
    for (int e = 0; e < W / 4; ++e) {
      const uint32_t a = __builtin_amdgcn_perm(r[4 * e + 1], r[4 * e], 0x0c0c0501u);
      const uint32_t b = __builtin_amdgcn_perm(r[4 * e + 3], r[4 * e + 2], 0x0c0c0501u);
      l[e] = a | (b << 16);
    }
    if constexpr (W == 4) {
      *reinterpret_cast<uint2*>(p.hi + i * 2) = make_uint2(h[0], h[1]);
      *reinterpret_cast<uint32_t*>(p.lo + i) = l[0];
    } else {
      *reinterpret_cast<uint4*>(p.hi + i * 2) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint2*>(p.lo + i) = make_uint2(l[0], l[1]);
    }
  }
}
template <class T, int W>
struct Kept {
  typedef uint32_t hv __attribute__((ext_vector_type(sizeof(T) == 4 ? W : W / 2)));
  typedef uint32_t lv __attribute__((ext_vector_type(W / 4)));
  hv h;
  lv l;
  __device__ __forceinline__ void load(const Planes& p, uint32_t i) {
    if constexpr (sizeof(T) == 4) {
      h = *reinterpret_cast<const hv*>(p.hi + i * 4);
    } else {
      h = *reinterpret_cast<const hv*>(p.hi + i * 2);
      l = *reinterpret_cast<const lv*>(p.lo + i);
    }
  }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(h[e]);
    // value e: half e % 2 of h[e / 2] above byte e % 4 of l[e / 4], as bytes h1 h0 l 0
    constexpr uint32_t kSel[4] = {0x0504000cu, 0x0706010cu, 0x0504020cu, 0x0706030cu};
    if constexpr (W == 4) return __uint_as_float(__builtin_amdgcn_perm(h[e / 2], ((const uint32_t&)l), kSel[e % 4]));
    else return __uint_as_float(__builtin_amdgcn_perm(h[e / 2], l[e / 4], kSel[e % 4]));
  }
};

// Epilogues.  E.tile(m0, n0) is the epilogue of a tile: its rows and columns
// count from there, so that an element is a uniform pointer and 32 bits of
// lane offset (at most 256 rows of at most 2^24 bytes): with 64-bit offsets from
// the tensors' own bases 8192 x 2048 x 4096 with gelu took 177 us instead of 174,
// and two row blocks of loads ahead (ring_op.hpp) did not fit the registers.  E(m, n, v[, u], cnt, pre, col) takes W <= 8
// columns n .. of row m, of which cnt are valid; pre<W>(m, n, cnt) and, for what
// depends on the columns alone, col<W>(n, cnt) load what it reads.  epi_apply()
// is all three.  `cols`: columns left from the tile's first one.  kDual: v and u
// are the two products of the same columns.  at(split): the epilogue of one K
// range (partials only); second(): of a pair's second product.
struct NoPre {};

// The element `i` elements on (32 bits of byte offset).
template <class T>
__device__ __forceinline__ T* on(T* p, uint32_t i) {
  return reinterpret_cast<T*>(reinterpret_cast<char*>(const_cast<typename std::remove_const<T>::type*>(p)) + i * (uint32_t)sizeof(T));
}

// y = act(v + bias) + residual; d, when given, keeps act'(v + bias) for the
// backward pass, in rows of ldd (a multiple of 8, at least cols; the columns
// past cols are written too and hold nothing).
template <class T>
struct EpiLinear {
  static constexpr bool kDual = false, kLight = false;
  T* y;
  T* y1;  // the output of a pair's second product
  Planes d;
  const T* bias;
  const T* res;
  int64_t ldy, ldd, ldr, cols;
  int act;
  __device__ __forceinline__ EpiLinear at(int) const { return *this; }
  __device__ __forceinline__ EpiLinear second() const {
    EpiLinear e = *this;
    e.y = y1;
    return e;
  }
  __device__ __forceinline__ EpiLinear tile(int64_t m0, int64_t n0) const {
    EpiLinear e = *this;
    e.y += m0 * ldy + n0;
    if (d.hi) e.d = d.template from<T>(m0 * ldd + n0);
    if (bias) e.bias += n0;
    if (res) e.res += m0 * ldr + n0;
    e.cols -= n0;
    return e;
  }
  template <int W>
  struct Pre {
    RawRow<T, W> r;
  };
  template <int W>
  struct Col {
    RawRow<T, W> b;
  };
  template <int W>
  __device__ __forceinline__ Col<W> col(uint32_t n, int cnt) const {
    Col<W> c;
    if (bias) c.b.load(on(bias, n), cnt);
    return c;
  }
  template <int W>
  __device__ __forceinline__ Pre<W> pre(uint32_t m, uint32_t n, int cnt) const {
    Pre<W> p;
    if (res) p.r.load(on(res, m * (uint32_t)ldr + n), cnt);
    return p;
  }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t m, uint32_t n, float (&v)[W], int cnt, const Pre<W>& p,
                                             const Col<W>& c) const {
    if (bias) {
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] += c.b[e];
    }
    if (act != ACT_NONE) {
      float f[W], df[W];
      if (d.hi) {
        act_eval<T, true, W>(act, v, f, df);
        keep<T, W>(d, m * (uint32_t)ldd + n, df);
      } else {
        act_eval<T, false, W>(act, v, f, df);
      }
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = f[e];
    }
    if (res) {
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] += p.r[e];
    }
    st_row<T, W>(on(y, m * (uint32_t)ldy + n), v, cnt);
  }
};

// v[e] = 0 from e = left on.
template <int W>
__device__ __forceinline__ void zero_from(float (&v)[W], int left) {
  if (left >= W) return;
#pragma unroll
  for (int e = 0; e < W; ++e) v[e] = e < left ? v[e] : 0.0f;
}

// h = act(a) b, rounded to T as the next product's operand; for the backward
// pass, when asked for, the factors p = b act'(a) of da and q = act(a) of db are
// kept: the activation is not evaluated again.  All [M x ld], cols = ld a
// multiple of 64, so that every access is whole and aligned.  Columns past
// `inner` are zeros whatever x holds: 0 * infinity in the product would reach y
// and grad_x through the padding.
template <class T>
struct EpiGate {
  static constexpr bool kDual = true, kLight = false;
  T* h;
  Planes p, q;
  int64_t ld, cols;
  int inner;
  int act;
  __device__ __forceinline__ EpiGate at(int) const { return *this; }
  __device__ __forceinline__ EpiGate second() const { return *this; }  // (no pairs)
  __device__ __forceinline__ EpiGate tile(int64_t m0, int64_t n0) const {
    EpiGate e = *this;
    const int64_t i = m0 * ld + n0;
    e.h += i;
    if (p.hi) {
      e.p = p.template from<T>(i);
      e.q = q.template from<T>(i);
    }
    e.cols -= n0;
    e.inner -= (int)n0;
    return e;
  }
  template <int W> using Pre = NoPre;
  template <int W> using Col = NoPre;
  template <int W>
  __device__ __forceinline__ NoPre pre(uint32_t, uint32_t, int) const { return {}; }
  template <int W>
  __device__ __forceinline__ NoPre col(uint32_t, int) const { return {}; }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t m, uint32_t n, float (&g)[W], float (&u)[W], int, NoPre, NoPre) const {
    const uint32_t o = m * (uint32_t)ld + n;
    zero_from<W>(g, inner - (int)n);
    zero_from<W>(u, inner - (int)n);
    float f[W], df[W];
    if (p.hi) {
      act_eval<T, true, W>(act, g, f, df);
#pragma unroll
      for (int e = 0; e < W; ++e) df[e] *= u[e];
      keep<T, W>(p, o, df);
      keep<T, W>(q, o, f);
    } else {
      act_eval<T, false, W>(act, g, f, df);
    }
#pragma unroll
    for (int e = 0; e < W; ++e) f[e] *= u[e];
    st_row<T, W>(on(h, o), f, W);
  }
};

// From dh (fp32, never rounded): da = dh p, db = dh q, rounded to T as the
// operands of the next products.  da and db are the two halves of rows of ldd;
// cols = ld a multiple of 64; columns past `inner` are zeros.
template <class T>
struct EpiGateGrad {
  static constexpr bool kDual = false, kLight = true;
  T* da;
  T* db;
  Planes p, q;
  int64_t ldd, ld, cols;
  int inner;
  __device__ __forceinline__ EpiGateGrad at(int) const { return *this; }
  __device__ __forceinline__ EpiGateGrad second() const { return *this; }  // (no pairs)
  __device__ __forceinline__ EpiGateGrad tile(int64_t m0, int64_t n0) const {
    EpiGateGrad e = *this;
    e.da += m0 * ldd + n0;
    e.db += m0 * ldd + n0;
    e.p = p.template from<T>(m0 * ld + n0);
    e.q = q.template from<T>(m0 * ld + n0);
    e.cols -= n0;
    e.inner -= (int)n0;
    return e;
  }
  template <int W> using Col = NoPre;
  template <int W>
  __device__ __forceinline__ NoPre col(uint32_t, int) const { return {}; }
  template <int W>
  struct Pre {
    Kept<T, W> p, q;
  };
  template <int W>
  __device__ __forceinline__ Pre<W> pre(uint32_t m, uint32_t n, int) const {
    Pre<W> x;
    x.p.load(p, m * (uint32_t)ld + n);
    x.q.load(q, m * (uint32_t)ld + n);
    return x;
  }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t m, uint32_t n, float (&v)[W], int, const Pre<W>& x, NoPre) const {
    float a[W], b[W];
    zero_from<W>(v, inner - (int)n);
#pragma unroll
    for (int e = 0; e < W; ++e) {
      a[e] = v[e] * x.p[e];
      b[e] = v[e] * x.q[e];
    }
    const uint32_t o = m * (uint32_t)ldd + n;
    st_row<T, W>(on(da, o), a, W);
    st_row<T, W>(on(db, o), b, W);
  }
};

// fp32 partial of one K range: [splits][M][ld], a dual product's second half
// `cols` columns behind its first (p1).  (ld a multiple of 4.)
template <bool DUAL>
struct EpiPart {
  static constexpr bool kDual = DUAL, kLight = false;
  float* p;
  float* p1;
  int64_t stride, ld, cols;
  int64_t half;  // elements of a pair's first product in each split
  __device__ __forceinline__ EpiPart moved(int64_t by) const { return {p + by, p1 + by, stride, ld, cols, half}; }
  __device__ __forceinline__ EpiPart at(int split) const { return moved(split * stride); }
  __device__ __forceinline__ EpiPart second() const { return moved(half); }
  __device__ __forceinline__ EpiPart tile(int64_t m0, int64_t n0) const {
    EpiPart e = moved(m0 * ld + n0);
    e.cols -= n0;
    return e;
  }
  template <int W> using Pre = NoPre;
  template <int W> using Col = NoPre;
  template <int W>
  __device__ __forceinline__ NoPre pre(uint32_t, uint32_t, int) const { return {}; }
  template <int W>
  __device__ __forceinline__ NoPre col(uint32_t, int) const { return {}; }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t m, uint32_t n, float (&v)[W], int cnt, NoPre, NoPre) const {
    st_row<float, W>(on(p, m * (uint32_t)ld + n), v, cnt);
  }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t m, uint32_t n, float (&v)[W], float (&u)[W], int cnt, NoPre, NoPre) const {
    st_row<float, W>(on(p, m * (uint32_t)ld + n), v, cnt);
    st_row<float, W>(on(p1, m * (uint32_t)ld + n), u, cnt);
  }
};

template <class Epi, int W>
__device__ __forceinline__ void epi_apply(const Epi& E, uint32_t m, uint32_t n, float (&v)[W], int cnt) {
  E(m, n, v, cnt, E.template pre<W>(m, n, cnt), E.template col<W>(n, cnt));
}
template <class Epi, int W>
__device__ __forceinline__ void epi_apply(const Epi& E, uint32_t m, uint32_t n, float (&v)[W], float (&u)[W], int cnt) {
  E(m, n, v, u, cnt, E.template pre<W>(m, n, cnt), E.template col<W>(n, cnt));
}

// Sum of the partials in split order, then the epilogue; a thread takes 4
// columns of a row.  cols a multiple of 4.  rows: M, or 2 M of a pair (the
// second product's behind the first's).  The grid has a second dimension past
// 2^22 workgroups (a launch has fewer than 2^32 threads in each).
template <class Epi>
__global__ __launch_bounds__(256) void k_part_reduce(const float* __restrict__ part, int splits, int64_t stride,
                                                     int64_t ld, int64_t M, int64_t rows, int64_t cols, Epi E) {
  const int64_t nq = cols / 4;
  const int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows * nq) return;
  int64_t m = i / nq;
  const int64_t n = (i - m * nq) * 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
  const float* p = part + m * ld + n;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float4 x = *reinterpret_cast<const float4*>(p + s * stride);
    v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
    if constexpr (Epi::kDual) {
      const float4 y = *reinterpret_cast<const float4*>(p + s * stride + cols);
      u[0] += y.x; u[1] += y.y; u[2] += y.z; u[3] += y.w;
    }
  }
  if (m >= M) {
    m -= M;
    E = E.second();
  }
  E = E.tile(m, n);
  const int cnt = E.cols >= 4 ? 4 : (int)E.cols;
  if (cnt <= 0) return;
  if constexpr (Epi::kDual) epi_apply(E, 0, 0, v, u, cnt);
  else epi_apply(E, 0, 0, v, cnt);
}

}  // namespace orda
