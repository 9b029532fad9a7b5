// norms.hip -- the norm over all elements of many tensors, their clipping, and
// copies of operands with padded rows.
//
// A launch takes a table of tensors in its arguments (no copy to the device,
// so it can be captured) and splits their rows into chunks; workgroup b of G
// takes chunks b, b + G, ... .  Both kernels are bound by memory: the norm reads
// every element once, clipping reads and writes it once, from the first 16-byte
// aligned address of a row on.  600 M elements, MI355X: the norm 5.8 TB/s in
// fp32 (torch's sum 4.0), 5.1 in bf16 behind a kernel that wrote 2.4 GB; clipping
// bf16 into fp32 6.5 TB/s, fp32 6.0.  Clipping takes one workgroup per 2048
// elements: with 8192 workgroups of many chunks it ran at 5.0 and 5.4 TB/s, and
// with nontemporal stores at 3.8 and 5.3.  Squares and sums are fp64, so
// neither tiny nor huge gradients lose anything, and every sum has a fixed
// order: a thread's elements, the lanes of a wave, the waves, the workgroups.
#include <algorithm>

#include "epilogue.hpp"
#include "op_launch.hpp"

namespace orda {

// The table of one launch, in its arguments: 80 tensors (4 KB), or 320 (15 KB)
// where there are more.  201 fp32 tensors of 60 M elements in one launch each
// for norm and clipping instead of three: 162 -> 141 us of kernels; 300 of 600 M
// bf16 elements 878 -> 849, 197 -> 93 us of host; 40 tensors in the large table
// 26 -> 32 us a pass (the arguments are copied).
constexpr int kSpanFew = 80, kSpanMany = 320;
template <int ROWS>
struct SpanTable {
  static constexpr int kRows = ROWS;
  int count;
  int chunk;   // elements of a chunk (a multiple of 2048)
  int chunks;  // in all
  int pad;
  struct Row {
    const void* p;
    void* out;
    int64_t cols, ld, ld_out;
    int per_row;  // chunks of a row
    int first;    // the tensor's first chunk
  } t[ROWS];
};

// The chunks of workgroup b (b, b + G, ...: the workgroups that run together
// walk memory side by side): f(tensor, row, the row's first element, elements
// [lo, hi) of the row).  A row's chunks are cut at 16-byte aligned addresses.
template <class T, class Table, class F>
__device__ __forceinline__ void for_chunks(const Table& S, const F& f) {
  int i = 0;
  for (int c = blockIdx.x; c < S.chunks; c += gridDim.x) {
    int n = S.count;  // i: the last tensor that starts at or before c
    while (n - i > 1) {
      const int m = (i + n) / 2;
      if (S.t[m].first <= c) i = m;
      else n = m;
    }
    int k = c - S.t[i].first, row = 0;
    if (S.t[i].per_row <= k) {
      row = k / S.t[i].per_row;
      k -= row * S.t[i].per_row;
    }
    const T* p = static_cast<const T*>(S.t[i].p) + row * S.t[i].ld;
    const int skew = (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));  // elements past an aligned address
    const int64_t lo = (int64_t)k * S.chunk - skew, hi = lmin(lo + S.chunk, S.t[i].cols);
    f(i, row, p, lo, hi);
  }
}

// What a thread adds up in: fp64, and the largest magnitude, which is one of the
// values, in fp32.
template <int KIND>
using NormSum = typename std::conditional<KIND == 0, float, double>::type;
template <int KIND>
__device__ __forceinline__ void norm_add(NormSum<KIND>& s, float x) {
  if constexpr (KIND == 2) s = fma((double)x, (double)x, s);
  else if constexpr (KIND == 1) s += (double)fabsf(x);
  else s = !(fabsf(x) <= s) && s == s ? fabsf(x) : s;  // (a NaN takes its place and stays)
}
template <int KIND, class S>
__device__ __forceinline__ S norm_join(S a, S b) {
  if constexpr (KIND != 0) return a + b;
  else return !(b <= a) && a == a ? b : a;
}

// A 16-byte vector of T as floats.
template <class T>
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      v[2 * i] = lo16<T>(w[i]);
      v[2 * i + 1] = hi16<T>(w[i]);
    } else {
      v[i] = __uint_as_float(w[i]);
    }
  }
}

// partials[b] (+)= workgroup b's share.
template <class T, int KIND, int ROWS>
__global__ __launch_bounds__(256) void k_grad_norm(SpanTable<ROWS> S, double* partials, int first) {
  constexpr int VE = 16 / (int)sizeof(T), U = 4;
  __shared__ NormSum<KIND> red[4];
  NormSum<KIND> s = 0;
  for_chunks<T>(S, [&](int, int, const T* p, int64_t lo, int64_t hi) {
    int64_t e = lo + (int64_t)threadIdx.x * VE;
    for (; e + (U - 1) * 256 * VE + VE <= hi && lo >= 0; e += U * 256 * VE) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const uint4*>(p + e + u * 256 * VE);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[VE];
        unpack16<T>(v[u], x);
#pragma unroll
        for (int i = 0; i < VE; ++i) norm_add<KIND>(s, x[i]);
      }
    }
    for (; e < hi; e += 256 * VE) {
      float x[VE];
      if (e >= 0 && e + VE <= hi) {
        unpack16<T>(*reinterpret_cast<const uint4*>(p + e), x);
#pragma unroll
        for (int i = 0; i < VE; ++i) norm_add<KIND>(s, x[i]);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (e + i >= 0 && e + i < hi) norm_add<KIND>(s, to_f32(p[e + i]));
      }
    }
  });
  for (int m = 1; m < 64; m <<= 1) s = norm_join<KIND>(s, __shfl_xor(s, m));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 4; ++i) s = norm_join<KIND>(s, red[i]);
  partials[blockIdx.x] = first ? (double)s : norm_join<KIND>(partials[blockIdx.x], (double)s);
}

// The norm from n partials, by all 256 threads of a workgroup (valid in all).
template <int KIND>
__device__ __forceinline__ float norm_total(const double* partials, int n) {
  __shared__ double red[4];
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 256) s = norm_join<KIND>(s, partials[i]);
  for (int m = 1; m < 64; m <<= 1) s = norm_join<KIND>(s, __shfl_xor(s, m));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = red[0];
  for (int i = 1; i < 4; ++i) s = norm_join<KIND>(s, red[i]);
  return (float)(KIND == 2 ? sqrt(s) : s);
}
template <int KIND>
__global__ __launch_bounds__(256) void k_grad_total(const double* partials, int n, float* total) {
  const float t = norm_total<KIND>(partials, n);
  if (threadIdx.x == 0) *total = t;
}

// g * min(1, max_norm / (total + 1e-6)); a NaN norm gives a NaN factor.  KIND >=
// 0: every workgroup adds up the norm's partials itself and the first writes
// it, which saves small sets a launch; else *total is there.
struct ClipParams {
  const double* partials;
  int n_partials;
  float* total;
  float max_norm;
  int in_place;
};
template <class T, class O, int KIND, int ROWS>
__global__ __launch_bounds__(256) void k_clip(SpanTable<ROWS> S, ClipParams P) {
  // 16 bytes a lane and access on the wider side: 16 in and 2 x 16 out leave
  // half of each line to another store (bf16 into fp32: 5.1 TB/s, 6.5 so)
  constexpr int VE = sizeof(O) == 4 ? 4 : 16 / (int)sizeof(T);
  typedef T in_vec __attribute__((ext_vector_type(VE)));
  // (outputs at any element: the hardware's unaligned stores)
  typedef O out_vec __attribute__((ext_vector_type(VE), aligned(sizeof(O))));
  float total;
  if constexpr (KIND >= 0) {
    total = norm_total<KIND>(P.partials, P.n_partials);
    if (blockIdx.x == 0 && threadIdx.x == 0) *P.total = total;
  } else {
    total = *P.total;
  }
  float f = P.max_norm / (total + 1e-6f);
  f = f > 1.0f ? 1.0f : f;
  if (P.in_place && f == 1.0f) return;
  auto put = [&](O* o, const in_vec& x) {
    out_vec y;
#pragma unroll
    for (int i = 0; i < VE; ++i) y[i] = from_f32<O>(to_f32(x[i]) * f);
    *reinterpret_cast<out_vec*>(o) = y;
  };
  for_chunks<T>(S, [&](int t, int row, const T* p, int64_t lo, int64_t hi) {
    O* o = static_cast<O*>(S.t[t].out) + row * S.t[t].ld_out;
#pragma unroll 2
    for (int64_t e = lo + (int64_t)threadIdx.x * VE; e < hi; e += 256 * VE) {
      if (e >= 0 && e + VE <= hi) {
        put(o + e, *reinterpret_cast<const in_vec*>(p + e));
      } else {
        for (int i = 0; i < VE; ++i)
          if (e + i >= 0 && e + i < hi) o[e + i] = from_f32<O>(to_f32(p[e + i]) * f);
      }
    }
  });
}

// A thread writes 16 bytes of a destination row: a source piece that lies
// inside its row as one load at the elements' own alignment, a row's last one
// element by element, zeros behind.
template <int ES>
__global__ __launch_bounds__(256) void k_pad_rows(PadParams P) {
  constexpr int VE = 16 / ES;
  typedef typename std::conditional<ES == 2, uint16_t, uint32_t>::type E;
  typedef E vec __attribute__((ext_vector_type(VE), aligned(ES)));
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < P.pieces; i += (int64_t)gridDim.x * 256) {
    int k = 0;
    while (k + 1 < P.n && i >= P.t[k + 1].first) ++k;
    const PadParams::Item& t = P.t[k];
    const int64_t per = t.ld_dst / VE, j = i - t.first, row = j / per, c = (j - row * per) * VE;
    const E* s = reinterpret_cast<const E*>(t.src) + row * t.ld_src + c;
    vec v;
    if (c + VE <= t.cols) {
      v = *reinterpret_cast<const vec*>(s);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = c + e < t.cols ? s[e] : (E)0;
    }
    *reinterpret_cast<uint4*>(t.dst + (row * t.ld_dst + c) * ES) = __builtin_bit_cast(uint4, v);
  }
}

hipError_t launch_pad_rows(const PadParams& P, int esize, hipStream_t s) {
  const int64_t g = (P.pieces + 255) / 256;
  const dim3 grid((unsigned)(g < 4096 ? g : 4096));
  if (esize == 2) hipLaunchKernelGGL((k_pad_rows<2>), grid, dim3(256), 0, s, P);
  else hipLaunchKernelGGL((k_pad_rows<4>), grid, dim3(256), 0, s, P);
  return hipGetLastError();
}

// Whether a span belongs to the tables of this dtype pair (-1: any) and place
// (1: in place, 0: not, -1: either).
static bool taken(const GradSpan& x, int in_dtype, int out_dtype, int place) {
  return x.in_dtype == in_dtype && (out_dtype < 0 || x.out_dtype == out_dtype) && (place < 0 || (x.out == x.p) == (place != 0));
}
// Chunks of one row: cut at 16-byte aligned addresses, so up to one more than
// its elements fill.
static int64_t chunks_of_row(int64_t cols, int dtype, int64_t chunk) {
  const int64_t ve = dtype == DT_F32 ? 4 : 8;
  return (cols + ve - 1 + chunk - 1) / chunk;
}
// Tables of the spans of one dtype pair; go(table, workgroups) per launch.
template <int ROWS, class Go>
static hipError_t tables_of(const GradSpan* g, int64_t n, int in_dtype, int out_dtype, int place, int64_t chunk, int max_groups, const Go& go) {
  const int es = in_dtype == DT_F32 ? 4 : 2;
  SpanTable<ROWS> S;
  S.count = S.chunks = 0;
  S.chunk = (int)chunk;
  S.pad = 0;
  auto flush = [&]() -> hipError_t {
    if (S.count == 0) return hipSuccess;
    const hipError_t e = go(S, S.chunks < max_groups ? S.chunks : max_groups);
    S.count = S.chunks = 0;
    return e;
  };
  for (int64_t i = 0; i < n; ++i) {
    const GradSpan& x = g[i];
    if (!taken(x, in_dtype, out_dtype, place)) continue;
    // a tensor of more chunks than a launch counts is cut into rows that fit
    int64_t r0 = 0, c0 = 0;
    const int64_t most = 1ll << 29;  // chunks of one entry
    while (r0 < x.rows) {
      const int64_t cols = x.rows == 1 ? std::min<int64_t>(x.cols - c0, most * chunk / 2) : x.cols;
      const int64_t per = chunks_of_row(cols, in_dtype, chunk);
      const int64_t rows = std::min<int64_t>(x.rows - r0, std::max<int64_t>(1, most / per));
      if (S.count == ROWS || S.chunks + per * rows > (1ll << 30)) {
        const hipError_t e = flush();
        if (e != hipSuccess) return e;
      }
      typename SpanTable<ROWS>::Row& t = S.t[S.count++];
      const int64_t oe = x.out_dtype == DT_F32 ? 4 : 2;
      t.p = static_cast<const char*>(x.p) + (r0 * x.ld + c0) * es;
      t.out = static_cast<char*>(x.out) + (r0 * x.ld_out + c0) * oe;
      t.cols = cols;
      t.ld = x.ld;
      t.ld_out = x.ld_out;
      t.per_row = (int)per;
      t.first = S.chunks;
      S.chunks += (int)(per * rows);
      if (x.rows == 1) {
        c0 += cols;
        if (c0 >= x.cols) ++r0;
      } else {
        r0 += rows;
      }
    }
  }
  return flush();
}

template <class Go>
static hipError_t for_tables(const GradSpan* g, int64_t n, int in_dtype, int out_dtype, int place, int64_t chunk, int max_groups, const Go& go) {
  int64_t spans = 0;
  for (int64_t i = 0; i < n; ++i) spans += taken(g[i], in_dtype, out_dtype, place);
  return spans > kSpanFew ? tables_of<kSpanMany>(g, n, in_dtype, out_dtype, place, chunk, max_groups, go)
                          : tables_of<kSpanFew>(g, n, in_dtype, out_dtype, place, chunk, max_groups, go);
}

static int64_t elements_of(const GradSpan* g, int64_t n) {
  int64_t total = 0;
  for (int64_t i = 0; i < n; ++i) total += g[i].rows * g[i].cols;
  return total;
}
// Elements of a chunk of the norm: one 16-byte access per thread of bf16 where
// that fills the chip, longer ones for large sets.  Of clipping: 2048.
constexpr int64_t kClipChunk = 2048, kNormLarge = 64ll << 20;
constexpr int kClipGroups = 1 << 23;  // (a launch has fewer than 2^32 threads; past them workgroups take several chunks)
static int64_t norm_chunk(int64_t elements) { return elements < kNormLarge ? 2048 : 16384; }

template <class T, int KIND, int ROWS>
static hipError_t norm_go(const SpanTable<ROWS>& S, double* partials, int groups, int first, hipStream_t s) {
  hipLaunchKernelGGL((k_grad_norm<T, KIND, ROWS>), dim3(groups), dim3(256), 0, s, S, partials, first);
  return hipGetLastError();
}
// The partials of all tensors: every launch has the same workgroups, the first
// one writes all partials.  Returns their number (0: no elements) in *groups: one
// for each chunk, of which every tensor and every row of a row-strided one has
// at least one, however short (300 tensors of 6 elements: 31 us a pass, with one
// workgroup per 2048 elements 342; 5000 rows of 8: 10 and 118).
template <int KIND>
static hipError_t norm_partials(const GradSpan* g, int64_t n, double* partials, int max_partials, int* groups, hipStream_t s) {
  const int64_t elements = elements_of(g, n), chunk = norm_chunk(elements);
  int64_t chunks = 0;
  for (int64_t i = 0; i < n && chunks < max_partials; ++i) {
    const int64_t per = chunks_of_row(g[i].cols, g[i].in_dtype, chunk);
    chunks = g[i].rows >= max_partials || per >= max_partials ? max_partials : chunks + g[i].rows * per;
  }
  const int count = (int)std::max<int64_t>(1, std::min<int64_t>(max_partials, chunks));
  int first = 1;
  for (int dt = 0; dt < 3; ++dt) {
    const hipError_t e = for_tables(g, n, dt, -1, -1, chunk, count, [&](const auto& S, int) {
      const int f = first;
      first = 0;
      switch (dt) {
        case DT_BF16: return norm_go<bf16, KIND>(S, partials, count, f, s);
        case DT_F16: return norm_go<f16, KIND>(S, partials, count, f, s);
        default: return norm_go<float, KIND>(S, partials, count, f, s);
      }
    });
    if (e != hipSuccess) return e;
  }
  *groups = first ? 0 : count;
  return hipSuccess;
}
template <int KIND>
static hipError_t norm_kind(const GradSpan* g, int64_t n, double* partials, int max_partials, float* total, hipStream_t s) {
  int groups = 0;
  const hipError_t e = norm_partials<KIND>(g, n, partials, max_partials, &groups, s);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((k_grad_total<KIND>), dim3(1), dim3(256), 0, s, partials, groups, total);
  return hipGetLastError();
}

hipError_t launch_grad_norm(const GradSpan* g, int64_t n, int kind, double* partials, int max_partials, float* total, hipStream_t s) {
  switch (kind) {
    case 2: return norm_kind<2>(g, n, partials, max_partials, total, s);
    case 1: return norm_kind<1>(g, n, partials, max_partials, total, s);
    default: return norm_kind<0>(g, n, partials, max_partials, total, s);
  }
}

template <class T, class O, int KIND, int ROWS>
static hipError_t clip_go(const SpanTable<ROWS>& S, int groups, const ClipParams& P, hipStream_t s) {
  hipLaunchKernelGGL((k_clip<T, O, KIND, ROWS>), dim3(groups), dim3(256), 0, s, S, P);
  return hipGetLastError();
}
template <class T, int KIND, int ROWS>
static hipError_t clip_out(const SpanTable<ROWS>& S, int groups, int out, const ClipParams& P, hipStream_t s) {
  switch (out) {
    case DT_BF16: return clip_go<T, bf16, KIND>(S, groups, P, s);
    case DT_F16: return clip_go<T, f16, KIND>(S, groups, P, s);
    default: return clip_go<T, float, KIND>(S, groups, P, s);
  }
}
template <int KIND>
static hipError_t clip_kind(const GradSpan* g, int64_t n, ClipParams P, hipStream_t s) {
  for (int in = 0; in < 3; ++in)
    for (int out = 0; out < 3; ++out)
      for (int place = 0; place < 2; ++place) {
        if (place && in != out) continue;
        P.in_place = place;
        const hipError_t e = for_tables(g, n, in, out, place, kClipChunk, kClipGroups, [&](const auto& S, int groups) {
          switch (in) {
            case DT_BF16: return clip_out<bf16, KIND>(S, groups, out, P, s);
            case DT_F16: return clip_out<f16, KIND>(S, groups, out, P, s);
            default: return clip_out<float, KIND>(S, groups, out, P, s);
          }
        });
        if (e != hipSuccess) return e;
      }
  return hipSuccess;
}

hipError_t launch_clip_grads(const GradSpan* g, int64_t n, const float* total, float max_norm, hipStream_t s) {
  return clip_kind<-1>(g, n, ClipParams{nullptr, 0, const_cast<float*>(total), max_norm, 0}, s);
}

// Norm, then clipping.  In sets below kFuseTotal elements the clipping kernels
// add up the partials (40 tensors, 12 M elements: 27.4 -> 25.7 us a pass; 201
// tensors, 60 M elements: 167 -> 182 us of kernels, so not there).
constexpr int64_t kFuseTotal = 16ll << 20;
template <int KIND>
static hipError_t clip_norm_kind(const GradSpan* g, int64_t n, double* partials, int max_partials, float* total, float max_norm, hipStream_t s) {
  const int64_t elements = elements_of(g, n);
  if (elements == 0 || elements >= kFuseTotal) {
    const hipError_t e = norm_kind<KIND>(g, n, partials, max_partials, total, s);
    return e != hipSuccess ? e : launch_clip_grads(g, n, total, max_norm, s);
  }
  int groups = 0;
  const hipError_t e = norm_partials<KIND>(g, n, partials, max_partials, &groups, s);
  return e != hipSuccess ? e : clip_kind<KIND>(g, n, ClipParams{partials, groups, total, max_norm, 0}, s);
}
hipError_t launch_clip_grad_norm(const GradSpan* g, int64_t n, int kind, double* partials, int max_partials, float* total, float max_norm, hipStream_t s) {
  switch (kind) {
    case 2: return clip_norm_kind<2>(g, n, partials, max_partials, total, max_norm, s);
    case 1: return clip_norm_kind<1>(g, n, partials, max_partials, total, max_norm, s);
    default: return clip_norm_kind<0>(g, n, partials, max_partials, total, max_norm, s);
  }
}

}  // namespace orda
