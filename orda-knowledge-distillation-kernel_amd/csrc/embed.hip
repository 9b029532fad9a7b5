// embed.hip -- the token embedding: rows of the weight, scaled, and the
// weight's gradient by sorted tokens.
//
// Forward: y[n] = scale W[t_n], one piece of 8 columns a thread, bound by
// memory.  A token outside [0, V) gives a row of zeros and no gradient.
//
// Backward: dW[v] = scale sum of dy[n] over t_n = v, and zeros in all other
// rows (most of the bytes with a large vocabulary).  Four launches:
//   sort   segments of 4096 tokens, each by one workgroup in LDS (radix, 8 bits
//          a pass, stable); the other workgroups fill the first rows of dW with
//          zeros meanwhile
//   merge  up to 16 sorted segments a round: an element's place is the sum of
//          its places in the others, found by 16 searches side by side (more
//          than 4096 tokens); beside the first round, the next rows of zeros
//   sum    a wave takes 512 columns of `chunk` sorted entries and adds up their
//          rows of dy in fp32; a run of one token that lies in the chunk goes
//          out rounded, one that reaches past it as an fp32 partial sum; other
//          waves fill the remaining rows that no token names
//   join   the partial sums of such runs, in order
// Equal tokens stay in their order throughout, so the sums do not depend on the
// run, and a token that fills the batch is added up by as many waves as any
// other.
//
// Memory bounds both passes.  16384 tokens over 128256 rows of 4096 in bf16: forward
// 268 MB in 53 us; backward 1.3 GB in 241 us (sort 23 and merge 21, with 128 MB of
// zeros each, sums and the other 750 MB of zeros 181, join 16), where a fill of all
// rows first and the sums behind it took 277.  Small batches are the sort's: 1999
// tokens in one workgroup take 10 us over a gradient of 0.8 MB, 14 with 78 MB of zeros
// beside it (11 at a fill's rate).
#include <algorithm>

#include "pieces.hpp"
#include "step_launch.hpp"

namespace orda {

__device__ __forceinline__ int64_t token_at(const void* ids, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int32_t*>(ids)[i];
}

// ------------------------------------------------------------- forward
// N pieces a thread, whose loads, each behind its token's, are in flight together
// (16384 rows of 4096 in bf16: 53 us, one piece a thread 56).
template <class W, class T, int N, bool EVEN>
__global__ __launch_bounds__(256) void k_embed(EmbedParams P, int64_t per_row, int64_t pieces) {
  for (int64_t i0 = (int64_t)blockIdx.x * (256 * N) + threadIdx.x; i0 < pieces; i0 += (int64_t)gridDim.x * (256 * N)) {
    int64_t row[N], t[N];
    Piece<EVEN> p[N];
    Raw8<W> w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t i = lmin(i0 + k * 256, pieces - 1);  // (the last piece again: the same values)
      row[k] = pieces <= 0xffffffffll ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row;
      p[k] = Piece<EVEN>(i - row[k] * per_row, P.hidden);
      t[k] = token_at(P.ids, P.wide, row[k]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (t[k] >= P.vocab) t[k] = -1;
      w[k].get(static_cast<const W*>(P.weight) + (t[k] < 0 ? 0 : t[k]) * P.ldw, p[k]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = t[k] >= 0 ? w[k][e] * P.scale : 0.0f;
      put8(static_cast<T*>(P.y) + row[k] * P.hidden, p[k], v);
    }
  }
}

// ------------------------------------------------------------- sort
constexpr int kSegment = 4096;  // tokens of one workgroup
constexpr int kFill = 4096;     // 16-byte stores of one that fills
constexpr int64_t kBeside = 128ll << 20;  // bytes of zeros beside the sort, and beside the merge

// Zeros in the bytes [begin, end) of p (from the 16 that begin lies in on), 64 KB
// of a workgroup of N threads in a row.
template <int N>
__device__ __forceinline__ void fill_zeros(void* p, int64_t begin, int64_t end, int64_t group, int64_t groups) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4* out = static_cast<uint4*>(p) + begin / 16;
  const int64_t bytes = end - begin / 16 * 16, n = bytes / 16;
  for (int64_t b = group; b * kFill < n; b += groups)
#pragma unroll 4
    for (int i = 0; i < kFill / N; ++i) {
      const int64_t at = b * kFill + i * N + threadIdx.x;
      if (at < n) out[at] = zero;
    }
  const int tail = (int)(bytes % 16) / 2;  // (elements of 2 or 4 bytes)
  if (group == 0 && (int)threadIdx.x < tail) reinterpret_cast<uint16_t*>(out + n)[threadIdx.x] = 0;
}

// Keys: the token, V for one that has no gradient (it sorts behind all others).
// Entries past the last token have all bits set and stay behind them.
__global__ __launch_bounds__(1024) void k_embed_sort(EmbedGradParams P, int passes, int segments, uint32_t* tokens, uint32_t* places, int64_t fill_end) {
  if ((int)blockIdx.x >= segments) {
    fill_zeros<1024>(P.dw, 0, fill_end, blockIdx.x - segments, gridDim.x - segments);
    return;
  }
  __shared__ uint32_t key[2][kSegment];
  __shared__ uint16_t from[2][kSegment];
  __shared__ uint32_t hist[16][256];
  __shared__ uint32_t total[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t base = (int64_t)blockIdx.x * kSegment;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = w * 256 + i * 64 + lane;
    uint32_t k = 0xffffffffu;
    if (base + at < P.tokens) {
      const int64_t t = token_at(P.ids, P.wide, base + at);
      k = t >= 0 && t < P.vocab && t != P.padding ? (uint32_t)t : (uint32_t)P.vocab;
    }
    key[0][at] = k;
    from[0][at] = (uint16_t)at;
  }
  int cur = 0;
  for (int pass = 0; pass < passes; ++pass, cur ^= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(hist)[threadIdx.x + 1024 * i] = 0;
    __syncthreads();
    // a key's rank among the keys of its wave's 256 with the same digit: those
    // of earlier rows of 64 (counted in hist), and of lower lanes
    uint32_t k[4], rank[4];
    uint16_t f[4];
    volatile uint32_t* mine = hist[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = w * 256 + i * 64 + lane;
      k[i] = key[cur][at];
      f[i] = from[cur][at];
      const uint32_t d = (k[i] >> (8 * pass)) & 255u;
      uint64_t same = ~0ull;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const uint64_t m = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? m : ~m;
      }
      const uint32_t before = __popcll(same & ((1ull << lane) - 1)), old = mine[d];
      rank[i] = old + before;
      __builtin_amdgcn_wave_barrier();
      if (before == 0) mine[d] = old + (uint32_t)__popcll(same);
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // exclusive sums over digits, within a digit over waves: 4 waves a thread
    const int d = threadIdx.x >> 2, q = (threadIdx.x & 3) * 4;
    uint32_t c[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = hist[q + j][d];
      sum += c[j];
    }
    uint32_t run = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t up = __shfl_up(run, o);
      if (lane >= o) run += up;
    }
    if (lane == 63) total[w] = run;
    __syncthreads();
    run -= sum;
    for (int i = 0; i < w; ++i) run += total[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      hist[q + j][d] = run;
      run += c[j];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t to = hist[w][(k[i] >> (8 * pass)) & 255u] + rank[i];
      key[cur ^ 1][to] = k[i];
      from[cur ^ 1][to] = f[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = threadIdx.x + 1024 * i;
    if (base + at < P.tokens) {
      tokens[base + at] = key[cur][at];
      places[base + at] = (uint32_t)(base + from[cur][at]);
    }
  }
}

// Groups of 16 sorted segments of `len` (a power of two) entries to one each.  A
// wave's entries lie in one segment; the 16 searches of a lane have their loads in
// flight together, step by step, none under a condition (16384 tokens and 128 MB of
// zeros beside them: 21 us, what the zeros take; with conditional loads and
// 64-bit places 30).
__global__ __launch_bounds__(64) void k_embed_merge(const uint32_t* tokens, const uint32_t* places, uint32_t* tokens_out, uint32_t* places_out, int64_t n, int64_t len,
                                                    int groups, void* dw, int64_t fill_begin, int64_t fill_end) {
  if ((int)blockIdx.x >= groups) {
    fill_zeros<64>(dw, fill_begin, fill_end, blockIdx.x - groups, gridDim.x - groups);
    return;
  }
  const int64_t first = (int64_t)blockIdx.x * 64, group = first / (16 * len) * (16 * len), e = lmin(first + threadIdx.x, n - 1);
  const int own = (int)((first - group) / len);
  const uint32_t t = tokens[e];
  uint32_t pos[16];
#pragma unroll
  for (int b = 0; b < 16; ++b) pos[b] = 0;
  for (uint32_t s = (uint32_t)len; s > 0; s >>= 1) {
    uint32_t v[16];
    auto size = [&](int b) { return (uint32_t)std::max<int64_t>(0, lmin(len, n - group - b * len)); };
    // (four segments at a time, as long as there are any; of an empty one the group's
    // first entry, unused)
#pragma unroll
    for (int q = 0; q < 16; q += 4)
      if (size(q))
#pragma unroll
        for (int b = q; b < q + 4; ++b) v[b] = tokens[group + (size(b) ? b * len : 0) + (max(min(pos[b] + s, size(b)), 1u) - 1)];
#pragma unroll
    for (int q = 0; q < 16; q += 4)
      if (size(q))
#pragma unroll
        for (int b = q; b < q + 4; ++b)  // (equal ones of earlier segments come first)
          if (pos[b] + s <= size(b) && v[b] < t + (b < own)) pos[b] += s;
  }
  int64_t to = e - own * len;
#pragma unroll
  for (int b = 0; b < 16; ++b) to += b == own ? 0 : pos[b];
  if (first + threadIdx.x < n) {
    tokens_out[to] = t;
    places_out[to] = places[e];
  }
}

// ------------------------------------------------------------- sums
struct EmbedSums {
  const uint32_t* tokens;
  const uint32_t* places;
  float* part;  // [chunks][2][hidden]: of a run that began before the chunk, and of one that goes on behind it
  int chunk;
  int slabs;    // of 512 columns
  int64_t chunks;
  int groups;      // workgroups that add up
  int64_t filled;  // rows of dW that are zero already
};

// 64 rows of dW: zeros in those that no token names, every fourth by one wave.
template <class W, bool EVEN>
__device__ __forceinline__ void fill_unnamed(const EmbedGradParams& P, const EmbedSums& S, int64_t first) {
  const int lane = threadIdx.x & 63;
  const int64_t row = first + lane, per_row = pieces_of(P.hidden);
  int64_t lo = 0, hi = P.tokens;  // the first entry that is not below `row` lies in [lo, hi]
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if ((int64_t)S.tokens[mid] < row) lo = mid + 1;
    else hi = mid;
  }
  const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const uint64_t unnamed = __ballot(row < P.vocab && (lo == P.tokens || (int64_t)S.tokens[lo] != row));
  for (uint64_t to = unnamed & (0x1111111111111111ull << wave_id()); to; to &= to - 1) {
    W* out = static_cast<W*>(P.dw) + (first + __builtin_ctzll(to)) * P.hidden;
    for (int64_t i = lane; i < per_row; i += 64) put8(out, Piece<EVEN>(i, P.hidden), zero);
  }
}

template <class W, class T, bool EVEN>
__global__ __launch_bounds__(256) void k_embed_sum(EmbedGradParams P, EmbedSums S) {
  constexpr int kAhead = 8;  // rows in flight
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x >= S.groups) {
    for (int64_t first = S.filled + (int64_t)(blockIdx.x - S.groups) * 64; first < P.vocab; first += (int64_t)(gridDim.x - S.groups) * 64)
      fill_unnamed<W, EVEN>(P, S, first);
    return;
  }
  const int64_t units = S.chunks * S.slabs;
  for (int64_t u = (int64_t)blockIdx.x * 4 + wave_id(); u < units; u += (int64_t)S.groups * 4) {
    const int64_t chunk = u / S.slabs, first = chunk * S.chunk;
    const int n = (int)lmin(S.chunk, P.tokens - first);
    const Piece<EVEN> at((u - chunk * S.slabs) * 64 + lane, P.hidden);
    uint32_t tok = (uint32_t)P.vocab, place = 0;
    if (lane < n) {
      tok = S.tokens[first + lane];
      place = S.places[first + lane];
    }
    const uint32_t before = first > 0 ? S.tokens[first - 1] : 0xffffffffu;
    const uint32_t after = first + n < P.tokens ? S.tokens[first + n] : 0xffffffffu;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    bool from_before = (uint32_t)__builtin_amdgcn_readlane((int)tok, 0) == before;
    for (int i0 = 0; i0 < n; i0 += kAhead) {
      Raw8<T> v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {  // (without a condition, so that none waits for another; behind the last entry its row again)
        const int64_t row = (uint32_t)__builtin_amdgcn_readlane((int)place, min(i0 + k, n - 1));
        v[k].get(static_cast<const T*>(P.dy) + row * P.ldg, at);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = i0 + k;
        const uint32_t t = (uint32_t)__builtin_amdgcn_readlane((int)tok, min(i, n - 1));
        if (i >= n || t >= (uint32_t)P.vocab) break;  // (those without a gradient are the last)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += v[k][e];
        const bool last = i + 1 == n;
        const uint32_t next = last ? after : (uint32_t)__builtin_amdgcn_readlane((int)tok, last ? i : i + 1);
        if (!last && next == t) continue;
        // the run's end in this chunk
        if (from_before || next == t) {
          put8(S.part + (2 * chunk + (from_before ? 0 : 1)) * P.hidden, at, acc);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] *= P.scale;
          put8(static_cast<W*>(P.dw) + (int64_t)t * P.hidden, at, acc);
        }
        from_before = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
      }
    }
  }
}

// A run that begins in chunk c and goes on: its sum in c and those of the
// chunks that it reaches, every eighth of them by one wave.
template <class W, bool EVEN>
__global__ __launch_bounds__(512) void k_embed_join(EmbedGradParams P, EmbedSums S) {
  __shared__ float join[8][8][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t units = S.chunks * S.slabs;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t chunk = u / S.slabs, first = chunk * S.chunk, end = first + S.chunk;
    if (end >= P.tokens) continue;
    const uint32_t t = S.tokens[end], last = S.tokens[end - 1], start = S.tokens[first], before = first > 0 ? S.tokens[first - 1] : 0xffffffffu;
    if (t >= (uint32_t)P.vocab || last != t) continue;
    if (start == t && before == t) continue;  // (it began before)
    // the chunks that begin with t
    int64_t more = 0;
    while (true) {
      const int64_t e = end + (more + lane) * S.chunk;
      const uint64_t same = __ballot(e < P.tokens && S.tokens[lmin(e, P.tokens - 1)] == t);
      if (~same) {
        more += __builtin_ctzll(~same);
        break;
      }
      more += 64;
    }
    const Piece<EVEN> at((u - chunk * S.slabs) * 64 + lane, P.hidden);
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (w == 0) {
      Raw8<float> v;
      v.get(S.part + (2 * chunk + 1) * P.hidden, at);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = v[e];
    }
#pragma unroll 4
    for (int64_t k = 1 + w; k <= more; k += 8) {
      Raw8<float> v;
      v.get(S.part + 2 * (chunk + k) * P.hidden, at);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += v[e];
    }
    __syncthreads();  // (the turn before has read join)
#pragma unroll
    for (int e = 0; e < 8; ++e) join[w][e][lane] = acc[e];
    __syncthreads();
    if (w) continue;
#pragma unroll
    for (int i = 1; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += join[i][e][lane];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= P.scale;
    put8(static_cast<W*>(P.dw) + (int64_t)t * P.hidden, at, acc);
  }
}

// ------------------------------------------------------------- launches
template <class W, class T>
static hipError_t embed_go(const EmbedParams& P, hipStream_t s) {
  const int64_t per_row = pieces_of(P.hidden), pieces = per_row * P.tokens;
  auto go = [&](auto each, auto even) {
    constexpr int N = decltype(each)::value;
    const unsigned groups = (unsigned)std::min<int64_t>((pieces + 256 * N - 1) / (256 * N), 1 << 23);
    hipLaunchKernelGGL((k_embed<W, T, N, decltype(even)::value>), dim3(groups), dim3(256), 0, s, P, per_row, pieces);
  };
  // (several pieces a thread where one each would be more workgroups than the card holds at a time)
  const bool many = pieces > 256 * 2048, even = P.hidden % 8 == 0;
  if (many) even ? go(std::integral_constant<int, 4>{}, std::true_type{}) : go(std::integral_constant<int, 4>{}, std::false_type{});
  else even ? go(std::integral_constant<int, 1>{}, std::true_type{}) : go(std::integral_constant<int, 1>{}, std::false_type{});
  return hipGetLastError();
}
template <class W>
static hipError_t embed_out(const EmbedParams& P, int out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case DT_BF16: return embed_go<W, bf16>(P, s);
    case DT_F16: return embed_go<W, f16>(P, s);
    default: return embed_go<W, float>(P, s);
  }
}
hipError_t launch_embed(const EmbedParams& P, int dtype, int out_dtype, hipStream_t s) {
  switch (dtype) {
    case DT_BF16: return embed_out<bf16>(P, out_dtype, s);
    case DT_F16: return embed_out<f16>(P, out_dtype, s);
    default: return embed_out<float>(P, out_dtype, s);
  }
}

// Sorted entries of a wave's chunk: 32, fewer where that would leave less than
// 16 waves to a CU.
static EmbedSums sums_of(int64_t tokens, int64_t hidden) {
  EmbedSums S{};
  S.slabs = (int)((hidden + 511) / 512);
  S.chunk = 32;
  while (S.chunk > 4 && (tokens + S.chunk - 1) / S.chunk * S.slabs < 4096) S.chunk /= 2;
  S.chunks = (tokens + S.chunk - 1) / S.chunk;
  return S;
}
static size_t up256(size_t n) { return (n + 255) / 256 * 256; }
static size_t list_bytes(int64_t tokens) { return up256((size_t)tokens * 4); }
size_t embed_grad_workspace(int64_t tokens, int64_t hidden) {
  const EmbedSums S = sums_of(tokens, hidden);
  return list_bytes(tokens) * (tokens > kSegment ? 4 : 2) + up256((size_t)S.chunks * 2 * hidden * 4);
}

template <class W, class T, bool EVEN>
static hipError_t sum_even(const EmbedGradParams& P, EmbedSums S, hipStream_t s) {
  const int64_t units = S.chunks * S.slabs;
  S.groups = (int)std::min<int64_t>((units + 3) / 4, 1 << 22);
  const int64_t fill = std::min<int64_t>((P.vocab - S.filled + 63) / 64, 1 << 20);
  hipLaunchKernelGGL((k_embed_sum<W, T, EVEN>), dim3((unsigned)(S.groups + fill)), dim3(256), 0, s, P, S);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || S.chunks == 1) return e;
  hipLaunchKernelGGL((k_embed_join<W, EVEN>), dim3((unsigned)std::min<int64_t>(units, 1 << 20)), dim3(512), 0, s, P, S);
  return hipGetLastError();
}
template <class W, class T>
static hipError_t sum_go(const EmbedGradParams& P, const EmbedSums& S, hipStream_t s) {
  return P.hidden % 8 == 0 ? sum_even<W, T, true>(P, S, s) : sum_even<W, T, false>(P, S, s);
}
template <class W>
static hipError_t sum_out(const EmbedGradParams& P, const EmbedSums& S, int out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case DT_BF16: return sum_go<W, bf16>(P, S, s);
    case DT_F16: return sum_go<W, f16>(P, S, s);
    default: return sum_go<W, float>(P, S, s);
  }
}

hipError_t launch_embed_grad(const EmbedGradParams& P, int dtype, int out_dtype, void* workspace, hipStream_t s) {
  EmbedSums S = sums_of(P.tokens, P.hidden);
  const size_t list = list_bytes(P.tokens);
  char* ws = static_cast<char*>(workspace);
  uint32_t* tokens[2];
  uint32_t* places[2];
  const int lists = P.tokens > kSegment ? 2 : 1;
  for (int i = 0; i < 2; ++i) {
    tokens[i] = reinterpret_cast<uint32_t*>(ws + (i % lists) * 2 * list);
    places[i] = reinterpret_cast<uint32_t*>(ws + (i % lists) * 2 * list + list);
  }
  S.part = reinterpret_cast<float*>(ws + lists * 2 * list);
  int passes = 1;
  while (passes < 4 && (P.vocab >> (8 * passes)) != 0) ++passes;
  const int segments = (int)((P.tokens + kSegment - 1) / kSegment);
  // As many rows as the card fills while it sorts, and while it merges.
  const int64_t row_bytes = P.hidden * (dtype == DT_F32 ? 4 : 2), beside = (kBeside + row_bytes - 1) / row_bytes;
  auto fill_groups = [&](int64_t rows) { return (rows * row_bytes + kFill * 16 - 1) / (kFill * 16); };
  S.filled = std::min(P.vocab, beside);
  hipLaunchKernelGGL(k_embed_sort, dim3((unsigned)(segments + fill_groups(S.filled))), dim3(1024), 0, s, P, passes, segments, tokens[0], places[0], S.filled * row_bytes);
  hipError_t e = hipGetLastError();
  int at = 0;
  for (int64_t len = kSegment; e == hipSuccess && len < P.tokens; len *= 16, at ^= 1) {
    const int64_t rows = len == kSegment ? std::min(P.vocab - S.filled, beside) : 0, begin = S.filled * row_bytes;
    const int groups = (int)((P.tokens + 63) / 64);
    hipLaunchKernelGGL(k_embed_merge, dim3((unsigned)(groups + fill_groups(rows))), dim3(64), 0, s, tokens[at], places[at], tokens[at ^ 1], places[at ^ 1], P.tokens,
                       len, groups, P.dw, begin, begin + rows * row_bytes);
    e = hipGetLastError();
    S.filled += rows;
  }
  if (e != hipSuccess) return e;
  S.tokens = tokens[at];
  S.places = places[at];
  switch (dtype) {
    case DT_BF16: return sum_out<bf16>(P, S, out_dtype, s);
    case DT_F16: return sum_out<f16>(P, S, out_dtype, s);
    default: return sum_out<float>(P, S, out_dtype, s);
  }
}

}  // namespace orda
