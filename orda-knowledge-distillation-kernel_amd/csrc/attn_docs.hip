// attn_docs.hip -- the document numbers of a packed batch as the attention
// kernels read them, and the sums of dk and dv over parts of a key's heads.
#include "epilogue.hpp"
#include "step_launch.hpp"

namespace orda {

// One wave per 64 positions: the numbers, -1 behind the last position and for
// padding, and the ranges of either half: (smallest, largest, whether there is
// padding, 0).  A block of padding has a range that no other meets.  What lies
// behind the last position counts for none of it: nothing there is loaded or kept.
__global__ __launch_bounds__(64) void k_attn_docs(const int32_t* ids, int64_t ld, int64_t S, int64_t padded, int* docs, int4* ranges) {
  const int64_t at = (int64_t)blockIdx.x * 64 + threadIdx.x, row = blockIdx.y;
  int d = at < S ? ids[row * ld + at] : -1;
  if (d < 0) d = -1;
  docs[row * padded + at] = d;
  int lo = d < 0 ? 0x7fffffff : d, hi = d;
  for (int o = 16; o; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o));
    hi = max(hi, __shfl_xor(hi, o));
  }
  const int half = threadIdx.x / 32, pad = (uint32_t)(__ballot(at < S && d < 0) >> (32 * half)) != 0;
  if (threadIdx.x % 32 == 0) ranges[row * (padded / 32) + 2 * blockIdx.x + half] = make_int4(lo, hi, pad, 0);
}

hipError_t launch_attn_docs(const int32_t* ids, int64_t ld, int64_t B, int64_t S, int64_t padded, int* docs, int4* ranges, hipStream_t s) {
  hipLaunchKernelGGL(k_attn_docs, dim3((unsigned)(padded / 64), (unsigned)B), dim3(64), 0, s, ids, ld, S, padded, docs, ranges);
  return hipGetLastError();
}

// dk (blockIdx.y = 0) and dv of 8 elements a thread: parts in their order.
template <class T>
__global__ __launch_bounds__(256) void k_attn_join(const float* partial, int64_t size, int parts, T* dk, T* dv, float scale) {
  const int64_t at = 8 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  T* out = blockIdx.y ? dv : dk;
  if (at >= size || !out) return;
  const float* p = partial + blockIdx.y * parts * size + at;
  float sum[8] = {};
  for (int i = 0; i < parts; ++i, p += size) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += v[e];
  }
  const float mul = blockIdx.y ? 1.0f : scale;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] *= mul;
  st_row<T, 8>(out + at, sum, 8);
}

hipError_t launch_attn_join(const AttnParams& P, int dtype, hipStream_t s) {
  const int64_t size = (int64_t)P.B * P.S * P.KV * P.D;
  const dim3 grid((unsigned)((size / 8 + 255) / 256), 2);
  if (dtype == DT_BF16)
    hipLaunchKernelGGL(k_attn_join<bf16>, grid, dim3(256), 0, s, P.partial, size, P.parts, static_cast<bf16*>(P.dk), static_cast<bf16*>(P.dv), P.scale);
  else
    hipLaunchKernelGGL(k_attn_join<f16>, grid, dim3(256), 0, s, P.partial, size, P.parts, static_cast<f16*>(P.dk), static_cast<f16*>(P.dv), P.scale);
  return hipGetLastError();
}

}  // namespace orda
