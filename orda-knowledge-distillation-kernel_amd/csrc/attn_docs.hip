// attn_docs.hip -- the document numbers of a packed batch as the attention
// kernels read them.
#include "step_launch.hpp"

namespace orda {

// One wave per 64 positions: the numbers, -1 behind the last position and for
// padding, and their range: (smallest, largest, whether there is padding, 0).
// A block of padding has a range that no other meets.
__global__ __launch_bounds__(64) void k_attn_docs(const int32_t* ids, int64_t ld, int64_t S, int64_t padded, int* docs, int4* ranges) {
  const int64_t at = (int64_t)blockIdx.x * 64 + threadIdx.x, row = blockIdx.y;
  int d = at < S ? ids[row * ld + at] : -1;
  if (d < 0) d = -1;
  docs[row * padded + at] = d;
  int lo = d < 0 ? 0x7fffffff : d, hi = d;
  for (int o = 32; o; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o));
    hi = max(hi, __shfl_xor(hi, o));
  }
  const bool pad = __any(d < 0);
  if (threadIdx.x == 0) ranges[row * (padded / 64) + blockIdx.x] = make_int4(lo, hi, pad, 0);
}

hipError_t launch_attn_docs(const int32_t* ids, int64_t ld, int64_t B, int64_t S, int64_t padded, int* docs, int4* ranges, hipStream_t s) {
  hipLaunchKernelGGL(k_attn_docs, dim3((unsigned)(padded / 64), (unsigned)B), dim3(64), 0, s, ids, ld, S, padded, docs, ranges);
  return hipGetLastError();
}

}  // namespace orda
