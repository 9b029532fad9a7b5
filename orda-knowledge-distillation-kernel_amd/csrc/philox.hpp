// philox.hpp -- the random bits of dropout: Philox4x32 with 10 rounds (Salmon,
// Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011),
// a bijection of a 128-bit counter under a 64-bit key, so that any element's
// bits follow from its index and nothing is stored for the backward pass.
//
// Key: the seed.  Counter: (element index / 8, site), 64 bits each.  An
// element takes 16 of the 128 bits; it is dropped where they are below
// threshold = p in steps of 2^-16.  (32 bits an element would be two calls for 8
// elements: 40 quarter-rate multiplications, 640 cycles of a wave for 512
// elements, more than the 512 elements' bytes take in bf16.  16 bits make it
// 320.  In rows of odd lengths a piece of 8 starts inside a block, as 7 of 8 rows do
// there, and takes two: 640 again.  1999 rows of 1111 in fp16 take a norm 10.3 us
// forward and 15.1 backward, of 1112 8.1 and 12.1.)
#pragma once
#include "orda_core.hpp"

namespace orda {

struct DropParams {
  uint64_t seed;
  const int64_t* seed_ptr;  // not null: the seed is read there
  uint64_t site;
  uint32_t threshold;  // 0: nothing is dropped; 65536: everything
  float factor;        // 65536 / (65536 - threshold)
};

__device__ __forceinline__ uint64_t seed_of(const DropParams& d) {
  return d.seed_ptr ? (uint64_t)*d.seed_ptr : d.seed;
}

// Bit e: element 8 block + e is kept.
__device__ __forceinline__ uint32_t keep_block(uint64_t block, uint64_t seed, uint64_t site, uint32_t threshold) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)site, c3 = (uint32_t)(site >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m |= (w[i] & 0xffffu) >= threshold ? 1u << (2 * i) : 0u;
    m |= (w[i] >> 16) >= threshold ? 2u << (2 * i) : 0u;
  }
  return m;
}

// Bit e: element `index` + e is kept, e < 8.  An index inside a block of 8 (rows
// of odd lengths; never where EVEN) takes two.
template <bool EVEN>
__device__ __forceinline__ uint32_t keep8(int64_t index, uint64_t seed, uint64_t site, uint32_t threshold) {
  const uint64_t block = (uint64_t)index >> 3;
  const int skip = EVEN ? 0 : (int)(index & 7);
  uint32_t m = keep_block(block, seed, site, threshold);
  if (skip) m = (m | keep_block(block + 1, seed, site, threshold) << 8) >> skip;
  return m;
}

}  // namespace orda
