// pieces.hpp -- rows in pieces of 8 consecutive elements, the unit of the row
// kernels (rownorm.hip, embed.hip).
//
// A row whose length is no multiple of 8 ends with a piece that is moved back, so
// that it holds the row's last 8 elements: the first `lo` of them belong to the
// piece before.  Loads and stores are whole vectors then, at any alignment (both
// pieces store the same values there), and only sums leave the first `lo` out.
// With a tail of single elements, loads that wait for one another, a norm of 1999
// rows of 1111 in fp16 took 13.8 us instead of 10.5.  Rows shorter than 8 are one
// piece of n elements.  EVEN: the row's length is a multiple of 8, so that a piece
// is a lane's own or nobody's; a norm's masks of single elements would not fit the
// scalar registers.
#pragma once
#include "epilogue.hpp"

namespace orda {

template <bool EVEN>
struct Piece {
  int64_t c;  // its first column
  int lo;     // its own elements are [lo, n); 8: it has none
  int n;      // 8, in rows shorter than that the row (uniform)
  __device__ __forceinline__ Piece() {}
  __device__ __forceinline__ Piece(int64_t index, int64_t cols) {
    const int64_t at = 8 * index;
    if (EVEN || cols >= 8) {
      n = 8;
      c = lmin(at, cols - 8);
      lo = (int)lmin(at - c, 8);
    } else {
      n = (int)cols;
      c = 0;
      lo = at < cols ? 0 : 8;
    }
  }
  __device__ __forceinline__ int count() const { return EVEN ? 8 : n; }
  __device__ __forceinline__ bool any() const { return lo < 8; }
  __device__ __forceinline__ bool own(int e) const { return EVEN ? lo == 0 : e >= lo && e < n; }
};

// Pieces a row has.
__host__ __device__ __forceinline__ int64_t pieces_of(int64_t cols) { return (cols + 7) / 8; }

// The 8 elements as they lie in memory: loaded early, unpacked later.
template <class T>
struct Raw8 : RawRow<T, 8> {
  // every lane loads (a piece without elements of its own reads its row's last)
  template <bool EVEN>
  __device__ __forceinline__ void get(const T* row, const Piece<EVEN>& p) { this->load(row + p.c, p.count()); }
};
template <class T, bool EVEN>
__device__ __forceinline__ void put8(T* row, const Piece<EVEN>& p, const float (&v)[8]) {
  if (p.any()) st_row<T, 8>(row + p.c, v, p.count());
}

}  // namespace orda
