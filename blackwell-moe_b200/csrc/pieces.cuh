// A row as pieces of 16 bytes; of 8, 4 or 2 where its length or a pointer allows no more.
#pragma once

#include <initializer_list>

#include "common.cuh"

namespace bwmoe {

template <int BYTES> struct Piece;
template <> struct Piece<16> { using type = uint4; };
template <> struct Piece<8> { using type = uint2; };
template <> struct Piece<4> { using type = uint32_t; };
template <> struct Piece<2> { using type = uint16_t; };

template <class P> __device__ __forceinline__ P zero_piece() {
  P z;
  memset(&z, 0, sizeof(P));
  return z;
}

// Whether no slot owns row r.  E > 0: the plan is this library's, `offsets` are its segments [E + 1], and the rows without a slot
// are those behind the last (n_rows = offsets[E]).  E = 0: any plan, and `offsets` is a slot of each row, -1 where there is none.
__device__ __forceinline__ bool no_slot(const int32_t* __restrict__ offsets, int E, int n_rows, int r) {
  return E > 0 ? r >= n_rows : offsets[r] < 0;
}

// Bytes of the widest piece that divides the row and every pointer.
inline int piece_bytes(size_t row_bytes, std::initializer_list<const void*> ptrs) {
  uintptr_t bits = (uintptr_t)row_bytes;
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

}  // namespace bwmoe
