// What an experts' product reads out of its lists: which rows of A and C its
// places have, and which tile a workgroup takes.  The lists live on the device
// and hold whatever their writer left there: nothing here overflows or leads
// out of the buffers, for any of an int's values.
#pragma once

#include <stdint.h>

namespace dw {

// Rows of A that a list names: place p of C's rows reads row list[p] / each
// (row 0 where the list says what is no place), or row p without a list.
struct RowList {
  const int32_t* list;
  uint32_t places, each;
  __host__ __device__ __forceinline__ uint32_t row(int p) const {
    if (!list) return (uint32_t)p;
    const uint32_t v = (uint32_t)list[p];
    return v < places ? v / each : 0u;
  }
};

// C's row that a list names, below 0 for none.
__host__ __device__ __forceinline__ int row_named(int32_t entry, int rows) { return entry < rows ? entry : -1; }

// The tile that workgroup `id` takes of `rows` x `columns` of them, row after row.
// Neighbouring workgroups go to the 8 XCDs in turn: each takes a run of tiles.  Lists
// that overlap may make more tiles than 31 bits count: what is left of their number
// are tiles of the first rows, or none.
__host__ __device__ __forceinline__ bool tile_number(int id, int rows, int columns, int* tile) {
  const int total = (int)((uint32_t)rows * (uint32_t)columns), per = total / 8, rest = total % 8, xcd = id % 8, in = id / 8;
  if (in >= per + (xcd < rest)) return false;
  *tile = xcd * per + (xcd < rest ? xcd : rest) + in;
  return true;
}

}  // namespace dw
