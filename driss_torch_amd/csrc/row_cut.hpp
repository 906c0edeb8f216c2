// How a row of a matrix on an aligned base falls to 16-byte vectors of kV elements, and which rows the kernels that cut them so can take.  Plain
// arithmetic, also for the host.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dt {

// A row of at least kV elements: `head` elements up to the first vector boundary (EDGES: rows that are no whole number of vectors), whole aligned vectors,
// and `tail` elements.  A shorter row may begin and end inside one vector; nothing here holds then (nvec is -1).
template <int kV, bool EDGES>
struct RowCut {
  int64_t from;    // the vector that the row's first element lies in
  int64_t vec0;    // first whole vector
  int nvec;        // whole vectors
  int skip, tail;  // elements of vector `from` that are the row's before; elements behind the last whole vector
  __host__ __device__ RowCut(int64_t row, int64_t cols) {
    const uint64_t first = (uint64_t)row * (uint64_t)cols;
    from = (int64_t)(first / kV);
    skip = EDGES ? (int)(first % kV) : 0;
    vec0 = from + (skip != 0);
    const int64_t rest = cols - (skip ? kV - skip : 0);
    nvec = (int)((uint64_t)rest / kV);
    tail = EDGES ? (int)((uint64_t)rest % kV) : 0;
  }
  __host__ __device__ int edge(int lane_of_row) const {  // the lane's single element, counted from vector `from`; -1: none
    const int head = skip ? kV - skip : 0;
    const int at_tail = (int)(vec0 - from + nvec - 1) * kV + lane_of_row;
    return lane_of_row < head ? skip + lane_of_row : lane_of_row >= kV && lane_of_row < kV + tail ? at_tail : -1;
  }
};

// Rows that int8_rows_kernel keeps in registers: cut into vectors of an aligned base, up to sixteen of them in each of 1024 threads.
inline bool int8_rows_in_registers(bool base_ok, int64_t cols, int kV) { return base_ok && cols >= kV && cols <= (int64_t)16 * 1024 * kV; }

}  // namespace dt
