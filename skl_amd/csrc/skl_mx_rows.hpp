// skl_mx_rows.hpp - which values of C a lane writes, and reads first, when a wave's part of a tile of skl_gemm_mxf4.hip goes out as rows. Plain
// address arithmetic, so that a program on the host can walk through it too (tests/c/mx_rows_check.cpp).
#pragma once

#include <cstddef>

// A part has 32 TN columns; 8 TN lanes hold a row of it, four values each, and a pass takes the rows that 64 lanes hold. Row r + at_row is the lane's in
// the pass that begins at row r.
template <int TN>
struct MxRows {
  static constexpr int kLanes = 8 * TN, kRowsAt = 64 / kLanes, kPasses = 32 / kRowsAt;  // lanes that hold a row, rows of a pass, passes per row of blocks
  unsigned at_row, at_col;
  float *part, *first;  // the lane's column in the part's row 0 and in its row at_row
  size_t rsc;

  // c: the part's first value. Its row 0 exists; any other may not.
  constexpr MxRows(float *c, size_t rsc_, size_t csc, unsigned lane)
      : at_row(lane / kLanes), at_col(lane % kLanes * 4u), part(c + (size_t)at_col * csc), first(part + (size_t)at_row * rsc_), rsc(rsc_) {}

  constexpr bool exists(unsigned r, unsigned rows) const { return r + at_row < rows; }
  constexpr float *row(unsigned r) const { return first + (size_t)r * rsc; }  // to be used where it exists
  // What is loaded without a branch: where the row does not exist, the part's row 0 (not `first`, which may be behind C itself).
  constexpr const float *readable(unsigned r, unsigned rows) const { return exists(r, rows) ? row(r) : part; }
};
