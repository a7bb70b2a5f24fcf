// Workgroups of the norm's launches, in plain C++ (tests/native/rms_grid.cpp compiles it alone).  A launch's work items stay below
// 2^32 in each dimension; what has more rows, or columns to join, takes them in turns.
#pragma once

#include <cstdint>

namespace came8 {

constexpr int64_t kRmsMaxDim = int64_t(1) << 30;
constexpr int64_t kRmsMaxGroups = int64_t(1) << 20;  // of up to 1024 threads
constexpr int kRmsJoinColumns = 32;                  // of a workgroup of the join, at a time

// `per` rows a workgroup
constexpr int64_t rms_row_groups(int64_t rows, int64_t per) {
  const int64_t n = (rows + per - 1) / per;
  return n < kRmsMaxGroups ? n : kRmsMaxGroups;
}
// 1024 chunks of `vec` columns a workgroup
constexpr int64_t rms_column_groups(int64_t dim, int64_t vec) { return (dim + 1024 * vec - 1) / (1024 * vec); }
constexpr int64_t rms_join_groups(int64_t dim) { return rms_row_groups(dim, kRmsJoinColumns); }

}  // namespace came8
