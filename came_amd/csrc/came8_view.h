// How far a product's tile sees of an operand in memory, in plain C++ (tests/native/ffn_view.cpp compiles it alone).
#pragma once

#include <cstdint>

namespace came8 {

// Bytes from a tile's first element to the matrix's last: after the last row, what lies between a row's end and the next row
// is not the matrix's (a slice of columns may end with its storage).  `extent`: the rows (or the columns, where those lie with
// the summed index from one to the next) from the tile's first on; ld: bytes from a row (or k) to the next.
constexpr int64_t view_bytes(bool rows, int64_t extent, int64_t K, int64_t ld, int64_t elem) {
  return rows ? (extent - 1) * ld + K * elem : (K - 1) * ld + extent * elem;
}

// What the hardware checks offsets against.  It checks words, and rows start on words (k_ffn_pack), so the last word may count
// whole: it holds a byte of the matrix.
constexpr int32_t buffer_bytes(int64_t left) {
  return left <= 0 ? 0 : left > 0x7ffffffcll ? 0x7ffffffc : int32_t((left + 3) & ~int64_t(3));
}

}  // namespace came8
