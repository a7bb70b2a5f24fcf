// Which shares of a sorted list end within one token's positions, in plain C++ (tests/native/shares.cpp compiles it alone).
#pragma once

#include <cstdint>

namespace came8 {

// Calls f(s, last) for every share s of `share` successive positions that ends within a token's [start, start + all): `last` is
// the last share that has the token where it begins in s and goes on, else -1.  The list's length is below 2^31, and so are
// its places; the end of a share may lie behind it: a list of nearly 2^31 has shares of 2^20, and those ends take 64 bits.
template <typename F>
constexpr void share_ends(int32_t start, int32_t all, int32_t share, F&& f) {
  const int32_t end = start + all;
  for (int64_t s = start / share; all > 0 && (s + 1) * share <= end; ++s)
    f(s, start >= s * share && end > (s + 1) * share ? (end - 1) / share : -1);
}

}  // namespace came8
