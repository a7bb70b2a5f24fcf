// The shares of came_amd/csrc/came8_shares.h for the host (tests/test_embedding_shares.py).
#include "../../came_amd/csrc/came8_shares.h"

// The pairs (s, last) of one token, at most `room` of them; how many there are
extern "C" int64_t share_ends(int64_t start, int64_t all, int64_t share, int64_t* pairs, int64_t room) {
  int64_t n = 0;
  came8::share_ends(int32_t(start), int32_t(all), int32_t(share), [&](int64_t s, int32_t last) {
    if (n < room) {
      pairs[2 * n] = s;
      pairs[2 * n + 1] = last;
    }
    ++n;
  });
  return n;
}
