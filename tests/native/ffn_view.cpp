// The views of came_amd/csrc/came8_view.h for the host (tests/test_ffn_view.py).
#include "../../came_amd/csrc/came8_view.h"

extern "C" {
int64_t view_bytes(int rows, int64_t extent, int64_t K, int64_t ld, int64_t elem) {
  return came8::view_bytes(rows != 0, extent, K, ld, elem);
}
int32_t buffer_bytes(int64_t left) { return came8::buffer_bytes(left); }
}
