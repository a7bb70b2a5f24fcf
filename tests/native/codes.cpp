// The codes of came_amd/csrc/came8_codes.h for the host (tests/test_nearest_codes.py).
#include "../../came_amd/csrc/came8_codes.h"

extern "C" void nearest_codes(const float* x, const float* c, const double* p, const double* a, float* out, long n) {
  for (long i = 0; i < n; ++i) out[i] = came8::nearest_code(x[i], c[i], p[i], a[i]);
}
