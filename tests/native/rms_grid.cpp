// The launches of came_amd/csrc/came8_rms_grid.h for the host (tests/test_rms_grid.py).
#include "../../came_amd/csrc/came8_rms_grid.h"

extern "C" {
int64_t max_dim() { return came8::kRmsMaxDim; }
int64_t row_groups(int64_t rows, int64_t per) { return came8::rms_row_groups(rows, per); }
int64_t column_groups(int64_t dim, int64_t vec) { return came8::rms_column_groups(dim, vec); }
int64_t join_groups(int64_t dim) { return came8::rms_join_groups(dim); }
}
