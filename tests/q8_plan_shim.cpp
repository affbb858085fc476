// q8_plan.h as a library of its own, for the tests of its rules on the CPU.
#include "../nemo_amd/csrc/q8_plan.h"

extern "C" void plan(int32_t M, int32_t n_seg, int32_t ragged, int32_t n_cols, int32_t K, int32_t out_bytes, int32_t n_cu, int64_t *to) {
  const Q8Plan p = q8_plan({M, n_seg, ragged, n_cols, K, out_bytes, n_cu});
  const int64_t v[] = {p.refusal, p.kernel, p.grid_x, p.grid_y, (int64_t)p.tiles, (int64_t)p.cuts, p.across, p.split, p.wc, p.rt};
  for (int64_t x : v) *to++ = x;
}
extern "C" int32_t max_cols() { return Q8_MAX_COLS; }
extern "C" int32_t rows_fit(int64_t n) { return q8_rows_fit(n); }
