// The host arithmetic of the paged cache (csrc/kernels/kv_plan.hpp) for tests without a GPU.
#include "kernels/kv_plan.hpp"

using namespace nve_b200;

extern "C" {
uint32_t kp_div(uint32_t n, uint32_t d) { return fast_div(n, make_fast_div(d)); }
int32_t kp_tiles(int32_t length, int32_t rows) { return tiles_of(length, rows); }
int32_t kp_tile_rows(int32_t width, int32_t bytes) { return kv_tile_rows(width, bytes); }
void kp_range(int32_t total, int32_t n, int32_t c, int32_t* out) {
  const TileSplit s = tile_split(total, n);
  out[0] = run_first(s, c);
  out[1] = run_first(s, c + 1);
}
int32_t kp_cta(int32_t total, int32_t n, int32_t t) { return cta_of_tile(tile_split(total, n), t); }
int32_t kp_slot(int32_t first, int32_t unit_first) { return part_slot(first, unit_first); }
}
