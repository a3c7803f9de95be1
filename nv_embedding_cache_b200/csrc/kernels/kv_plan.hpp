// Arithmetic the kernels of the paged cache and their host code share, plain C++ so that it can be checked without a
// GPU: division by an invariant, and the cut of the attention's tiles into runs.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define NVE_KV_FN __host__ __device__ __forceinline__
#else
#define NVE_KV_FN inline
#endif

namespace nve_b200 {

// n / d for 0 <= n < 2^31, 1 <= d < 2^31, by one multiply: magic = ceil(2^(31 + l) / d), l = ceil(log2 d), is below
// 2^32 and at most 2^(31 + l) / d + 1, and the error n / 2^(31 + l) that this 1 brings stays below 1 / d
// (Granlund and Montgomery 1994).
struct FastDiv {
  uint32_t d, magic, shift;
};
inline FastDiv make_fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  if (d <= 1) return f;
  uint32_t l = 0;
  while ((uint64_t{1} << l) < d) l++;
  f.shift = l - 1;
  f.magic = static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + d - 1) / d);
  return f;
}
NVE_KV_FN uint32_t fast_div(uint32_t n, const FastDiv& f) {
  return f.d <= 1 ? n : static_cast<uint32_t>((static_cast<uint64_t>(n) * f.magic) >> 32) >> f.shift;
}

// ---- tiles of the attention -----------------------------------------------------------------------
// Tiles (kv_tile_rows rows of one unit = a key head and a chunk of its query heads) are numbered sequence by sequence,
// inside a sequence unit by unit, inside a unit along the length.  n CTAs take runs of them in order, the first `more`
// of `each` + 1 tiles, the others of `each`: the work is the same for all, whatever the lengths are.  n <= total, so no
// run is empty.
// Rows of a tile: 16 KB of keys and 16 KB of values for rows of 128 and 256 bytes (the width is padded to 64, 128 or
// 256 values); 128 rows at most, so that short sequences still make several tiles.
constexpr int kKvMaxTile = 128;
NVE_KV_FN constexpr int kv_padded_width(int width) { return width <= 64 ? 64 : (width <= 128 ? 128 : 256); }
NVE_KV_FN constexpr int kv_tile_rows(int width, int value_bytes) {
  return kv_padded_width(width) * value_bytes <= 128 ? kKvMaxTile : 64;
}

NVE_KV_FN int32_t tiles_of(int32_t length, int32_t tile_rows) {   // a power of two
  return static_cast<int32_t>((static_cast<uint32_t>(length) + tile_rows - 1) / static_cast<uint32_t>(tile_rows));
}

struct TileSplit {
  int32_t each, more;
};
NVE_KV_FN TileSplit tile_split(int32_t total, int32_t n) { return {total / n, total % n}; }
NVE_KV_FN int32_t run_first(TileSplit s, int32_t c) { return c * s.each + (c < s.more ? c : s.more); }
// The CTA whose run holds tile t.
NVE_KV_FN int32_t cta_of_tile(TileSplit s, int32_t t) {
  const int32_t longer = s.more * (s.each + 1);              // tiles of the longer runs
  return t < longer ? t / (s.each + 1) : s.more + (t - longer) / s.each;
}
// A CTA leaves at most two unfinished units: the one its run begins in and the one it ends in.  Slot of the unit that
// begins at tile `unit_first` in the scratch of a CTA whose run begins at tile `first`.
NVE_KV_FN int32_t part_slot(int32_t first, int32_t unit_first) { return first >= unit_first ? 0 : 1; }

}  // namespace nve_b200
