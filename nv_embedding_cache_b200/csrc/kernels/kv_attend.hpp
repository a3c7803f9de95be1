// Parameters and launchers of the attention over the paged cache (kernels: kv_attend.cuh, kv_join.cu).
#pragma once

#include "kv_common.cuh"

namespace nve_b200 {

struct KvAttendParams {
  KvView cache;
  KvTable table;
  const uint8_t* q;
  int64_t q_seq, q_head;             // bytes
  uint8_t* out;
  int64_t out_seq, out_head;         // bytes
  float* lse;                        // may be nullptr
  bool q_bf16;                       // type of q and out
  int32_t q_heads;
  int32_t group;                     // query heads of one key head
  int32_t chunk;                     // query heads one unit takes (group split over `chunks` units)
  int32_t chunks;
  int32_t tile_rows;                 // kv_tile_rows of this width and type
  int32_t rows_per_unit;             // padded rows of a unit in the scratch: 8, 16, 32 or 64
  float scale_log2;                  // scale * log2(e)
  // scratch
  float* part_acc;                   // [ctas][2][rows_per_unit][width]
  float2* part_ml;                   // [ctas][2][rows_per_unit] (maximum, sum), base 2
  float* unit_lse;                   // [sequences * heads * chunks][rows_per_unit] base-2 lse of units one CTA did alone
  float* scores;                     // [tiles][chunk][tile_rows] base-2 scores, nullptr without weights
  int32_t ctas;                      // grid of the split kernel
};

// Most CTAs the split kernel can use at once, for this variant on the current device.
int kv_attend_resident(nve_data_type_t cache_dtype, int width, int rows_per_unit);
void launch_kv_attend(const KvAttendParams& p, nve_data_type_t cache_dtype, cudaStream_t stream);
void launch_kv_join(const KvAttendParams& p, int sms, cudaStream_t stream);

// one per stored type, in a translation unit of its own
template <typename ST>
struct KvAttendVariant {
  static int resident(int width, int rows_per_unit);
  static void launch(const KvAttendParams& p, cudaStream_t stream);
};

#ifdef __CUDACC__
// The walk over tiles in the order of kv_plan.hpp.
struct TileCursor {
  int32_t b, head, chunk, j;         // sequence, key head, chunk of its query heads, tile inside the unit
  int32_t length, tiles;             // of sequence b

  // Next tile; sequences without rows have none.
  __device__ __forceinline__ void advance(const KvTable& t, int32_t heads, int32_t chunks, int32_t tile_rows) {
    if (++j < tiles) return;
    j = 0;
    if (++chunk < chunks) return;
    chunk = 0;
    if (++head < heads) return;
    head = 0;
    do {
      if (++b >= t.sequences) return;
      length = kv_length(t, b, nullptr);
      tiles = tiles_of(length, tile_rows);
    } while (tiles == 0);
  }
};
#endif

}  // namespace nve_b200
