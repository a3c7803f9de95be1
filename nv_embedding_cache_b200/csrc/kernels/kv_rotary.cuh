// Rotation of head rows, and the same with the paged cache as destination (see kv_rotary.cu).
#pragma once

#include "kv_common.cuh"

namespace nve_b200 {

struct RowGroup {
  const uint8_t* in;
  uint8_t* out;                     // nullptr: the group's rows go to the cache
  int64_t in_token, in_head, out_token, out_head;
  int32_t heads;
};

struct RotaryParams {
  RowGroup g[3];                    // queries, keys, values; heads == 0: none
  int32_t rows;                     // heads of all groups
  const int32_t* positions;
  int64_t axis_stride, token_stride;
  int32_t axes;
  const float* inv_freq;
  const int32_t* pair_axis;
  int32_t pairs;
  int32_t width;
  float sign;                       // -1: backward
  int32_t* status;
  int32_t tokens;
  // filled by the launcher
  int32_t items;                    // work items of one row
  int32_t turned_items;             // the first of them hold pairs, the others are copied
  int32_t tokens_per_block;
  int32_t lanes;                    // threads that share the items of a row
  int32_t row_lanes;                // threads that share the rows of a token, for one item
  // append
  bool to_cache;
  bool zero_padding;                // queries of padding tokens become zeros
  KvView cache;
  KvTable table;
  const int32_t* offsets;           // nullptr: per_sequence tokens each
  int32_t per_sequence;
  int32_t* new_lengths;
};

void launch_rotary(RotaryParams p, nve_data_type_t dtype, nve_data_type_t cache_dtype, bool interleaved, int sms,
                   cudaStream_t stream);

}  // namespace nve_b200
