// Shared by the kernels of the paged key/value cache: the cache view, page addressing with its bounds
// checks, the walk over (sequence, head, tile) units, and small load / convert helpers.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "kv_plan.hpp"
#include "nve_b200_kv.h"

namespace nve_b200 {

struct KvView {
  uint8_t* keys;
  uint8_t* values;
  int64_t k_page, k_slot, k_head;   // bytes
  int64_t v_page, v_slot, v_head;
  float* weights;                   // [num_pages][heads][page_size]
  const float* key_scale;
  const float* value_scale;
  int32_t* status;
  uint32_t num_pages;
  int32_t page_size;
  int32_t heads;
  int32_t width;
  FastDiv page_div;
};

struct KvTable {
  const int32_t* pages;
  int64_t stride;
  const int32_t* lengths;
  int32_t sequences;
  int32_t capacity;                 // rows a sequence may have
};

__device__ __forceinline__ void kv_flag(int32_t* status, int32_t bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// Length of sequence b, held inside [0, capacity].
__device__ __forceinline__ int32_t kv_length(const KvTable& t, int32_t b, int32_t* status) {
  const int32_t n = __ldg(t.lengths + b);
  if (n < 0 || n > t.capacity) {
    kv_flag(status, NVE_B200_KV_BAD_LENGTH);
    return n < 0 ? 0 : t.capacity;
  }
  return n;
}

// Page and slot of row i of sequence b; page -1 (and the flag) when the id is no page of the pool.
__device__ __forceinline__ int32_t kv_locate(const KvView& c, const int32_t* pages, int64_t stride, int32_t b,
                                             int32_t i, int32_t* slot) {
  const uint32_t p = fast_div(static_cast<uint32_t>(i), c.page_div);
  *slot = i - static_cast<int32_t>(p) * c.page_size;
  const int32_t page = __ldg(pages + b * stride + p);
  if (static_cast<uint32_t>(page) >= c.num_pages) {
    kv_flag(c.status, NVE_B200_KV_BAD_PAGE);
    return -1;
  }
  return page;
}

__device__ __forceinline__ int64_t kv_weight_index(const KvView& c, int32_t page, int32_t head, int32_t slot) {
  return (static_cast<int64_t>(page) * c.heads + head) * c.page_size + slot;
}

}  // namespace nve_b200
