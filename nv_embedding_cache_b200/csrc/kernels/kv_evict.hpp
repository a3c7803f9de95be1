// Eviction from the paged cache by accumulated weight (kernels: kv_evict.cu).
#pragma once

#include "kv_common.cuh"

namespace nve_b200 {

struct KvEvictParams {
  KvView cache;
  KvTable table;
  const int32_t* new_pages;
  int64_t new_stride;
  int32_t budget, sinks, recent;
  int32_t* kept;                     // [sequences][heads][budget]
  int32_t* new_lengths;
  int32_t row_bytes;
};

void launch_kv_evict(const KvEvictParams& p, int sms, cudaStream_t stream);

}  // namespace nve_b200
