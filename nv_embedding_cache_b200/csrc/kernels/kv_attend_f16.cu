// Attention over the paged cache with fp16 rows.
#include "kv_attend.cuh"

namespace nve_b200 {
template struct KvAttendVariant<__half>;
}
