// Attention over the paged cache with bf16 rows.
#include "kv_attend.cuh"

namespace nve_b200 {
template struct KvAttendVariant<__nv_bfloat16>;
}
