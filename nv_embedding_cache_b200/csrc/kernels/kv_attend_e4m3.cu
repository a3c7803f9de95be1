// Attention over the paged cache with E4M3 rows.
#include "kv_attend.cuh"

namespace nve_b200 {
template struct KvAttendVariant<__nv_fp8_e4m3>;
}
