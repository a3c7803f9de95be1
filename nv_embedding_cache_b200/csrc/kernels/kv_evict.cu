// Eviction from the paged cache by accumulated weight: choose the rows that stay, then move them.
//
// Choosing, for every (sequence, head): the `budget` largest weights, equal ones by index.  A thread-block cluster
// takes one list, its CTAs equal runs of it.  The weights become unsigned keys in the same order (rows that must
// stay the largest of all) and stay in shared memory; a radix select over digits of 11, 11 and 10 bits finds the key of the last
// row that stays: every CTA counts its run, the counts are added up in the first CTA's shared memory (DSMEM), which finds
// the digit.  A second pass turns ballots into places in ascending order.  No sort, no scratch in memory, the weights
// are read once: 4 bytes per row and head.  Latency bounds it (three rounds of counting and cluster barriers).
//
// Moving: rows of 2 width values per kept row and head, read from anywhere, written page after page; HBM bounds it.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "../common.hpp"
#include "kv_evict.hpp"

namespace nve_b200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kMaxCached = 40 * 1024;      // keys one CTA keeps in shared memory
constexpr uint32_t kMustStay = 0xffffffffu;
constexpr uint32_t kLowest = 0x007fffffu;  // key of -inf

// Larger weight, larger key; +0 and -0 alike; NaN as -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return kLowest;
  if (w == 0.0f) return 0x80000000u;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <bool CACHED>
__global__ void __launch_bounds__(kThreads) select_kernel(const KvEvictParams p) {
  extern __shared__ uint32_t cached[];
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t s_warp[kWarps][2];
  __shared__ uint32_t s_found[2];          // in the first CTA: digit, rows of larger digits
  __shared__ uint32_t s_counts[2];         // of this CTA: keys above the limit, keys at it
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int list = blockIdx.x / ranks;     // (sequence, head)
  const int b = list / p.cache.heads, h = list - b * p.cache.heads;
  const int length = kv_length(p.table, b, p.cache.status);
  const int count = min(length, p.budget);
  int32_t* const kept = p.kept + static_cast<int64_t>(list) * p.budget;
  if (h == 0 && rank == 0 && tid == 0) p.new_lengths[b] = count;
  for (int j = count + rank * kThreads + tid; j < p.budget; j += ranks * kThreads) kept[j] = -1;
  if (length <= p.budget) {                // the same in every CTA of the cluster
    for (int j = rank * kThreads + tid; j < length; j += ranks * kThreads) kept[j] = j;
    return;
  }

  // runs of whole warps' steps
  const int step = ((length + ranks - 1) / ranks + 31) & ~31;
  const int first = min(rank * step, length), last = min(first + step, length);
  auto load_key = [&](int i) -> uint32_t {
    if (i < p.sinks || i >= length - p.recent) return kMustStay;
    int32_t slot;
    const int32_t page = kv_locate(p.cache, p.table.pages, p.table.stride, b, i, &slot);
    return page < 0 ? kLowest : weight_key(p.cache.weights[kv_weight_index(p.cache, page, h, slot)]);
  };
  auto key_at = [&](int i) -> uint32_t { return CACHED ? cached[i - first] : load_key(i); };

  uint32_t prefix = 0;                     // digits found so far
  uint32_t need = static_cast<uint32_t>(p.budget);   // rows still to take among keys with this prefix
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t bins = pass == 2 ? 1024u : 2048u;
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = first + tid; i < last; i += kThreads) {
      uint32_t k;
      if (CACHED && pass == 0) {
        k = load_key(i);
        cached[i - first] = k;
      } else {
        k = key_at(i);
      }
      const bool mine = pass == 0 || (k >> (pass == 1 ? 21 : 10)) == prefix;
      if (mine) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
    }
    cluster.sync();
    if (rank != 0) {
      uint32_t* const sum = cluster.map_shared_rank(hist, 0);
      for (int i = tid; i < static_cast<int>(bins); i += kThreads)
        if (hist[i] != 0) atomicAdd(sum + i, hist[i]);
    }
    cluster.sync();
    if (rank == 0) {
      // largest digit d with (rows of digits >= d) >= need
      constexpr int kEach = kBins / kThreads;
      uint32_t mine[kEach], own = 0;
#pragma unroll
      for (int x = 0; x < kEach; x++) {    // thread 0 has the largest digits
        const int d = kBins - 1 - (tid * kEach + x);
        mine[x] = hist[d];
        own += mine[x];
      }
      uint32_t incl = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      if (lane == 31) s_warp[warp][0] = incl;
      __syncthreads();
      uint32_t above = incl - own;
      for (int w = 0; w < warp; w++) above += s_warp[w][0];
#pragma unroll
      for (int x = 0; x < kEach; x++) {
        if (above < need && above + mine[x] >= need) {
          s_found[0] = static_cast<uint32_t>(kBins - 1 - (tid * kEach + x));
          s_found[1] = above;
        }
        above += mine[x];
      }
    }
    cluster.sync();
    const uint32_t* const found = cluster.map_shared_rank(s_found, 0);
    prefix = (prefix << (pass == 2 ? 10 : 11)) | found[0];
    need -= found[1];
  }
  // keys above `prefix` stay, of those equal to it the first `need`
  const int per_warp = ((last - first + kWarps - 1) / kWarps + 31) & ~31;
  const int w_first = min(first + warp * per_warp, last), w_last = min(w_first + per_warp, last);
  uint32_t above = 0, equal = 0;
  for (int i = w_first; i < w_last; i += 32) {
    const int at = i + lane;
    const uint32_t k = at < w_last ? key_at(at) : 0;
    above += __popc(__ballot_sync(0xffffffffu, at < w_last && k > prefix));
    equal += __popc(__ballot_sync(0xffffffffu, at < w_last && k == prefix));
  }
  if (lane == 0) {
    s_warp[warp][0] = above;
    s_warp[warp][1] = equal;
  }
  __syncthreads();
  if (tid < 2) {
    uint32_t sum = 0;
    for (int w = 0; w < kWarps; w++) sum += s_warp[w][tid];
    s_counts[tid] = sum;
  }
  cluster.sync();
  uint32_t n_above = 0, n_equal = 0;       // before this warp's run
  for (int r = 0; r < rank; r++) {
    const uint32_t* const c = cluster.map_shared_rank(s_counts, r);
    n_above += c[0];
    n_equal += c[1];
  }
  for (int w = 0; w < warp; w++) {
    n_above += s_warp[w][0];
    n_equal += s_warp[w][1];
  }
  const uint32_t below = (1u << lane) - 1u;
  for (int i = w_first; i < w_last; i += 32) {
    const int at = i + lane;
    const uint32_t k = at < w_last ? key_at(at) : 0;
    const bool is_above = at < w_last && k > prefix, is_equal = at < w_last && k == prefix;
    const uint32_t ma = __ballot_sync(0xffffffffu, is_above), me = __ballot_sync(0xffffffffu, is_equal);
    const uint32_t a = n_above + __popc(ma & below), e = n_equal + __popc(me & below);
    if (is_above || (is_equal && e < need)) kept[a + min(e, need)] = at;
    n_above += __popc(ma);
    n_equal += __popc(me);
  }
  cluster.sync();                          // no CTA leaves while another still reads its shared memory
}

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 32;

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const KvEvictParams p, int32_t blocks_per_list,
                                                            FastDiv chunk_div) {
  __shared__ int64_t src[2][kMoveRows], dst[2][kMoveRows];
  const int list = blockIdx.x / blocks_per_list, j0 = (blockIdx.x - list * blocks_per_list) * kMoveRows;
  const int b = list / p.cache.heads, h = list - b * p.cache.heads;
  const int count = min(kv_length(p.table, b, nullptr), p.budget);
  if (j0 >= count) return;
  const int rows = min(kMoveRows, count - j0);
  if (static_cast<int>(threadIdx.x) < rows) {
    const int j = j0 + threadIdx.x;
    const int32_t from = p.kept[static_cast<int64_t>(list) * p.budget + j];
    int32_t s_slot, d_slot;
    const int32_t sp = kv_locate(p.cache, p.table.pages, p.table.stride, b, from, &s_slot);
    const int32_t dp = kv_locate(p.cache, p.new_pages, p.new_stride, b, j, &d_slot);
    const bool ok = sp >= 0 && dp >= 0;
    src[0][threadIdx.x] = ok ? sp * p.cache.k_page + s_slot * p.cache.k_slot + h * p.cache.k_head : -1;
    src[1][threadIdx.x] = sp * p.cache.v_page + s_slot * p.cache.v_slot + h * p.cache.v_head;
    dst[0][threadIdx.x] = dp * p.cache.k_page + d_slot * p.cache.k_slot + h * p.cache.k_head;
    dst[1][threadIdx.x] = dp * p.cache.v_page + d_slot * p.cache.v_slot + h * p.cache.v_head;
    if (ok) p.cache.weights[kv_weight_index(p.cache, dp, h, d_slot)] = p.cache.weights[kv_weight_index(p.cache, sp, h, s_slot)];
  }
  __syncthreads();
  const int chunks = p.row_bytes / 16, work = rows * 2 * chunks;   // keys of a row, then its values
  constexpr int U = 4;
  for (int w0 = threadIdx.x; w0 < work; w0 += kMoveThreads * U) {
    uint4 x[U];
    uint8_t* to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int w = w0 + u * kMoveThreads;
      to[u] = nullptr;
      if (w >= work) continue;
      const int r2 = static_cast<int>(fast_div(w, chunk_div)), c = w - r2 * chunks;
      const int r = r2 >> 1, kv = r2 & 1;
      if (src[0][r] < 0) continue;
      x[u] = *reinterpret_cast<const uint4*>((kv ? p.cache.values : p.cache.keys) + src[kv][r] + c * 16);
      to[u] = (kv ? p.cache.values : p.cache.keys) + dst[kv][r] + c * 16;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (to[u] != nullptr) *reinterpret_cast<uint4*>(to[u]) = x[u];
  }
}

template <bool CACHED>
void launch_select(const KvEvictParams& p, int ranks, size_t smem, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};    // one bit per device
  int dev = 0;
  NVE_B200_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (CACHED && !(done.load(std::memory_order_acquire) & bit)) {
    NVE_B200_CUDA(cudaFuncSetAttribute(select_kernel<CACHED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCached * 4));
    done.fetch_or(bit, std::memory_order_acq_rel);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.table.sequences * p.cache.heads * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(ranks);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  NVE_B200_CUDA(cudaLaunchKernelEx(&cfg, select_kernel<CACHED>, p));
}

}  // namespace

void launch_kv_evict(const KvEvictParams& p, int sms, cudaStream_t stream) {
  const int64_t lists = static_cast<int64_t>(p.table.sequences) * p.cache.heads;
  // CTAs of a cluster: enough for every SM to have work, as long as each still has 2048 rows; more where a run
  // would not fit into shared memory
  int ranks = 1;
  while (ranks < kMaxCluster && ((lists * ranks < sms && p.table.capacity / ranks >= 4096) ||
                                 p.table.capacity / ranks > kMaxCached - 64)) {
    ranks *= 2;
  }
  const int step = ((p.table.capacity + ranks - 1) / ranks + 31) & ~31;
  if (step <= kMaxCached) launch_select<true>(p, ranks, size_t(step) * 4, stream);
  else launch_select<false>(p, ranks, 0, stream);
  const int32_t most = std::min(p.budget, p.table.capacity);
  if (most == 0) return;
  const int32_t per_list = static_cast<int32_t>(ceil_div(most, kMoveRows));
  move_kernel<<<static_cast<unsigned>(lists * per_list), kMoveThreads, 0, stream>>>(
      p, per_list, make_fast_div(static_cast<uint32_t>(p.row_bytes / 16)));
  NVE_B200_CUDA(cudaGetLastError());
}

}  // namespace nve_b200
