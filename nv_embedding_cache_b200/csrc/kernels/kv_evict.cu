// Eviction from the paged cache by accumulated weight: choose the rows that stay, then move them.
//
// Choosing, for every (sequence, head): the `budget` largest weights, equal ones by index.  A thread-block cluster
// takes one list, its CTAs equal runs of it.  The weights become unsigned keys in the same order (rows that must stay
// the largest of all) and stay in shared memory; a radix select over digits of 11, 11 and 10 bits finds the key of
// the last row that stays: every CTA counts the digits of its run, then every CTA adds up all CTAs' counts over
// DSMEM and finds the digit for itself, which takes one cluster barrier a digit.  Then ballots become places in
// ascending order.  No sort, no scratch in memory, the weights are read once: 4 bytes per row and head.  Latency bounds
// it (a chain of page lookup, weights, three rounds of counting, places).
//
// Moving: rows of 2 width values per kept row and head, read from anywhere, written page after page; HBM bounds it.  A
// warp looks up sixteen rows, a lane each, and copies them without a barrier.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "../common.hpp"
#include "kv_evict.hpp"

namespace nve_b200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kEach = kBins / kThreads;    // digits a thread looks after
constexpr int kMaxCluster = 8;
constexpr int kMaxCached = 40 * 1024;      // keys one CTA keeps in shared memory
constexpr uint32_t kMustStay = 0xffffffffu;
constexpr uint32_t kZero = 0x80000000u;    // key of a row that never drew any attention
constexpr uint32_t kLowest = 0x007fffffu;  // key of -inf

// Larger weight, larger key; +0 and -0 alike; NaN as -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return kLowest;
  if (w == 0.0f) return kZero;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <bool CACHED>
__global__ void __launch_bounds__(kThreads) select_kernel(const KvEvictParams p) {
  extern __shared__ __align__(16) uint32_t cached[];
  __shared__ __align__(16) uint32_t hist[2][kBins];
  __shared__ uint32_t s_warp[kWarps][2];
  __shared__ uint32_t s_found[2];          // digit, rows of larger digits
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
  const int fixed_end = length - p.recent;
  auto load_key = [&](int i) -> uint32_t {
    if (i < p.sinks || i >= fixed_end) return kMustStay;
    int32_t slot;
    const int32_t page = kv_locate(p.cache, p.table.pages, p.table.stride, b, i, &slot);
    return page < 0 ? kLowest : weight_key(p.cache.weights[kv_weight_index(p.cache, page, h, slot)]);
  };
  auto key_at = [&](int i) -> uint32_t { return CACHED ? cached[i - first] : load_key(i); };
  for (int i = tid; i < kBins; i += kThreads) hist[0][i] = hist[1][i] = 0;
  if (CACHED) {
    // four rows of a page at once where pages hold fours (runs begin at multiples of 32)
    if (p.cache.page_size % 4 == 0 && reinterpret_cast<uint64_t>(p.cache.weights) % 16 == 0) {
#pragma unroll 4
      for (int i = first + tid * 4; i < last; i += kThreads * 4) {
        int32_t slot;
        const int32_t page = kv_locate(p.cache, p.table.pages, p.table.stride, b, i, &slot);
        float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (page >= 0) w = *reinterpret_cast<const float4*>(p.cache.weights + kv_weight_index(p.cache, page, h, slot));
        const float v[4] = {w.x, w.y, w.z, w.w};
        uint32_t k[4];
#pragma unroll
        for (int x = 0; x < 4; x++)
          k[x] = i + x < p.sinks || i + x >= fixed_end ? kMustStay : (page < 0 ? kLowest : weight_key(v[x]));
        *reinterpret_cast<uint4*>(cached + (i - first)) = make_uint4(k[0], k[1], k[2], k[3]);
      }
    } else {
#pragma unroll 4
      for (int i = first + tid; i < last; i += kThreads) cached[i - first] = load_key(i);
    }
  }
  __syncthreads();

  uint32_t prefix = 0;                     // digits found so far
  // rows still to take among keys with this prefix; those that must stay are not counted
  uint32_t need = static_cast<uint32_t>(p.budget - p.sinks - p.recent);
#pragma unroll 1
  for (int pass = 0; pass < 3 && need > 0; pass++) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t bins = pass == 2 ? 1024u : 2048u;
    uint32_t* const mine = hist[pass & 1];
    if (pass == 2) {                       // every CTA is past the barrier after which none reads the first counts
      for (int i = tid; i < kBins; i += kThreads) mine[i] = 0;
      __syncthreads();
    }
    for (int i0 = first; i0 < last; i0 += kThreads) {
      const int i = i0 + tid;
      const uint32_t k = i < last ? key_at(i) : kMustStay;
      const bool counts = k != kMustStay && (pass == 0 || (k >> (pass == 1 ? 21 : 10)) == prefix);
      // rows that never drew any attention are many and alike: one addition a warp
      const uint32_t zeros = __ballot_sync(0xffffffffu, counts && k == kZero);
      if (counts && (k != kZero || lane == __ffs(zeros) - 1)) {
        atomicAdd(&mine[(k >> shift) & (bins - 1)], k == kZero ? static_cast<uint32_t>(__popc(zeros)) : 1u);
      }
    }
    cluster.sync();
    // largest digit d with (rows of digits >= d) >= need; thread 0 has the largest digits
    const int lowest = kBins - (tid + 1) * kEach;
    uint32_t sum[kEach] = {};
    for (int r = 0; r < ranks; r++) {
      const uint2 x = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(mine, r) + lowest);
      sum[0] += x.x;
      sum[1] += x.y;
    }
    uint32_t incl = sum[0] + sum[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) s_warp[warp][0] = incl;
    __syncthreads();
    uint32_t above = incl - sum[0] - sum[1];
    {
      uint32_t x = lane < warp ? s_warp[lane][0] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      above += x;
    }
#pragma unroll
    for (int x = kEach - 1; x >= 0; x--) {
      if (above < need && above + sum[x] >= need) {
        s_found[0] = static_cast<uint32_t>(lowest + x);
        s_found[1] = above;
      }
      above += sum[x];
    }
    __syncthreads();
    prefix = (prefix << (pass == 2 ? 10 : 11)) | s_found[0];
    need -= s_found[1];
    __syncthreads();
  }
  if (p.budget == p.sinks + p.recent) prefix = kMustStay - 1;   // nothing else stays
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
constexpr int kMoveRows = 16;                               // rows a warp moves
constexpr int kMoveBlockRows = kMoveRows * kMoveThreads / 32;

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const KvEvictParams p, int32_t blocks_per_list,
                                                            FastDiv chunk_div) {
  const int list = blockIdx.x / blocks_per_list;
  const int b = list / p.cache.heads, h = list - b * p.cache.heads;
  const int lane = threadIdx.x & 31;
  const int j0 = (blockIdx.x - list * blocks_per_list) * kMoveBlockRows + (threadIdx.x >> 5) * kMoveRows;
  const int count = min(kv_length(p.table, b, nullptr), p.budget);
  const int rows = min(kMoveRows, count - j0);
  if (rows <= 0) return;                                    // the whole warp
  // lanes 0-15 look up the keys of a row, lanes 16-31 its values
  const bool values = lane >= kMoveRows;
  const int mine = lane & (kMoveRows - 1);
  const uint8_t* src = nullptr;
  uint8_t* dst = nullptr;
  if (mine < rows) {
    const int j = j0 + mine;
    const int32_t from = p.kept[static_cast<int64_t>(list) * p.budget + j];
    int32_t s_slot, d_slot;
    const int32_t sp = kv_locate(p.cache, p.table.pages, p.table.stride, b, from, &s_slot);
    const int32_t dp = kv_locate(p.cache, p.new_pages, p.new_stride, b, j, &d_slot);
    if (sp >= 0 && dp >= 0) {
      const int64_t page = values ? p.cache.v_page : p.cache.k_page, slot = values ? p.cache.v_slot : p.cache.k_slot;
      uint8_t* const pool = (values ? p.cache.values : p.cache.keys) + h * (values ? p.cache.v_head : p.cache.k_head);
      src = pool + sp * page + s_slot * slot;
      dst = pool + dp * page + d_slot * slot;
      if (!values) p.cache.weights[kv_weight_index(p.cache, dp, h, d_slot)] = p.cache.weights[kv_weight_index(p.cache, sp, h, s_slot)];
    }
  }
  // keys and values of the rows: 2 * rows lines of `chunks` 16-byte pieces, line 2 r + 1 the values of row r
  const int chunks = p.row_bytes / 16, work = rows * 2 * chunks;
  constexpr int U = 4;
  for (int w0 = 0; w0 < work; w0 += 32 * U) {
    uint4 x[U];
    uint8_t* to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int w = w0 + u * 32 + lane;
      const int line = static_cast<int>(fast_div(w, chunk_div)), c = w - line * chunks;
      const int owner = ((line >> 1) & (kMoveRows - 1)) + (line & 1) * kMoveRows;
      const uint64_t s = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(src), owner);
      const uint64_t d = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(dst), owner);
      to[u] = nullptr;
      if (w < work && s != 0) {
        x[u] = *reinterpret_cast<const uint4*>(s + c * 16);
        to[u] = reinterpret_cast<uint8_t*>(d + c * 16);
      }
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
  const int32_t per_list = static_cast<int32_t>(ceil_div(most, kMoveBlockRows));
  move_kernel<<<static_cast<unsigned>(lists * per_list), kMoveThreads, 0, stream>>>(
      p, per_list, make_fast_div(static_cast<uint32_t>(p.row_bytes / 16)));
  NVE_B200_CUDA(cudaGetLastError());
}

}  // namespace nve_b200
