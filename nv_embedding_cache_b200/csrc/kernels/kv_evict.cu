// Eviction from the paged cache by accumulated weight: choose the rows that stay, then move them.
//
// Choosing, for every (sequence, head): the `budget` largest weights, equal ones by index.  A thread-block cluster
// takes one list, its CTAs equal runs of it.  The weights become unsigned keys in the same order (rows that must stay
// the largest of all) and stay in shared memory; a radix select over digits of 11, 11 and 10 bits finds the key of
// the last row that stays: every CTA counts the digits of its run, and after one cluster barrier a digit a warp of
// every CTA finds it for itself from all CTAs' counts, read over DSMEM: first among 64 sums of 32 digits, then among
// those 32 (reading all 2048 counts of eight CTAs instead: 33 us against 21 for 32 lists of 26 000 rows).  Then ballots
// become places in ascending order.  No sort, no scratch in memory, the weights are read once: 4 bytes per row and head.
// Latency bounds it (a chain of page lookup, weights, three rounds of counting, places): 10 us for 128 lists of 1000
// rows, 24 us for 4 of 131 071.
//
// Moving: rows of 2 width values per kept row and head, read from anywhere, written page after page; HBM bounds it.
// Small blocks, many per SM: a block looks its rows up, a thread each, and copies them with four 16-byte pieces of a
// thread in flight.  Warps that do both for themselves, or look the next rows up while they copy, keep fewer loads in
// flight and took 60 and 69 us where this takes 48 (32 lists of 8192 rows of 256 bytes: 5.6 TB/s).
// New pages are looked up before the wait for the choosing launch.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "../common.hpp"
#include "kv_evict.hpp"
#include "kv_launch.cuh"

namespace nve_b200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kBins = 2048;
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

template <bool CACHED, int kThreads>
__global__ void __launch_bounds__(kThreads) select_kernel(const KvEvictParams p) {
  constexpr int kWarps = kThreads / 32;
  extern __shared__ __align__(16) uint32_t cached[];
  __shared__ __align__(16) uint32_t hist[2][kBins];
  __shared__ uint32_t coarse[2][64];       // sums of 32 counts
  __shared__ uint32_t s_warp[kWarps][2];
  __shared__ uint32_t s_found[3];          // digit, rows of larger digits, rows of this digit
  __shared__ uint32_t s_counts[2];         // of this CTA: keys above the limit, keys at it
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int list = blockIdx.x / ranks;     // (sequence, head)
  const int b = list / p.cache.heads, h = list - b * p.cache.heads;
  grid_wait();
  grid_release();
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
  auto all_sync = [&]() {
    if (ranks > 1) cluster.sync();
    else __syncthreads();
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
          k[x] = i + x < p.sinks || i + x >= fixed_end || i + x >= last ? kMustStay : (page < 0 ? kLowest : weight_key(v[x]));
        *reinterpret_cast<uint4*>(cached + (i - first)) = make_uint4(k[0], k[1], k[2], k[3]);
      }
    } else {
#pragma unroll 4
      for (int i = first + tid; i < last; i += kThreads) cached[i - first] = load_key(i);
    }
    for (int i = last - first + tid; i < step; i += kThreads) cached[i] = kMustStay;   // behind the run
  }
  __syncthreads();

  uint32_t prefix = 0;                     // digits found so far
  bool decided = false;
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
    const int known = pass == 1 ? 21 : 10;                  // bits below those of the prefix
    // rows that never drew any attention are many and alike: one addition a warp
    const auto add_zeros = [&](uint32_t of_this_thread) {
      const uint32_t zeros = __reduce_add_sync(0xffffffffu, of_this_thread);
      if (lane == 0 && zeros != 0) atomicAdd(&mine[(kZero >> shift) & (bins - 1)], zeros);
    };
    const auto add = [&](uint32_t k, uint32_t& zeros) {
      if (k == kMustStay || (pass != 0 && (k >> known) != prefix)) return;
      if (k == kZero) zeros++;
      else atomicAdd(&mine[(k >> shift) & (bins - 1)], 1u);
    };
    if (CACHED) {                          // four keys a load; those behind the run must stay, so they are not counted
      for (int i0 = 0; i0 < step; i0 += kThreads * 4) {
        const int i = i0 + tid * 4;
        uint32_t zeros = 0;
        if (i < step) {
          const uint4 k = *reinterpret_cast<const uint4*>(cached + i);
          add(k.x, zeros);
          add(k.y, zeros);
          add(k.z, zeros);
          add(k.w, zeros);
        }
        add_zeros(zeros);
      }
    } else {
      for (int i0 = first; i0 < last; i0 += kThreads) {
        uint32_t zeros = 0;
        if (i0 + tid < last) add(load_key(i0 + tid), zeros);
        add_zeros(zeros);
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int c = warp; c < 64; c += kWarps) {
      const uint32_t x = __reduce_add_sync(0xffffffffu, mine[c * 32 + lane]);
      if (lane == 0) coarse[pass & 1][c] = x;
    }
    all_sync();
    // largest digit d with (rows of digits >= d) >= need; lane 0 has the largest digits
    if (warp == 0) {
      uint32_t hi = 0, lo = 0;
      if (ranks == 1) {
        hi = coarse[pass & 1][63 - 2 * lane];
        lo = coarse[pass & 1][62 - 2 * lane];
      } else {
#pragma unroll
        for (int r = 0; r < kMaxCluster; r++) {
          if (r < ranks) {
            const uint32_t* const theirs = cluster.map_shared_rank(coarse[pass & 1], r);
            hi += theirs[63 - 2 * lane];
            lo += theirs[62 - 2 * lane];
          }
        }
      }
      const auto before = [&](uint32_t x) {                 // sum over the lanes before this one
        uint32_t incl = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        return incl - x;
      };
      uint32_t above = before(hi + lo);
      const bool in_hi = above < need && above + hi >= need;
      const bool in_lo = above + hi < need && above + hi + lo >= need;
      if (in_lo) above += hi;
      const int src = __ffs(__ballot_sync(0xffffffffu, in_hi || in_lo)) - 1;
      const int c = __shfl_sync(0xffffffffu, in_hi ? 63 - 2 * lane : 62 - 2 * lane, src);
      above = __shfl_sync(0xffffffffu, above, src);
      const int digit = c * 32 + 31 - lane;
      uint32_t x = 0;
      if (ranks == 1) {
        x = mine[digit];
      } else {
#pragma unroll
        for (int r = 0; r < kMaxCluster; r++)
          if (r < ranks) x += cluster.map_shared_rank(mine, r)[digit];
      }
      above += before(x);
      if (above < need && above + x >= need) {
        s_found[0] = static_cast<uint32_t>(digit);
        s_found[1] = above;
        s_found[2] = x;
      }
    }
    __syncthreads();
    prefix = (prefix << (pass == 2 ? 10 : 11)) | s_found[0];
    need -= s_found[1];
    const bool all_of_it = need == s_found[2];   // whatever their lower digits are
    __syncthreads();
    if (all_of_it) {
      // keys above `prefix` 0..0 - 1: all of these, and none is left to choose among equals
      prefix = (pass == 2 ? prefix : prefix << shift) - 1;
      need = 0;
      decided = true;
      break;
    }
  }
  if (!decided && need == 0) prefix = kMustStay - 1;            // nothing but what must stay
  // keys above `prefix` stay, of those equal to it the first `need`
  const int per_warp = ((last - first + kWarps - 1) / kWarps + 31) & ~31;
  const int w_first = min(first + warp * per_warp, last), w_last = min(w_first + per_warp, last);
  uint32_t above = 0, equal = 0;
#pragma unroll 4
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
  all_sync();
  uint32_t n_above = 0, n_equal = 0;       // before this warp's run
#pragma unroll
  for (int r = 0; r < kMaxCluster; r++) {
    if (r < rank) {
      const uint32_t* const c = cluster.map_shared_rank(s_counts, r);
      n_above += c[0];
      n_equal += c[1];
    }
  }
  for (int w = 0; w < warp; w++) {
    n_above += s_warp[w][0];
    n_equal += s_warp[w][1];
  }
  const uint32_t below = (1u << lane) - 1u;
#pragma unroll 4
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
  if (ranks > 1) cluster.sync();           // no CTA leaves while another still reads its shared memory
}

constexpr int kMoveThreads = 128;
constexpr int kMoveRows = 32;              // rows a block moves

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const KvEvictParams p, int32_t blocks_per_list,
                                                            FastDiv chunk_div) {
  __shared__ const uint8_t* src[2 * kMoveRows];   // keys of row r at 2 r, values at 2 r + 1; nullptr: left out
  __shared__ uint8_t* dst[2 * kMoveRows];
  const int list = blockIdx.x / blocks_per_list, j0 = (blockIdx.x - list * blocks_per_list) * kMoveRows;
  const int b = list / p.cache.heads, h = list - b * p.cache.heads;
  const int count = min(kv_length(p.table, b, nullptr), p.budget);
  const int rows = min(kMoveRows, count - j0), j = j0 + static_cast<int>(threadIdx.x);
  int32_t dp = -1, d_slot = 0;
  if (static_cast<int>(threadIdx.x) < rows) dp = kv_locate(p.cache, p.new_pages, p.new_stride, b, j, &d_slot);
  grid_wait();
  grid_release();
  if (rows <= 0) return;
  if (static_cast<int>(threadIdx.x) < rows) {
    const int32_t from = p.kept[static_cast<int64_t>(list) * p.budget + j];
    int32_t s_slot;
    const int32_t sp = kv_locate(p.cache, p.table.pages, p.table.stride, b, from, &s_slot);
    const bool ok = sp >= 0 && dp >= 0;
    src[2 * threadIdx.x] = ok ? p.cache.keys + sp * p.cache.k_page + s_slot * p.cache.k_slot + h * p.cache.k_head : nullptr;
    src[2 * threadIdx.x + 1] = ok ? p.cache.values + sp * p.cache.v_page + s_slot * p.cache.v_slot + h * p.cache.v_head : nullptr;
    dst[2 * threadIdx.x] = p.cache.keys + dp * p.cache.k_page + d_slot * p.cache.k_slot + h * p.cache.k_head;
    dst[2 * threadIdx.x + 1] = p.cache.values + dp * p.cache.v_page + d_slot * p.cache.v_slot + h * p.cache.v_head;
    if (ok) p.cache.weights[kv_weight_index(p.cache, dp, h, d_slot)] = p.cache.weights[kv_weight_index(p.cache, sp, h, s_slot)];
  }
  __syncthreads();
  const int chunks = p.row_bytes / 16, work = rows * 2 * chunks;
  constexpr int U = 4;
  for (int w0 = threadIdx.x; w0 < work; w0 += kMoveThreads * U) {
    uint4 x[U];
    uint8_t* to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int w = w0 + u * kMoveThreads;
      to[u] = nullptr;
      if (w >= work) continue;
      const int line = static_cast<int>(fast_div(w, chunk_div)), c = w - line * chunks;
      const uint8_t* const s = src[line];
      if (s == nullptr) continue;
      x[u] = *reinterpret_cast<const uint4*>(s + c * 16);
      to[u] = dst[line] + c * 16;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (to[u] != nullptr) *reinterpret_cast<uint4*>(to[u]) = x[u];
  }
}

template <bool CACHED, int kThreads>
void launch_select(const KvEvictParams& p, int ranks, size_t smem, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};    // one bit per device
  int dev = 0;
  NVE_B200_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t{1} << (dev & 63);
  const auto kernel = select_kernel<CACHED, kThreads>;
  if (CACHED && !(done.load(std::memory_order_acquire) & bit)) {
    NVE_B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCached * 4));
    done.fetch_or(bit, std::memory_order_acq_rel);
  }
  launch_overlapped(kernel, static_cast<int64_t>(p.table.sequences) * p.cache.heads * ranks, kThreads, smem,
                    static_cast<unsigned>(ranks), stream, p);
}

}  // namespace

void launch_kv_evict(const KvEvictParams& p, int sms, cudaStream_t stream) {
  const int64_t lists = static_cast<int64_t>(p.table.sequences) * p.cache.heads;
  // CTAs of a cluster: enough for every SM to have work, as long as each still has 2048 rows; more where a run
  // would not fit into shared memory
  int ranks = 1;
  while (ranks < kMaxCluster && ((lists * ranks * 2 <= sms && p.table.capacity / ranks >= 4096) ||
                                 p.table.capacity / ranks > kMaxCached - 64)) {
    ranks *= 2;
  }
  const int step = ((p.table.capacity + ranks - 1) / ranks + 31) & ~31;
  if (step <= 4096) launch_select<true, 256>(p, ranks, size_t(step) * 4, stream);
  else if (step <= kMaxCached) launch_select<true, 1024>(p, ranks, size_t(step) * 4, stream);
  else launch_select<false, 1024>(p, ranks, 0, stream);
  const int32_t most = std::min(p.budget, p.table.capacity);
  if (most == 0) return;
  const int32_t per_list = static_cast<int32_t>(ceil_div(most, kMoveRows));
  launch_overlapped(move_kernel, lists * per_list, kMoveThreads, 0, 1, stream, p, per_list,
                    make_fast_div(static_cast<uint32_t>(p.row_bytes / 16)));
}

}  // namespace nve_b200
