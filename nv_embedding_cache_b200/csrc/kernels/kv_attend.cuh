// Attention of one new token per sequence over the paged cache: the kernel that reads the cache.
//
//   s_j = scale q.k_j,   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = s_j log2(e)
// in one pass over the rows with a running maximum m, its sum and the weighted sum of values (fp32).
//
// What bounds it: 2 width values are read per (row, key head) and 4 width flops done per query head of the group, so
// even 16 query heads on one key head ask for a few per cent of the tensor rate: memory does.  Everything here is
// there to keep loads in flight on every SM, whatever the batch looks like:
//  * the tiles (64 or 128 rows of one key head) of the whole batch are one list, cut into equal runs, one per resident CTA
//    (kv_plan.hpp): one long sequence and a ragged batch load all SMs alike.  A unit that falls into several
//    runs leaves (m, sum, weighted sum) per run in scratch and is joined by kv_join.cu.
//  * a CTA's tiles are one stream through a ring of shared-memory stages.  Two warps do nothing but look rows up in
//    the page table and fill the ring with cp.async (16 bytes each: a page may end anywhere in a tile, rows have
//    any strides), four warps compute; full and empty barriers per stage, no barrier over all warps.  The ring
//    runs on across units, the queries of a unit travel with its first tile.
//  * mma.sync m16n8k16, not tcgen05, with the cache as the left operand: keys (16 rows x 16 values) times queries
//    (16 values x 8 heads), values transposed (16 values x 16 rows) times probabilities (16 rows x 8 heads).  A unit has as
//    few as one query head; eight columns are the least there is, and the scores stay in the registers that the second
//    product takes them from (transposed by movmatrix).  In a tcgen05 product they would go through TMEM and shared
//    memory every tile, for a rate that the loads cannot feed.
// Measured: 126 us for 64 sequences of 300 to 6000 rows, 32 query heads on 8, bf16 rows of 128 (6.1 TB/s of DRAM traffic, 0.94
// of a copy's rate), 90 us for one of 131 072 rows, 185 us for 128 sequences over E4M3 rows (5.9 TB/s with the scores).
// With up to 16 query heads each computing warp takes its share of the tile's rows and has its own running maximum, and the
// warps are joined when the unit ends; with more, warps take 16 heads each and share the rows.
//
// Probabilities are rounded to the type of the values (f16 for E4M3 rows: exact for them, see below) before the
// second product: relative 2^-9 (bf16) or 2^-12 of each, below the rounding of the output; the sum is taken before that.
// E4M3 rows become f16 on the way to the tensor cores, which is exact; the scales go into the scores and the output.
#pragma once

#include <algorithm>
#include <atomic>

#include "../common.hpp"
#include "bulk_copy.cuh"
#include "kv_attend.hpp"
#include "kv_launch.cuh"

namespace nve_b200 {

namespace kv {

constexpr int kComputeWarps = 4;
constexpr int kLoadWarps = 2;
constexpr int kThreads = (kComputeWarps + kLoadWarps) * 32;
constexpr float kNegInf = -__builtin_huge_valf();

// The cache is read once: its lines are the first to leave L2 again, and the scores, which the join reads, stay (64
// sequences of 3000 rows: 149 -> 138 us for both launches).
__device__ __forceinline__ uint64_t read_once() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0),
               "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async16_full(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
// The barrier gets this thread's arrival when its copies so far are done.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kComputeWarps * 32) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
// 8x8 matrix of 16-bit values, a row per four lanes, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four E4M3 values as two f16x2; exact
__device__ __forceinline__ void e4m3_to_f16(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ void store16(uint8_t* p, float x, bool bf16) {
  if (bf16) *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(x);
  else *reinterpret_cast<__half*>(p) = __float2half_rn(x);
}
// over the lanes that hold the same columns (rows lane / 4)
__device__ __forceinline__ float column_max(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float column_sum(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// ST: stored type.  DP: width rounded up to 64, 128 or 256.  WM: warps along the query heads.  NT: columns of 8 heads of a
// warp.
template <typename ST, int DP, int WM, int NT>
struct Shape {
  static constexpr bool kE4m3 = sizeof(ST) == 1;
  static constexpr int kRowBytes = DP * sizeof(ST);
  static constexpr int kChunks = kRowBytes / 16;          // 16-byte chunks of a row
  static constexpr int kTile = kv_tile_rows(DP, sizeof(ST));
  static constexpr int kTileBytes = kTile * kRowBytes;    // keys or values of a tile
  static constexpr int kWT = kComputeWarps / WM;          // warps along the rows
  static constexpr int kWarpRows = kTile / kWT;           // rows of a tile one warp takes
  static constexpr int kUnitRows = 8 * NT * WM;           // query rows
  static constexpr int kQBytes = kUnitRows * DP * 2;
  // A stage holds a tile and the queries of the unit that may begin with it.  Two CTAs per SM of three or more stages
  // where they fit, else one: 130 KB and more in flight per SM; the memory's latency times its rate asks for 45 KB.
  static constexpr int kStageBytes = 2 * kTileBytes + kQBytes;
  static constexpr int kMinCtas = 3 * kStageBytes <= 111000 ? 2 : 1;
  static constexpr int kStages = kMinCtas == 2 ? (111000 / kStageBytes < 5 ? 111000 / kStageBytes : 5)
                                               : (222000 / kStageBytes < 5 ? 222000 / kStageBytes : 5);
  static constexpr int kMaskWords = kTile / 32;
  static constexpr int kOffsBytes = kTile * 16;
  static constexpr int kSmem = kStages * kStageBytes + kOffsBytes + kComputeWarps * 8 * NT * 8 + kStages * kMaskWords * 4 +
                               kUnitRows * 4 + kStages * 16 + 16;
  static_assert(kStages >= 2, "stages");
};

// Byte offset of 16-byte chunk c of row r: chunks of 128 bytes are permuted by the row, so that the eight rows one
// ldmatrix takes at the same c lie in different banks.
template <int ROW_BYTES>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if constexpr (ROW_BYTES >= 128) return r * ROW_BYTES + ((c ^ (r & 7)) << 4);
  else return r * ROW_BYTES + ((c ^ ((r >> 1) & 3)) << 4);       // 64-byte rows: two per 128 bytes
}

template <typename ST, int DP, int WM, int NT>
__global__ void __launch_bounds__(kThreads, Shape<ST, DP, WM, NT>::kMinCtas) attend_kernel(const KvAttendParams p) {
  using S = Shape<ST, DP, WM, NT>;
  constexpr int kHeads = 8 * NT;                           // query heads of a warp
  constexpr bool kE4m3 = S::kE4m3;
  constexpr bool kBf16 = std::is_same<ST, __nv_bfloat16>::value;
  constexpr int kSteps = DP / 16;                          // k steps of the first product, column blocks of the second
  constexpr int kBlocks = S::kWarpRows / 16;               // 16-row blocks of a warp's rows
  constexpr bool kKeepQ = DP <= 128;                       // the queries stay in registers; wider ones in shared memory
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const qbuf = smem + S::kStages * 2 * S::kTileBytes;
  longlong2* const offs = reinterpret_cast<longlong2*>(qbuf + S::kStages * S::kQBytes);             // [kTile]
  uint64_t* const full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(offs) + S::kOffsBytes);   // [kStages]
  uint64_t* const empty = full + S::kStages;                                                        // [kStages]
  float2* const ml = reinterpret_cast<float2*>(empty + S::kStages);                                 // [warps][kHeads]
  uint32_t* const masks = reinterpret_cast<uint32_t*>(ml + kComputeWarps * kHeads);                 // [kStages][kMaskWords]
  float* const q_up = reinterpret_cast<float*>(masks + S::kStages * S::kMaskWords);                 // [kUnitRows]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int width = p.cache.width;
  const int units = p.cache.heads * p.chunks;

  if (tid == 0) {
    for (int s = 0; s < S::kStages; s++) {
      // every loading thread's copies, and each loading warp's word on which rows are there
      mbar_init(full + s, kLoadWarps * 32 + kLoadWarps);
      mbar_init(empty + s, kComputeWarps);
    }
  }
  grid_wait();
  // ---- the number of tiles, and where this CTA's run of them begins
  __shared__ int32_t s_sum[kThreads / 32];
  __shared__ int32_t s_start[3];
  {
    int32_t mine = 0;
    for (int b = tid; b < p.table.sequences; b += kThreads) mine += tiles_of(kv_length(p.table, b, p.cache.status), S::kTile);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
  }
  int32_t total = 0;                                        // below 2^31, as the host has seen to
#pragma unroll
  for (int w = 0; w < kThreads / 32; w++) total += s_sum[w];
  total *= units;
  // no tile names a sequence without rows
  for (int b = blockIdx.x; b < p.table.sequences; b += gridDim.x) {
    if (kv_length(p.table, b, nullptr) == 0) {
      for (int i = tid; i < p.q_heads * width; i += kThreads) {
        const int h = i / width, d = i - h * width;
        store16(p.out + b * p.out_seq + h * p.out_head + d * 2, 0.0f, p.q_bf16);
      }
      if (p.lse != nullptr) {
        for (int h = tid; h < p.q_heads; h += kThreads) p.lse[static_cast<int64_t>(b) * p.q_heads + h] = kNegInf;
      }
    }
  }
  if (total == 0) return;
  const int32_t n_ctas = min(static_cast<int32_t>(gridDim.x), total), me = blockIdx.x;
  if (me >= n_ctas) return;
  const TileSplit split = tile_split(total, n_ctas);
  const int32_t first_tile = run_first(split, me);
  const int n_tiles = run_first(split, me + 1) - first_tile;

  if (warp == 0) {                                          // 32 sequences a step
    int32_t before = 0;
    for (int base = 0; base < p.table.sequences; base += 32) {
      const int b = base + lane;
      const int nt = b < p.table.sequences ? tiles_of(kv_length(p.table, b, nullptr), S::kTile) : 0;
      const int32_t here = nt * units;
      int32_t incl = here;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const int32_t at = first_tile - (before + incl - here);
      const bool found = at >= 0 && at < here;
      if (found) {
        s_start[0] = b;
        s_start[1] = at / nt;
        s_start[2] = at % nt;
      }
      if (__any_sync(0xffffffffu, found)) break;
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  __syncthreads();
  TileCursor at;
  at.b = s_start[0];
  at.head = s_start[1] / p.chunks;
  at.chunk = s_start[1] - at.head * p.chunks;
  at.j = s_start[2];
  at.length = kv_length(p.table, at.b, nullptr);
  at.tiles = tiles_of(at.length, S::kTile);
  int stage = 0;
  uint32_t phase = 0;                                       // of the stage's barriers

  grid_release();                                           // the join reads what this grid writes after its wait only

  if (warp >= kComputeWarps) {
    // ================================ loading warps ================================
    constexpr int kOwnRows = S::kTile / kLoadWarps;         // rows of a tile this warp looks after
    constexpr int kEach = kOwnRows / 32;
    const int lw = warp - kComputeWarps;
    const int row_chunks = width * static_cast<int>(sizeof(ST)) / 16, q_chunks = width / 8;
    const int pair_chunks = (row_chunks + 1) & ~1;          // what the products read
    const uint64_t policy = read_once();
    longlong2* const own = offs + lw * kOwnRows;
    // addresses of this lane's rows (keys, values) of the tile `at`; 0: no such row
    auto locate = [&](longlong2 (&o)[kEach]) {
#pragma unroll
      for (int x = 0; x < kEach; x++) {
        const int32_t row = at.j * S::kTile + lw * kOwnRows + x * 32 + lane;
        o[x] = make_longlong2(0, 0);
        if (row < at.length) {
          int32_t slot;
          const int32_t page = kv_locate(p.cache, p.table.pages, p.table.stride, at.b, row, &slot);
          if (page >= 0) {
            o[x].x = reinterpret_cast<int64_t>(p.cache.keys) + page * p.cache.k_page + slot * p.cache.k_slot + at.head * p.cache.k_head;
            o[x].y = reinterpret_cast<int64_t>(p.cache.values) + page * p.cache.v_page + slot * p.cache.v_slot + at.head * p.cache.v_head;
          }
        }
      }
    };
    // A step of the warp copies 32 chunks, kRowsStep whole rows.  The permutation of the chunks repeats every 8 rows, so
    // a lane's place in the stage is one of kPeriod bases and a constant.
    static_assert(S::kChunks <= 32, "a row is at most one step");
    constexpr int kRowsStep = 32 / S::kChunks;
    constexpr int kPeriod = 8 / kRowsStep;
    constexpr int kCopies = kOwnRows / kRowsStep;
    const int r_lane = lane / S::kChunks, c_lane = lane % S::kChunks;
    longlong2 next[kEach];
    locate(next);
    int q_at = 0;                                           // buffer of the unit's queries
#pragma unroll 1
    for (int i = 0; i < n_tiles; i++) {
      if (!mbar_wait_bounded(empty + stage, phase ^ 1)) {   // the first round passes at once
        kv_flag(p.cache.status, NVE_B200_KV_TIMED_OUT);
        break;
      }
      __syncwarp();
      bool all_there = row_chunks == S::kChunks;
#pragma unroll
      for (int x = 0; x < kEach; x++) {
        own[x * 32 + lane] = next[x];
        const uint32_t mask = __ballot_sync(0xffffffffu, next[x].x != 0);
        if (lane == 0) masks[stage * S::kMaskWords + lw * kEach + x] = mask;
        all_there = all_there && mask == 0xffffffffu;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(full + stage);
      const bool first = i == 0 || at.j == 0;
      const TileCursor now = at;
      at.advance(p.table, p.cache.heads, p.chunks, S::kTile);
      if (i + 1 < n_tiles) locate(next);                    // its page ids arrive while this tile's copies are issued
      const uint32_t k_addr = smem_addr(smem) + stage * 2 * S::kTileBytes + lw * kOwnRows * S::kRowBytes;
      if (all_there) {
#pragma unroll
        for (int y = 0; y < kPeriod; y++) {
          const uint32_t to = k_addr + chunk_at<S::kRowBytes>(y * kRowsStep + r_lane, c_lane);
          const longlong2* const from = own + y * kRowsStep + r_lane;
#pragma unroll
          for (int x = 0; x < kCopies / kPeriod; x++) {
            const longlong2 o = from[x * 8];
            const uint32_t dst = to + x * 8 * S::kRowBytes;
            cp_async16_full(dst, reinterpret_cast<const uint8_t*>(o.x) + c_lane * 16, policy);
            cp_async16_full(dst + S::kTileBytes, reinterpret_cast<const uint8_t*>(o.y) + c_lane * 16, policy);
          }
        }
      } else {
        // the lane's chunk moves on by 32 chunks of rows of pair_chunks
        const int r_step = 32 / pair_chunks, c_step = 32 - r_step * pair_chunks;
        int r = lane / pair_chunks, c = lane - r * pair_chunks;
#pragma unroll 2
        for (int x = 0; x < kOwnRows / 32 * pair_chunks; x++) {
          const longlong2 o = own[r];
          // the chunk that makes the count even, and rows that are not there, become zeros: a NaN left in a page
          // never meets the products
          const bool ok = o.x != 0 && c < row_chunks;
          const uint32_t dst = k_addr + chunk_at<S::kRowBytes>(r, c);
          cp_async16(dst, ok ? reinterpret_cast<const uint8_t*>(o.x) + c * 16 : p.cache.keys, ok, policy);
          cp_async16(dst + S::kTileBytes, ok ? reinterpret_cast<const uint8_t*>(o.y) + c * 16 : p.cache.values, ok, policy);
          r += r_step;
          c += c_step;
          if (c >= pair_chunks) {
            c -= pair_chunks;
            r++;
          }
        }
      }
      if (first) {                                          // the unit's queries
        if (i > 0) q_at = q_at + 1 == S::kStages ? 0 : q_at + 1;
        const uint32_t q_addr = smem_addr(qbuf) + q_at * S::kQBytes;
        const int q_first = now.chunk * p.chunk;
        const int n = min(p.chunk, p.group - q_first);
        const uint8_t* const src = p.q + now.b * p.q_seq + (now.head * p.group + q_first) * p.q_head;
        for (int id = lw * 32 + lane; id < S::kUnitRows * (DP / 8); id += kLoadWarps * 32) {
          const int r = id / (DP / 8), c = id % (DP / 8);
          const bool ok = r < n && c < q_chunks;
          cp_async16(q_addr + chunk_at<DP * 2>(r, c), ok ? src + r * p.q_head + c * 16 : p.q, ok, policy);
        }
      }
      cp_async_arrive(full + stage);
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
      __syncwarp();
    }
    cp_async_wait_all();
    return;
  }

  // ================================ computing warps ================================
  const int wm = warp % WM, wt = warp / WM;                 // heads kHeads wm.., rows kWarpRows wt.. of the tile
  const int row = lane >> 2, col = (lane & 3) * 2;          // of a product's 16 x 8 results: rows row, row + 8, columns col, col + 1
  // steps of 16 values that hold any: the columns behind them are neither copied nor multiplied
  const int steps = kE4m3 ? ((width + 31) / 32) * 2 : (width + 15) / 16;
  float acc[kSteps][NT][4];                                 // values x heads
  float m_run[NT][2], l_run[NT][2];                         // of heads col, col + 1; the sum of this lane's rows
  uint32_t qf[kKeepQ ? kSteps : 1][NT][2];
  float scale[NT][2];
  bool from_start = false;                                  // this CTA has the current unit from its first tile
  int q_use = 0;

#pragma unroll 1
  for (int i = 0; i < n_tiles; i++) {
    if (!mbar_wait_bounded(full + stage, phase)) {          // all warps wait for the same event: all give up
      kv_flag(p.cache.status, NVE_B200_KV_TIMED_OUT);
      return;
    }
    const int head = at.head;
    const int unit_first = at.chunk * p.chunk;              // first query head of the unit inside its group
    const int unit_heads = min(p.chunk, p.group - unit_first);
    // queries of one step (16 values): the two registers of head `row` of each column block
    auto load_q = [&](int step, uint32_t (&b)[NT][2]) {
      const uint32_t base = smem_addr(qbuf) + q_use * S::kQBytes;
      if constexpr (kE4m3) {
        // a lane gets four consecutive values of an E4M3 row; the values of q are dealt out alike
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const uint32_t addr = base + chunk_at<DP * 2>(wm * kHeads + n * 8 + row, step * 2 + ((lane & 3) >> 1)) + (lane & 1) * 8;
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(b[n][0]), "=r"(b[n][1]) : "r"(addr) : "memory");
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const uint32_t addr = base + chunk_at<DP * 2>(wm * kHeads + n * 8 + row, step * 2 + x) + col * 2;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(b[n][x]) : "r"(addr) : "memory");
          }
      }
    };
    if (i == 0 || at.j == 0) {
      if (i > 0) q_use = q_use + 1 == S::kStages ? 0 : q_use + 1;
      from_start = at.j == 0;
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int s = 0; s < kSteps; s++)
#pragma unroll
          for (int e = 0; e < 4; e++) acc[s][n][e] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; e++) {
          m_run[n][e] = kNegInf;
          l_run[n][e] = 0.0f;
          scale[n][e] = p.scale_log2;
        }
      }
      if constexpr (kE4m3) {
        // Queries meet E4M3 rows as f16.  bf16 ones are brought into its range row by row: divided by the power of
        // two of the row's largest value, which the scores get back; exact but for values 2^-24 below that.
        if (p.q_bf16) {
          for (int r = warp; r < S::kUnitRows; r += kComputeWarps) {
            uint32_t* const words = reinterpret_cast<uint32_t*>(qbuf + q_use * S::kQBytes) + r * (DP / 2);
            float2 v[DP / 64];
            uint32_t top = 0;
#pragma unroll
            for (int x = 0; x < DP / 64; x++) {
              const uint32_t w = words[x * 32 + lane];
              v[x] = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
              const uint32_t ea = (__float_as_uint(v[x].x) >> 23) & 255u, eb = (__float_as_uint(v[x].y) >> 23) & 255u;
              top = max(top, max(ea == 255u ? 0u : ea, eb == 255u ? 0u : eb));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (top == 0) top = 127;
            top = min(top, 253u);
            const float down = __uint_as_float((254u - top) << 23);
#pragma unroll
            for (int x = 0; x < DP / 64; x++) words[x * 32 + lane] = pack2<false>(v[x].x * down, v[x].y * down);
            if (lane == 0) q_up[r] = __uint_as_float(top << 23);
          }
          compute_sync();
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) scale[n][e] *= q_up[wm * kHeads + n * 8 + col + e];
        }
        if (p.cache.key_scale != nullptr) {
          const float s = __ldg(p.cache.key_scale + head);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) scale[n][e] *= s;
        }
      }
      if constexpr (kKeepQ) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) load_q(s, qf[s]);
      }
    }

    const uint32_t k_addr = smem_addr(smem) + stage * 2 * S::kTileBytes, v_addr = k_addr + S::kTileBytes;
    const int left = at.length - at.j * S::kTile;           // rows of the tile that exist
    const int w0 = wt * S::kWarpRows;

    if (w0 < left && wm * kHeads < unit_heads) {            // uniform in the warp
      // ---- scores of kWarpRows rows x kHeads heads; one block alone is added up in two halves, so that the products
      // do not wait for one another
      constexpr int kSets = kBlocks * NT == 1 ? 2 : 1;
      float sc[kBlocks][NT][4];
      float more[4] = {};
#pragma unroll
      for (int blk = 0; blk < kBlocks; blk++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[blk][n][e] = 0.0f;
      if constexpr (!kE4m3) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
          if (s >= steps) break;
          uint32_t b[NT][2];
          if constexpr (kKeepQ) {
#pragma unroll
            for (int n = 0; n < NT; n++) b[n][0] = qf[s][n][0], b[n][1] = qf[s][n][1];
          } else {
            load_q(s, b);
          }
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) {
            uint32_t a[4];    // rows 0-7, 8-15 of values 0-7 of the step, then of values 8-15
            ldsm4(a, k_addr + chunk_at<S::kRowBytes>(w0 + blk * 16 + (lane & 15), s * 2 + (lane >> 4)));
#pragma unroll
            for (int n = 0; n < NT; n++) {
              if (kSets == 2 && (s & 1)) mma16816<kBf16>(more, a, b[n][0], b[n][1]);
              else mma16816<kBf16>(sc[blk][n], a, b[n][0], b[n][1]);
            }
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          if (s >= steps) break;
          uint32_t b[2][NT][2];
#pragma unroll
          for (int u = 0; u < 2; u++) {
            if constexpr (kKeepQ) {
#pragma unroll
              for (int n = 0; n < NT; n++) b[u][n][0] = qf[s + u][n][0], b[u][n][1] = qf[s + u][n][1];
            } else {
              load_q(s + u, b[u]);
            }
          }
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) {
            // a 16-byte chunk is 16 values of a row, one step; a lane gets values 4 (lane & 3) to 4 (lane & 3) + 3
            uint32_t kf[4];   // rows 0-7, 8-15 of step s; the same of step s + 1
            ldsm4(kf, k_addr + chunk_at<S::kRowBytes>(w0 + blk * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), s + (lane >> 4)));
#pragma unroll
            for (int u = 0; u < 2; u++) {
              uint32_t a[4];
              e4m3_to_f16(kf[2 * u], a[0], a[2]);
              e4m3_to_f16(kf[2 * u + 1], a[1], a[3]);
#pragma unroll
              for (int n = 0; n < NT; n++) {
                if (kSets == 2 && u == 1) mma16816<false>(more, a, b[u][n][0], b[u][n][1]);
                else mma16816<false>(sc[blk][n], a, b[u][n][0], b[u][n][1]);
              }
            }
          }
        }
      }
      // ---- base-2 scores, -inf for rows that are not there; running maximum
      uint32_t there[kBlocks];
      bool all_there = true;
#pragma unroll
      for (int blk = 0; blk < kBlocks; blk++) {
        const int r0 = w0 + blk * 16;
        there[blk] = (masks[stage * S::kMaskWords + (r0 >> 5)] >> (r0 & 31)) & 0xffffu;
        all_there = all_there && there[blk] == 0xffffu;
      }
#pragma unroll
      for (int blk = 0; blk < kBlocks; blk++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[blk][n][e] = (kSets == 2 ? sc[blk][n][e] + more[e] : sc[blk][n][e]) * scale[n][e & 1];
      if (!all_there) {                                     // uniform in the warp
#pragma unroll
        for (int blk = 0; blk < kBlocks; blk++)
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (!((there[blk] >> (row + (e >> 1) * 8)) & 1u)) sc[blk][n][e] = kNegInf;
      }
      if (p.scores != nullptr) {
        float* const to = p.scores + ((static_cast<int64_t>(first_tile) + i) * p.chunk + wm * kHeads + col) * S::kTile + w0 + row;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            if (wm * kHeads + n * 8 + col + e >= unit_heads) continue;
#pragma unroll
            for (int blk = 0; blk < kBlocks; blk++) {
              to[(n * 8 + e) * S::kTile + blk * 16] = sc[blk][n][e];
              to[(n * 8 + e) * S::kTile + blk * 16 + 8] = sc[blk][n][e + 2];
            }
          }
      }
      float base[NT][2], fade[NT][2];
      bool moved = false;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float top = m_run[n][e];
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) top = fmaxf(top, fmaxf(sc[blk][n][e], sc[blk][n][e + 2]));
          top = column_max(top);
          base[n][e] = top == kNegInf ? 0.0f : top;
          fade[n][e] = exp2_fast(m_run[n][e] - base[n][e]);
          moved = moved || top != m_run[n][e];
          m_run[n][e] = top;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
          for (int s = 0; s < kSteps; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[s][n][e] *= fade[n][e & 1];
          l_run[n][0] *= fade[n][0];
          l_run[n][1] *= fade[n][1];
        }
      }
      // ---- probabilities and the weighted sum of values
      uint32_t b[kBlocks][NT][2];
#pragma unroll
      for (int blk = 0; blk < kBlocks; blk++)
#pragma unroll
        for (int n = 0; n < NT; n++) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            pr[e] = exp2_fast(sc[blk][n][e] - base[n][e & 1]);
            l_run[n][e & 1] += pr[e];
          }
          b[blk][n][0] = transposed(pack2<kBf16>(pr[0], pr[1]));
          b[blk][n][1] = transposed(pack2<kBf16>(pr[2], pr[3]));
        }
      if constexpr (!kE4m3) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
          if (s >= steps) break;
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) {
            uint32_t a[4];    // transposed: values 0-7, 8-15 of rows 0-7, then of rows 8-15
            ldsm4_t(a, v_addr + chunk_at<S::kRowBytes>(w0 + blk * 16 + (lane & 7) + ((lane >> 4) << 3), s * 2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int n = 0; n < NT; n++) mma16816<kBf16>(acc[s][n], a, b[blk][n][0], b[blk][n][1]);
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          if (s >= steps) break;
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) {
            // transposed 16-bit units: a lane gets values 2u, 2u + 1 (u = lane / 4) of two rows, byte by byte; even
            // values become rows 0-7 of the product, odd ones rows 8-15
            uint32_t vf[4];
            ldsm4_t(vf, v_addr + chunk_at<S::kRowBytes>(w0 + blk * 16 + (lane & 15), s + (lane >> 4)));
#pragma unroll
            for (int u = 0; u < 2; u++) {
              uint32_t a[4];
              e4m3_to_f16(__byte_perm(vf[2 * u], 0, 0x3120), a[0], a[1]);
              e4m3_to_f16(__byte_perm(vf[2 * u + 1], 0, 0x3120), a[2], a[3]);
#pragma unroll
              for (int n = 0; n < NT; n++) mma16816<false>(acc[s + u][n], a, b[blk][n][0], b[blk][n][1]);
            }
          }
        }
      }
    }

    // ---- end of the unit, or of this CTA's part of it: join the warps that shared its rows
    const bool to_end = at.j + 1 == at.tiles;
    if (to_end || i + 1 == n_tiles) {
      const bool whole = from_start && to_end;
      const float v_scale = kE4m3 && p.cache.value_scale != nullptr ? __ldg(p.cache.value_scale + head) : 1.0f;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float l = column_sum(l_run[n][e]);
          if (row == 0) ml[warp * kHeads + n * 8 + col + e] = make_float2(m_run[n][e], l);
        }
      compute_sync();                                       // every warp is done with this stage's tile
      float* const sums = reinterpret_cast<float*>(smem + stage * 2 * S::kTileBytes);   // [warps][8][DP]
      const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + part_slot(first_tile, first_tile + i - at.j)) * S::kUnitRows;
      const int64_t unit_at = (static_cast<int64_t>(at.b) * units + head * p.chunks + at.chunk) * S::kUnitRows;
#pragma unroll
      for (int n = 0; n < NT; n++) {
        if (n * 8 >= unit_heads) break;                     // (for every warp: heads of wm 0 come first)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float m = kNegInf;
#pragma unroll
          for (int x = 0; x < S::kWT; x++) m = fmaxf(m, ml[(x * WM + wm) * kHeads + n * 8 + col + e].x);
          const float f = exp2_fast(m_run[n][e] - (m == kNegInf ? 0.0f : m));
          // value v of head h at v ^ 8 (h / 2 mod 4): the lanes of a store fall into different banks
          float* const to = sums + (warp * 8 + col + e) * DP;
#pragma unroll
          for (int s = 0; s < kSteps; s++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
              const int v = s * 16 + (kE4m3 ? row * 2 + x : row + x * 8);
              to[v ^ ((col >> 1) << 3)] = acc[s][n][2 * x + e] * f;
            }
        }
        compute_sync();
        // warp w puts out heads w, w + 4, ..
        for (int rr = warp; rr < WM * 8; rr += kComputeWarps) {
          const int w = rr >> 3, h8 = rr & 7;
          const int hr = w * kHeads + n * 8 + h8;           // query head inside the unit
          if (hr >= unit_heads) continue;
          float m = kNegInf, l = 0.0f;
#pragma unroll
          for (int x = 0; x < S::kWT; x++) m = fmaxf(m, ml[(x * WM + w) * kHeads + n * 8 + h8].x);
          const float from = m == kNegInf ? 0.0f : m;
#pragma unroll
          for (int x = 0; x < S::kWT; x++) {
            const float2 o = ml[(x * WM + w) * kHeads + n * 8 + h8];
            l += o.y * exp2_fast(o.x - from);
          }
          const int q_head = head * p.group + unit_first + hr;
          const float inv = l == 0.0f ? 0.0f : v_scale / l;
#pragma unroll
          for (int y = 0; y < DP / 32; y++) {
            const int d = y * 32 + lane;
            if (d >= width) break;
            float v = 0.0f;
#pragma unroll
            for (int x = 0; x < S::kWT; x++) v += sums[((x * WM + w) * 8 + h8) * DP + (d ^ ((h8 >> 1) << 3))];
            if (whole) store16(p.out + at.b * p.out_seq + q_head * p.out_head + d * 2, v * inv, p.q_bf16);
            else p.part_acc[(part + hr) * width + d] = v;
          }
          if (lane == 0) {
            if (whole) {
              const float lse2 = l == 0.0f ? kNegInf : m + log2f(l);
              if (p.scores != nullptr) p.unit_lse[unit_at + hr] = lse2;
              if (p.lse != nullptr) p.lse[static_cast<int64_t>(at.b) * p.q_heads + q_head] = lse2 * 0.69314718055994530942f;
            } else {
              p.part_ml[part + hr] = make_float2(m, l);
            }
          }
        }
        compute_sync();
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + stage);
    if (++stage == S::kStages) {
      stage = 0;
      phase ^= 1;
    }
    at.advance(p.table, p.cache.heads, p.chunks, S::kTile);
  }
}

template <typename ST, int DP, int WM, int NT>
struct Launcher {
  static void prepare() {
    static std::atomic<uint64_t> done{0};                   // one bit per device
    int dev = 0;
    NVE_B200_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = uint64_t{1} << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return;
    NVE_B200_CUDA(cudaFuncSetAttribute(attend_kernel<ST, DP, WM, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Shape<ST, DP, WM, NT>::kSmem));
    done.fetch_or(bit, std::memory_order_acq_rel);
  }
  static int resident() {
    static std::atomic<int> cached[64];
    int dev = 0;
    NVE_B200_CUDA(cudaGetDevice(&dev));
    int n = cached[dev & 63].load(std::memory_order_acquire);
    if (n > 0) return n;
    prepare();
    int per_sm = 0;
    NVE_B200_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attend_kernel<ST, DP, WM, NT>, kThreads,
                                                               Shape<ST, DP, WM, NT>::kSmem));
    n = std::max(1, per_sm) * sm_count();
    cached[dev & 63].store(n, std::memory_order_release);
    return n;
  }
  static void launch(const KvAttendParams& p, cudaStream_t stream) {
    prepare();
    launch_overlapped(attend_kernel<ST, DP, WM, NT>, p.ctas, kThreads, Shape<ST, DP, WM, NT>::kSmem, 1, stream, p);
  }
};

// fn(Launcher{}) for the variant of this width and number of padded query rows
template <typename ST, int DP, typename Fn>
auto with_rows(int rows_per_unit, Fn&& fn) {
  if (rows_per_unit == 8) return fn(Launcher<ST, DP, 1, 1>{});
  if (rows_per_unit == 16) return fn(Launcher<ST, DP, 1, 2>{});
  if (rows_per_unit == 32) return fn(Launcher<ST, DP, 2, 2>{});
  return fn(Launcher<ST, DP, 4, 2>{});
}
template <typename ST, typename Fn>
auto with_variant(int width, int rows_per_unit, Fn&& fn) {
  switch (kv_padded_width(width)) {
    case 64: return with_rows<ST, 64>(rows_per_unit, fn);
    case 128: return with_rows<ST, 128>(rows_per_unit, fn);
    default: return with_rows<ST, 256>(rows_per_unit, fn);
  }
}

}  // namespace kv

template <typename ST>
int KvAttendVariant<ST>::resident(int width, int rows_per_unit) {
  return kv::with_variant<ST>(width, rows_per_unit, [](auto v) { return decltype(v)::resident(); });
}
template <typename ST>
void KvAttendVariant<ST>::launch(const KvAttendParams& p, cudaStream_t stream) {
  kv::with_variant<ST>(p.cache.width, p.rows_per_unit, [&](auto v) { decltype(v)::launch(p, stream); });
}

}  // namespace nve_b200
