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
//  * mma.sync m16n8k16, not tcgen05: a tile has as few as one query row, a 128-row tcgen05 tile would be 8 to
//    128 times padding and its accumulator would have to leave TMEM for the running maximum every 64 rows.  Here
//    the scores stay in the registers that the second product takes them from.
// With up to 16 query heads each of the four warps takes a quarter of the tile's rows and has its own running maximum,
// and the four are joined when the unit ends; with more, warps take 16 heads each and share the rows.
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

namespace nve_b200 {

namespace kv {

constexpr int kComputeWarps = 4;
constexpr int kLoadWarps = 2;
constexpr int kThreads = (kComputeWarps + kLoadWarps) * 32;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16_full(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

// ST: stored type.  DP: width rounded up to 64, 128 or 256.  WM: warps along the query heads.
template <typename ST, int DP, int WM>
struct Shape {
  static constexpr bool kE4m3 = sizeof(ST) == 1;
  static constexpr int kRowBytes = DP * sizeof(ST);
  static constexpr int kChunks = kRowBytes / 16;          // 16-byte chunks of a row
  static constexpr int kTile = kv_tile_rows(DP, sizeof(ST));
  static constexpr int kTileBytes = kTile * kRowBytes;    // keys or values of a tile
  static constexpr int kWT = kComputeWarps / WM;          // warps along the rows
  static constexpr int kWarpRows = kTile / kWT;           // rows of a tile one warp takes
  static constexpr int kUnitRows = 16 * WM;               // query rows
  static constexpr int kQBytes = kUnitRows * DP * 2;
  // A stage holds a tile and the queries of the unit that may begin with it.  Two CTAs per SM of three or more stages
  // where they fit, else one: 130 KB and more in flight per SM; the memory's latency times its rate asks for 45 KB.
  static constexpr int kStageBytes = 2 * kTileBytes + kQBytes;
  static constexpr int kMinCtas = 3 * kStageBytes <= 111000 ? 2 : 1;
  static constexpr int kStages = kMinCtas == 2 ? (111000 / kStageBytes < 5 ? 111000 / kStageBytes : 5)
                                               : (222000 / kStageBytes < 5 ? 222000 / kStageBytes : 5);
  static constexpr int kMaskWords = kTile / 32;
  static constexpr int kOffsBytes = kTile * 16;
  static constexpr int kSmem = kStages * kStageBytes + kOffsBytes + kComputeWarps * 16 * 8 + kStages * kMaskWords * 4 +
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

template <typename ST, int DP, int WM>
__global__ void __launch_bounds__(kThreads, Shape<ST, DP, WM>::kMinCtas) attend_kernel(const KvAttendParams p) {
  using S = Shape<ST, DP, WM>;
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
  float2* const ml = reinterpret_cast<float2*>(empty + S::kStages);                                 // [warps][16]
  uint32_t* const masks = reinterpret_cast<uint32_t*>(ml + kComputeWarps * 16);                     // [kStages][kMaskWords]
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
  // ---- the number of tiles, and where this CTA's run of them begins
  __shared__ int64_t s_sum[kThreads / 32];
  __shared__ int32_t s_start[3];
  {
    int64_t mine = 0;
    for (int b = tid; b < p.table.sequences; b += kThreads) mine += tiles_of(kv_length(p.table, b, p.cache.status), S::kTile);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
  }
  int64_t total = 0;
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
  const int32_t n_ctas = static_cast<int32_t>(min(static_cast<int64_t>(gridDim.x), total));
  if (static_cast<int32_t>(blockIdx.x) >= n_ctas) return;
  const TileRange range = tile_range(total, n_ctas, blockIdx.x);
  const int n_tiles = range.last - range.first;

  if (warp == 0) {                                          // 32 sequences a step
    int64_t before = 0;
    for (int base = 0; base < p.table.sequences; base += 32) {
      const int b = base + lane;
      const int nt = b < p.table.sequences ? tiles_of(kv_length(p.table, b, nullptr), S::kTile) : 0;
      const int64_t here = static_cast<int64_t>(nt) * units;
      int64_t incl = here;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const int64_t at = range.first - (before + incl - here);
      const bool found = at >= 0 && at < here;
      if (found) {
        s_start[0] = b;
        s_start[1] = static_cast<int32_t>(at) / nt;
        s_start[2] = static_cast<int32_t>(at) % nt;
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

  // the join may be scheduled from here on; it waits for this grid's end before it reads what is written here
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp >= kComputeWarps) {
    // ================================ loading warps ================================
    constexpr int kOwnRows = S::kTile / kLoadWarps;         // rows of a tile this warp looks after
    constexpr int kEach = kOwnRows / 32;
    const int lw = warp - kComputeWarps;
    const int row_chunks = width * static_cast<int>(sizeof(ST)) / 16, q_chunks = width / 8;
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
            cp_async16_full(dst, reinterpret_cast<const uint8_t*>(o.x) + c_lane * 16);
            cp_async16_full(dst + S::kTileBytes, reinterpret_cast<const uint8_t*>(o.y) + c_lane * 16);
          }
        }
      } else {
#pragma unroll 2
        for (int x = 0; x < kCopies; x++) {
          const int r = x * kRowsStep + r_lane;
          const longlong2 o = own[r];
          // chunks behind the row's width and rows that are not there become zeros: a NaN left in a page never meets
          // the products
          const bool ok = o.x != 0 && c_lane < row_chunks;
          const uint32_t dst = k_addr + chunk_at<S::kRowBytes>(r, c_lane);
          cp_async16(dst, ok ? reinterpret_cast<const uint8_t*>(o.x) + c_lane * 16 : p.cache.keys, ok);
          cp_async16(dst + S::kTileBytes, ok ? reinterpret_cast<const uint8_t*>(o.y) + c_lane * 16 : p.cache.values, ok);
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
          cp_async16(q_addr + chunk_at<DP * 2>(r, c), ok ? src + r * p.q_head + c * 16 : p.q, ok);
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
  const int wm = warp % WM, wt = warp / WM;                 // heads 16 wm.., rows kWarpRows wt.. of the tile
  float acc[kSteps][2][4];
  float m_run[2], l_run[2];
  uint32_t qf[kKeepQ ? kSteps : 1][4];
  float row_scale[2];
  bool from_start = false;                                  // this CTA has the current unit from its first tile
  int q_use = 0;

#pragma unroll 1
  for (int i = 0; i < n_tiles; i++) {
    if (!mbar_wait_bounded(full + stage, phase)) {          // all four warps wait for the same event: all give up
      kv_flag(p.cache.status, NVE_B200_KV_TIMED_OUT);
      return;
    }
    const int head = at.head;
    const int unit_first = at.chunk * p.chunk;              // first query head of the unit inside its group
    const int unit_heads = min(p.chunk, p.group - unit_first);
    const bool lower = wm * 16 < unit_heads, upper = wm * 16 + 8 < unit_heads;   // rows 0-7, 8-15 hold heads
    auto load_q = [&](int step, uint32_t (&a)[4]) {
      const uint32_t base = smem_addr(qbuf) + q_use * S::kQBytes;
      if constexpr (!kE4m3) {
        // rows 0-7, 8-15 of columns 0-7 of the step, then of columns 8-15
        ldsm4(a, base + chunk_at<DP * 2>(wm * 16 + (lane & 15), step * 2 + (lane >> 4)));
      } else {
        // a lane gets four consecutive values of an E4M3 row; the columns of q are dealt out alike
        const int c = step * 2 + ((lane & 3) >> 1), in = (lane & 1) * 8;
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const uint32_t addr = base + chunk_at<DP * 2>(wm * 16 + (lane >> 2) + half * 8, c) + in;
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(a[half]), "=r"(a[half + 2]) : "r"(addr) : "memory");
        }
      }
    };
    if (i == 0 || at.j == 0) {
      if (i > 0) q_use = q_use + 1 == S::kStages ? 0 : q_use + 1;
      from_start = at.j == 0;
#pragma unroll
      for (int s = 0; s < kSteps; s++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[s][0][e] = acc[s][1][e] = 0.0f;
      m_run[0] = m_run[1] = kNegInf;
      l_run[0] = l_run[1] = 0.0f;
      row_scale[0] = row_scale[1] = p.scale_log2;
      if constexpr (kE4m3) {
        // Queries meet E4M3 rows as f16.  bf16 ones are brought into its range row by row: divided by the power of
        // two of the row's largest value, which the scores get back; exact but for values 2^-24 below that.
        if (p.q_bf16) {
          for (int r = warp; r < S::kUnitRows; r += kComputeWarps) {
            uint32_t* const row = reinterpret_cast<uint32_t*>(qbuf + q_use * S::kQBytes) + r * (DP / 2);
            float2 v[DP / 64];
            uint32_t top = 0;
#pragma unroll
            for (int x = 0; x < DP / 64; x++) {
              const uint32_t w = row[x * 32 + lane];
              v[x] = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
              const uint32_t ea = (__float_as_uint(v[x].x) >> 23) & 255u, eb = (__float_as_uint(v[x].y) >> 23) & 255u;
              top = max(top, max(ea == 255u ? 0u : ea, eb == 255u ? 0u : eb));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (top == 0) top = 127;
            top = min(top, 253u);
            const float down = __uint_as_float((254u - top) << 23);
#pragma unroll
            for (int x = 0; x < DP / 64; x++) row[x * 32 + lane] = pack2<false>(v[x].x * down, v[x].y * down);
            if (lane == 0) q_up[r] = __uint_as_float(top << 23);
          }
          compute_sync();
          row_scale[0] *= q_up[wm * 16 + (lane >> 2)];
          row_scale[1] *= q_up[wm * 16 + (lane >> 2) + 8];
        }
        if (p.cache.key_scale != nullptr) {
          const float s = __ldg(p.cache.key_scale + head);
          row_scale[0] *= s;
          row_scale[1] *= s;
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

    if (w0 < left && lower) {                               // uniform in the warp
      // ---- scores of 16 heads x kWarpRows rows; one block alone is added up in two halves, so that the products
      // do not wait for one another
      constexpr int kSets = kBlocks == 1 ? 2 : 1;
      float sc[kBlocks][2][4];
      float more[2][4];
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          more[n][e] = 0.0f;
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) sc[blk][n][e] = 0.0f;
        }
      if constexpr (!kE4m3) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
          uint32_t a[4];
          if constexpr (kKeepQ) {
#pragma unroll
            for (int e = 0; e < 4; e++) a[e] = qf[s][e];
          } else {
            load_q(s, a);
          }
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) {
            uint32_t kf[4];   // rows 0-7: columns 0-7, 8-15 of the step; rows 8-15: the same
            ldsm4(kf, k_addr + chunk_at<S::kRowBytes>(w0 + blk * 16 + (lane & 7) + ((lane >> 4) << 3), s * 2 + ((lane >> 3) & 1)));
            if (kSets == 2 && (s & 1)) {
              mma16816<kBf16>(more[0], a, kf[0], kf[1]);
              mma16816<kBf16>(more[1], a, kf[2], kf[3]);
            } else {
              mma16816<kBf16>(sc[blk][0], a, kf[0], kf[1]);
              mma16816<kBf16>(sc[blk][1], a, kf[2], kf[3]);
            }
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          uint32_t a[2][4];
#pragma unroll
          for (int u = 0; u < 2; u++) {
            if constexpr (kKeepQ) {
#pragma unroll
              for (int e = 0; e < 4; e++) a[u][e] = qf[s + u][e];
            } else {
              load_q(s + u, a[u]);
            }
          }
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) {
            // a 16-byte chunk is 16 values of a row, one step; a lane gets values 4 (lane & 3) to 4 (lane & 3) + 3
            uint32_t kf[4];   // rows 0-7, 8-15 of step s; the same of step s + 1
            ldsm4(kf, k_addr + chunk_at<S::kRowBytes>(w0 + blk * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), s + (lane >> 4)));
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
              for (int n = 0; n < 2; n++) {
                uint32_t b0, b1;
                e4m3_to_f16(kf[2 * u + n], b0, b1);
                if (kSets == 2 && u == 1) mma16816<false>(more[n], a[u], b0, b1);
                else mma16816<false>(sc[blk][n], a[u], b0, b1);
              }
          }
        }
      }
      // ---- base-2 scores, -inf for rows that are not there; running maximum
      float top[2] = {m_run[0], m_run[1]};
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
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float x = kSets == 2 ? sc[blk][n][e] + more[n][e] : sc[blk][n][e];
            sc[blk][n][e] = x * row_scale[e >> 1];
          }
      if (!all_there) {                                     // uniform in the warp
#pragma unroll
        for (int blk = 0; blk < kBlocks; blk++)
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (!((there[blk] >> (n * 8 + (lane & 3) * 2 + (e & 1))) & 1u)) sc[blk][n][e] = kNegInf;
      }
#pragma unroll
      for (int blk = 0; blk < kBlocks; blk++)
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) top[e >> 1] = fmaxf(top[e >> 1], sc[blk][n][e]);
      if (p.scores != nullptr) {
        float* const to = p.scores + ((static_cast<int64_t>(range.first) + i) * p.chunk + wm * 16 + (lane >> 2)) * S::kTile + w0 + (lane & 3) * 2;
#pragma unroll
        for (int half = 0; half < 2; half++) {
          if (wm * 16 + half * 8 + (lane >> 2) >= unit_heads) continue;
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++)
#pragma unroll
            for (int n = 0; n < 2; n++)
              *reinterpret_cast<float2*>(to + half * 8 * S::kTile + blk * 16 + n * 8) =
                  make_float2(sc[blk][n][2 * half], sc[blk][n][2 * half + 1]);
        }
      }
      float base[2] = {0.0f, 0.0f}, fade[2] = {1.0f, 1.0f};
#pragma unroll
      for (int half = 0; half < 2; half++) {
        if (half == 1 && !upper) continue;
        top[half] = quad_max(top[half]);
        base[half] = top[half] == kNegInf ? 0.0f : top[half];
        fade[half] = exp2_fast(m_run[half] - base[half]);
      }
      if (__any_sync(0xffffffffu, top[0] != m_run[0] || (upper && top[1] != m_run[1]))) {
#pragma unroll
        for (int s = 0; s < kSteps; s++)
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[s][n][e] *= fade[e >> 1];
        l_run[0] *= fade[0];
        l_run[1] *= fade[1];
        m_run[0] = top[0];
        if (upper) m_run[1] = top[1];
      }
      // ---- probabilities and the weighted sum of values
      uint32_t a[kBlocks][4];
#pragma unroll
      for (int blk = 0; blk < kBlocks; blk++) {
        float pr[2][4] = {};
#pragma unroll
        for (int half = 0; half < 2; half++) {
          if (half == 1 && !upper) continue;
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              pr[n][2 * half + e] = exp2_fast(sc[blk][n][2 * half + e] - base[half]);
              l_run[half] += pr[n][2 * half + e];
            }
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
          a[blk][2 * n] = pack2<kBf16>(pr[n][0], pr[n][1]);
          a[blk][2 * n + 1] = pack2<kBf16>(pr[n][2], pr[n][3]);
        }
      }
      if constexpr (!kE4m3) {
#pragma unroll
        for (int s = 0; s < kSteps; s++)
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) {
            uint32_t vf[4];   // rows 0-7, 8-15 of columns 0-7, then of columns 8-15
            ldsm4_t(vf, v_addr + chunk_at<S::kRowBytes>(w0 + blk * 16 + (lane & 15), s * 2 + (lane >> 4)));
            mma16816<kBf16>(acc[s][0], a[blk], vf[0], vf[1]);
            mma16816<kBf16>(acc[s][1], a[blk], vf[2], vf[3]);
          }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; s += 2)
#pragma unroll
          for (int blk = 0; blk < kBlocks; blk++) {
            // transposed 16-bit units: a lane gets columns 2u, 2u + 1 (u = lane / 4) of two rows, byte by byte; the bytes
            // are dealt out to the products of the even and of the odd columns
            uint32_t vf[4];
            ldsm4_t(vf, v_addr + chunk_at<S::kRowBytes>(w0 + blk * 16 + (lane & 15), s + (lane >> 4)));
#pragma unroll
            for (int u = 0; u < 2; u++) {
              uint32_t even0, even1, odd0, odd1;
              e4m3_to_f16(__byte_perm(vf[2 * u], 0, 0x3120), even0, odd0);
              e4m3_to_f16(__byte_perm(vf[2 * u + 1], 0, 0x3120), even1, odd1);
              mma16816<false>(acc[s + u][0], a[blk], even0, even1);
              mma16816<false>(acc[s + u][1], a[blk], odd0, odd1);
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
      for (int half = 0; half < 2; half++) {
        const float l = quad_sum(l_run[half]);
        if ((lane & 3) == 0) ml[warp * 16 + half * 8 + (lane >> 2)] = make_float2(m_run[half], l);
      }
      compute_sync();                                       // every warp is done with this stage's tile
      float* const sums = reinterpret_cast<float*>(smem + stage * 2 * S::kTileBytes);   // [warps][8][DP]
      const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + part_slot(range.first, range.first + i - at.j)) * S::kUnitRows;
      const int64_t unit_at = (static_cast<int64_t>(at.b) * units + head * p.chunks + at.chunk) * S::kUnitRows;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        if (half * 8 >= unit_heads) break;                  // (for every warp: rows of wm 0 come first)
        {
          const int row = lane >> 2;
          float m = kNegInf;
#pragma unroll
          for (int x = 0; x < S::kWT; x++) m = fmaxf(m, ml[(x * WM + wm) * 16 + half * 8 + row].x);
          const float f = exp2_fast(m_run[half] - (m == kNegInf ? 0.0f : m));
          float* const to = sums + (warp * 8 + row) * DP;
#pragma unroll
          for (int s = 0; s < kSteps; s++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
              float2 v;
              int col;
              if constexpr (!kE4m3) {
                v = make_float2(acc[s][x][2 * half] * f, acc[s][x][2 * half + 1] * f);
                col = s * 16 + x * 8 + (lane & 3) * 2;
              } else {
                v = make_float2(acc[s][0][2 * half + x] * f, acc[s][1][2 * half + x] * f);
                col = s * 16 + (lane & 3) * 4 + x * 2;
              }
              *reinterpret_cast<float2*>(to + (col ^ ((row & 3) << 3))) = v;
            }
          }
        }
        compute_sync();
        // warp w puts out rows w, w + 4, ..
        for (int rr = warp; rr < WM * 8; rr += kComputeWarps) {
          const int w = rr >> 3, row = rr & 7;
          const int hr = w * 16 + half * 8 + row;           // query head inside the unit
          if (hr >= unit_heads) continue;
          float m = kNegInf, l = 0.0f;
#pragma unroll
          for (int x = 0; x < S::kWT; x++) m = fmaxf(m, ml[(x * WM + w) * 16 + half * 8 + row].x);
          const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
          for (int x = 0; x < S::kWT; x++) {
            const float2 o = ml[(x * WM + w) * 16 + half * 8 + row];
            l += o.y * exp2_fast(o.x - base);
          }
          const int q_head = head * p.group + unit_first + hr;
          const float inv = l == 0.0f ? 0.0f : v_scale / l;
#pragma unroll
          for (int y = 0; y < DP / 32; y++) {
            const int d = y * 32 + lane;
            if (d >= width) break;
            float v = 0.0f;
#pragma unroll
            for (int x = 0; x < S::kWT; x++) v += sums[((x * WM + w) * 8 + row) * DP + (d ^ ((row & 3) << 3))];
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

template <typename ST, int DP, int WM>
struct Launcher {
  static void prepare() {
    static std::atomic<uint64_t> done{0};                   // one bit per device
    int dev = 0;
    NVE_B200_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = uint64_t{1} << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return;
    NVE_B200_CUDA(cudaFuncSetAttribute(attend_kernel<ST, DP, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Shape<ST, DP, WM>::kSmem));
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
    NVE_B200_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attend_kernel<ST, DP, WM>, kThreads,
                                                               Shape<ST, DP, WM>::kSmem));
    n = std::max(1, per_sm) * sm_count();
    cached[dev & 63].store(n, std::memory_order_release);
    return n;
  }
  static void launch(const KvAttendParams& p, cudaStream_t stream) {
    prepare();
    attend_kernel<ST, DP, WM><<<p.ctas, kThreads, Shape<ST, DP, WM>::kSmem, stream>>>(p);
    NVE_B200_CUDA(cudaGetLastError());
  }
};

// fn(Launcher<ST, DP, WM>{}) for the variant of this width and number of padded query rows
template <typename ST, typename Fn>
auto with_variant(int width, int rows_per_unit, Fn&& fn) {
  if (width <= 64) {
    if (rows_per_unit == 16) return fn(Launcher<ST, 64, 1>{});
    if (rows_per_unit == 32) return fn(Launcher<ST, 64, 2>{});
    return fn(Launcher<ST, 64, 4>{});
  }
  if (width <= 128) {
    if (rows_per_unit == 16) return fn(Launcher<ST, 128, 1>{});
    if (rows_per_unit == 32) return fn(Launcher<ST, 128, 2>{});
    return fn(Launcher<ST, 128, 4>{});
  }
  if (rows_per_unit == 16) return fn(Launcher<ST, 256, 1>{});
  if (rows_per_unit == 32) return fn(Launcher<ST, 256, 2>{});
  return fn(Launcher<ST, 256, 4>{});
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
