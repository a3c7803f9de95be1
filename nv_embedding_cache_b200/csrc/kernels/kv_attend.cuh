// Attention of one new token per sequence over the paged cache: the kernel that reads the cache.
//
//   s_j = scale q.k_j,   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = s_j log2(e)
// in one pass over the rows with a running maximum m, its sum and the weighted sum of values (fp32).
//
// What bounds it: 2 width values are read per (row, key head) and 4 width flops done per query head of the group, so
// even 16 query heads on one key head ask for a few per cent of the tensor rate: memory does.  Everything here is
// there to keep loads in flight on every SM, whatever the batch looks like:
//  * the tiles (64 rows of one key head) of the whole batch are one list, cut into equal runs, one per resident CTA
//    (kv_plan.hpp): one long sequence and a ragged batch load all SMs alike.  A unit that falls into several
//    runs leaves (m, sum, weighted sum) per run in scratch and is joined by kv_join.cu.
//  * a CTA's tiles are one stream through a ring of shared-memory stages filled by cp.async (16 bytes each, a
//    page may end anywhere in a tile); the ring runs on across units, the queries of a unit travel with its
//    first tile.
//  * mma.sync m16n8k16, not tcgen05: a tile has as few as one query row, a 128-row tcgen05 tile would be 8 to
//    128 times padding and its accumulator would have to leave TMEM for the running maximum every 64 rows.  Here
//    the scores stay in the registers that the second product takes them from.
// Four warps; with up to 16 query heads each warp takes 16 rows of the tile and its own running maximum, and
// the four are joined when the unit ends; with more, warps take 16 heads each and share the rows.
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

constexpr int kThreads = 128;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
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
// two E4M3 values (bits 0-15) as f16x2; exact
__device__ __forceinline__ uint32_t e4m3_to_f16(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}
__device__ __forceinline__ float to_float(const uint8_t* p, bool bf16) {
  return bf16 ? __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p)) : __half2float(*reinterpret_cast<const __half*>(p));
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
  static constexpr int kTileBytes = kKvTile * kRowBytes;  // keys or values of a tile
  static constexpr int kWT = 4 / WM;                      // warps along the rows
  static constexpr int kWarpRows = kKvTile / kWT;         // rows of a tile one warp takes
  static constexpr int kUnitRows = 16 * WM;               // query rows
  static constexpr int kQBytes = kUnitRows * DP * 2;
  // A stage holds a tile and the queries of the unit that may begin with it.  Stages until an SM holds three CTAs of
  // three or more, else two, else one: 100 to 150 KB in flight per SM either way, which is what the memory's latency
  // times its rate asks for (about 45 KB), with room for the CTA that is between two waits.
  static constexpr int kStageBytes = 2 * kTileBytes + kQBytes;
  static constexpr int kStages = 3 * kStageBytes <= 72000 ? (73000 / kStageBytes < 6 ? 73000 / kStageBytes : 6)
                                 : 3 * kStageBytes <= 111000 ? 3
                                 : (222000 / kStageBytes < 5 ? 222000 / kStageBytes : 5);
  static constexpr int kMinCtas = 3 * kStageBytes <= 72000 ? 3 : (3 * kStageBytes <= 111000 ? 2 : 1);
  static constexpr int kMasks = 8;                        // ring of row masks, longer than the ring of stages
  static constexpr int kOffsBytes = 2 * kKvTile * 16;
  static constexpr int kSmem = kStages * kStageBytes + kOffsBytes + 4 * 16 * 8 + kMasks * 8 + kUnitRows * 4;
  static_assert(kStages >= 2 && kStages < kMasks, "stages");
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
  longlong2* const offs = reinterpret_cast<longlong2*>(qbuf + S::kStages * S::kQBytes);             // [2][kKvTile]
  float2* const ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(offs) + S::kOffsBytes);   // [4][16]
  uint32_t* const masks = reinterpret_cast<uint32_t*>(ml + 4 * 16);                                 // [kMasks][2]
  float* const q_up = reinterpret_cast<float*>(masks + S::kMasks * 2);                              // [kUnitRows]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp % WM, wt = warp / WM;                // heads 16 wm.., rows kWarpRows wt.. of the tile
  const int width = p.cache.width;
  const int row_chunks = width * static_cast<int>(sizeof(ST)) / 16;
  const int q_chunks = width / 8;
  const int units = p.cache.heads * p.chunks;

  // ---- the number of tiles, and where this CTA's run of them begins
  __shared__ int64_t s_sum[4];
  __shared__ int32_t s_start[3];
  {
    int64_t mine = 0;
    for (int b = tid; b < p.table.sequences; b += kThreads) mine += tiles_of(kv_length(p.table, b, p.cache.status));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
  }
  const int64_t total = (s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]) * units;
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
      const int nt = b < p.table.sequences ? tiles_of(kv_length(p.table, b, nullptr)) : 0;
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
  TileCursor take;                                          // the tile whose rows are located next
  take.b = s_start[0];
  take.unit = s_start[1];
  take.j = s_start[2];
  take.length = kv_length(p.table, take.b, nullptr);
  take.tiles = tiles_of(take.length);
  TileCursor issue = take, use = take;                      // the tile whose copies are issued next; the tile in use

  // Offsets of the row of the `take` tile this thread (tid < kKvTile) looks after; negative: no such row.
  auto locate = [&]() -> longlong2 {
    const int32_t row = take.j * kKvTile + tid;
    longlong2 o = make_longlong2(-1, -1);
    if (row < take.length) {
      int32_t slot;
      const int32_t page = kv_locate(p.cache, p.table.pages, p.table.stride, take.b, row, &slot);
      const int32_t head = take.unit / p.chunks;
      if (page >= 0) {
        o.x = page * p.cache.k_page + slot * p.cache.k_slot + head * p.cache.k_head;
        o.y = page * p.cache.v_page + slot * p.cache.v_slot + head * p.cache.v_head;
      }
    }
    return o;
  };
  auto keep_located = [&](int i, longlong2 o) {             // warps 0 and 1, tile number i of this CTA
    offs[(i & 1) * kKvTile + tid] = o;
    const uint32_t mask = __ballot_sync(0xffffffffu, o.x >= 0);
    if (lane == 0) masks[(i % S::kMasks) * 2 + warp] = mask;
  };
  int q_issue = 0, q_use = 0;                               // buffers of the units the two cursors are in
  auto issue_tile = [&](int i) {                            // copies of tile number i into its stage
    const uint32_t k_addr = smem_addr(smem) + (i % S::kStages) * 2 * S::kTileBytes, v_addr = k_addr + S::kTileBytes;
    const longlong2* const o = offs + (i & 1) * kKvTile;
#pragma unroll
    for (int x = 0; x < kKvTile * S::kChunks / kThreads; x++) {
      const int id = x * kThreads + tid;
      const int r = id / S::kChunks, c = id % S::kChunks;
      const longlong2 at = o[r];
      // chunks behind the row's width and rows that are not there become zeros: a NaN left in a page never meets
      // the products
      const bool ok = at.x >= 0 && c < row_chunks;
      const uint32_t to = chunk_at<S::kRowBytes>(r, c);
      cp_async16(k_addr + to, ok ? p.cache.keys + at.x + c * 16 : p.cache.keys, ok);
      cp_async16(v_addr + to, ok ? p.cache.values + at.y + c * 16 : p.cache.values, ok);
    }
    if (i == 0 || issue.j == 0) {                           // the unit's queries
      if (i > 0) q_issue = q_issue + 1 == S::kStages ? 0 : q_issue + 1;
      const uint32_t q_addr = smem_addr(qbuf) + q_issue * S::kQBytes;
      const int head = issue.unit / p.chunks, first = (issue.unit % p.chunks) * p.chunk;
      const int n = min(p.chunk, p.group - first);
      const uint8_t* const src = p.q + issue.b * p.q_seq + (head * p.group + first) * p.q_head;
      for (int id = tid; id < S::kUnitRows * (DP / 8); id += kThreads) {
        const int r = id / (DP / 8), c = id % (DP / 8);
        const bool ok = r < n && c < q_chunks;
        cp_async16(q_addr + chunk_at<DP * 2>(r, c), ok ? src + r * p.q_head + c * 16 : p.q, ok);
      }
    }
    issue.advance(p.table, units);
  };

  // ---- fill the ring; rows are located one tile ahead of their copies
  if (tid < kKvTile) keep_located(0, locate());
  take.advance(p.table, units);
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; i++) {
    __syncthreads();
    if (i < n_tiles) issue_tile(i);
    cp_commit();
    if (i + 1 < n_tiles) {
      if (tid < kKvTile) keep_located(i + 1, locate());
      take.advance(p.table, units);
    }
  }

  float acc[kSteps][2][4];
  float m_run[2], l_run[2];
  uint32_t qf[kKeepQ ? kSteps : 1][4];
  float row_scale[2];
  bool from_start = false;                                  // this CTA has the current unit from its first tile

#pragma unroll 1
  for (int i = 0; i < n_tiles; i++) {
    cp_wait<S::kStages - 2>();
    __syncthreads();
    const int ahead = i + S::kStages - 1;
    if (ahead < n_tiles) issue_tile(ahead);
    cp_commit();
    const bool locates = ahead + 1 < n_tiles;
    longlong2 next = make_longlong2(-1, -1);
    if (locates) {
      if (tid < kKvTile) next = locate();
      take.advance(p.table, units);
    }

    const int head = use.unit / p.chunks;
    const int unit_first = (use.unit % p.chunks) * p.chunk; // first query head of the unit inside its group
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
    if (i == 0 || use.j == 0) {
      if (i > 0) q_use = q_use + 1 == S::kStages ? 0 : q_use + 1;
      from_start = use.j == 0;
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
          for (int r = warp; r < S::kUnitRows; r += 4) {
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
          __syncthreads();
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

    const uint32_t k_addr = smem_addr(smem) + (i % S::kStages) * 2 * S::kTileBytes, v_addr = k_addr + S::kTileBytes;
    const int left = use.length - use.j * kKvTile;          // rows of the tile that exist

#pragma unroll
    for (int blk = 0; blk < kBlocks; blk++) {
      const int r0 = wt * S::kWarpRows + blk * 16;
      if (r0 >= left || !lower) break;                      // uniform in the warp
      // ---- scores of 16 heads x 16 rows
      float sc[2][4] = {};
      if constexpr (!kE4m3) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
          uint32_t kf[4];   // rows 0-7: columns 0-7, 8-15 of the step; rows 8-15: the same
          ldsm4(kf, k_addr + chunk_at<S::kRowBytes>(r0 + (lane & 7) + ((lane >> 4) << 3), s * 2 + ((lane >> 3) & 1)));
          uint32_t a[4];
          if constexpr (kKeepQ) {
#pragma unroll
            for (int e = 0; e < 4; e++) a[e] = qf[s][e];
          } else {
            load_q(s, a);
          }
          mma16816<kBf16>(sc[0], a, kf[0], kf[1]);
          mma16816<kBf16>(sc[1], a, kf[2], kf[3]);
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          // a 16-byte chunk is 16 values of a row, one step; a lane gets values 4 (lane & 3) to 4 (lane & 3) + 3
          uint32_t kf[4];   // rows 0-7, 8-15 of step s; the same of step s + 1
          ldsm4(kf, k_addr + chunk_at<S::kRowBytes>(r0 + (lane & 7) + (((lane >> 3) & 1) << 3), s + (lane >> 4)));
#pragma unroll
          for (int u = 0; u < 2; u++) {
            uint32_t a[4];
            if constexpr (kKeepQ) {
#pragma unroll
              for (int e = 0; e < 4; e++) a[e] = qf[s + u][e];
            } else {
              load_q(s + u, a);
            }
            mma16816<false>(sc[0], a, e4m3_to_f16(kf[2 * u]), e4m3_to_f16(kf[2 * u] >> 16));
            mma16816<false>(sc[1], a, e4m3_to_f16(kf[2 * u + 1]), e4m3_to_f16(kf[2 * u + 1] >> 16));
          }
        }
      }
      // ---- base-2 scores, -inf for rows that are not there; running maximum
      const uint32_t mask = masks[(i % S::kMasks) * 2 + (r0 >> 5)] >> (r0 & 31);
      float top[2] = {m_run[0], m_run[1]};
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int r = n * 8 + (lane & 3) * 2 + (e & 1);
          sc[n][e] = (mask >> r) & 1u ? sc[n][e] * row_scale[e >> 1] : kNegInf;
          top[e >> 1] = fmaxf(top[e >> 1], sc[n][e]);
        }
      if (p.scores != nullptr) {
        float* const to = p.scores + ((static_cast<int64_t>(range.first) + i) * p.chunk + wm * 16 + (lane >> 2)) * kKvTile + r0 + (lane & 3) * 2;
#pragma unroll
        for (int half = 0; half < 2; half++) {
          if (wm * 16 + half * 8 + (lane >> 2) >= unit_heads) continue;
#pragma unroll
          for (int n = 0; n < 2; n++)
            *reinterpret_cast<float2*>(to + half * 8 * kKvTile + n * 8) = make_float2(sc[n][2 * half], sc[n][2 * half + 1]);
        }
      }
      float base[2], fade[2];
#pragma unroll
      for (int half = 0; half < 2; half++) {
        if (half == 1 && !upper) {
          base[1] = 0.0f;
          fade[1] = 1.0f;
          continue;
        }
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
      float pr[2][4] = {};
#pragma unroll
      for (int half = 0; half < 2; half++) {
        if (half == 1 && !upper) continue;
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            pr[n][2 * half + e] = exp2_fast(sc[n][2 * half + e] - base[half]);
            l_run[half] += pr[n][2 * half + e];
          }
      }
      // ---- weighted sum of values
      uint32_t a[4];
#pragma unroll
      for (int n = 0; n < 2; n++) {
        a[2 * n] = pack2<kBf16>(pr[n][0], pr[n][1]);
        a[2 * n + 1] = pack2<kBf16>(pr[n][2], pr[n][3]);
      }
      if constexpr (!kE4m3) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
          uint32_t vf[4];   // rows 0-7, 8-15 of columns 0-7, then of columns 8-15
          ldsm4_t(vf, v_addr + chunk_at<S::kRowBytes>(r0 + (lane & 15), s * 2 + (lane >> 4)));
          mma16816<kBf16>(acc[s][0], a, vf[0], vf[1]);
          mma16816<kBf16>(acc[s][1], a, vf[2], vf[3]);
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          // transposed 16-bit units: a lane gets columns 2u, 2u + 1 (u = lane / 4) of two rows, byte by byte; the bytes
          // are dealt out to the products of the even and of the odd columns
          uint32_t vf[4];
          ldsm4_t(vf, v_addr + chunk_at<S::kRowBytes>(r0 + (lane & 15), s + (lane >> 4)));
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const uint32_t x = __byte_perm(vf[2 * u], 0, 0x3120), y = __byte_perm(vf[2 * u + 1], 0, 0x3120);
            mma16816<false>(acc[s + u][0], a, e4m3_to_f16(x), e4m3_to_f16(y));
            mma16816<false>(acc[s + u][1], a, e4m3_to_f16(x >> 16), e4m3_to_f16(y >> 16));
          }
        }
      }
    }
    if (locates && tid < kKvTile) keep_located(ahead + 1, next);

    // ---- end of the unit, or of this CTA's part of it: join the warps that shared its rows
    const bool to_end = use.j + 1 == use.tiles;
    if (to_end || i + 1 == n_tiles) {
      const bool whole = from_start && to_end;
      const float v_scale = kE4m3 && p.cache.value_scale != nullptr ? __ldg(p.cache.value_scale + head) : 1.0f;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const float l = quad_sum(l_run[half]);
        if ((lane & 3) == 0) ml[warp * 16 + half * 8 + (lane >> 2)] = make_float2(m_run[half], l);
      }
      __syncthreads();
      float* const sums = reinterpret_cast<float*>(smem + (i % S::kStages) * 2 * S::kTileBytes);   // [4][8][DP]
      const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + part_slot(range.first, range.first + i - use.j)) * S::kUnitRows;
      const int64_t unit_at = (static_cast<int64_t>(use.b) * units + use.unit) * S::kUnitRows;
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
        __syncthreads();
        for (int rr = 0; rr < WM * 8; rr++) {
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
          for (int d = tid; d < width; d += kThreads) {
            float v = 0.0f;
#pragma unroll
            for (int x = 0; x < S::kWT; x++) v += sums[((x * WM + w) * 8 + row) * DP + (d ^ ((row & 3) << 3))];
            if (whole) store16(p.out + use.b * p.out_seq + q_head * p.out_head + d * 2, v * inv, p.q_bf16);
            else p.part_acc[(part + hr) * width + d] = v;
          }
          if (tid == 0) {
            if (whole) {
              const float lse2 = l == 0.0f ? kNegInf : m + log2f(l);
              if (p.scores != nullptr) p.unit_lse[unit_at + hr] = lse2;
              if (p.lse != nullptr) p.lse[static_cast<int64_t>(use.b) * p.q_heads + q_head] = lse2 * 0.69314718055994530942f;
            } else {
              p.part_ml[part + hr] = make_float2(m, l);
            }
          }
        }
        __syncthreads();
      }
    }
    use.advance(p.table, units);
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
