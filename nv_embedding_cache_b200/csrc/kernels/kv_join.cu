// Second launch of the attention over the paged cache: joins the units that several CTAs shared, and turns the scores
// into the weight every row drew.
//
// Join: out = sum_c 2^(m_c - M) acc_c / sum_c 2^(m_c - M) l_c over the CTAs c that had a part of the unit, M the
// largest m_c; always in ascending c, so the result is the same on every run.  One block per (sequence, query head).
// Weights: row j of key head h grows by sum_g 2^(x_gj - lse_g).  One warp per run of tiles, two rows a lane; the scores
// were written by the first launch moments ago and mostly come from L2 (4 bytes per query head and row, against
// 2 width values of the cache: 6 % of its bytes for eight heads on bf16 rows of 128).
#include <algorithm>

#include "../common.hpp"
#include "kv_attend.hpp"

namespace nve_b200 {

namespace {

constexpr int kThreads = 128;
constexpr float kNegInf = -__builtin_huge_valf();

struct Parts {
  int32_t first, last;               // CTAs that had a part of the unit
};
__device__ __forceinline__ Parts parts_of(int64_t total, int32_t n, int32_t first_tile, int32_t tiles) {
  return {cta_of_tile(total, n, first_tile), cta_of_tile(total, n, first_tile + tiles - 1)};
}
// Scratch row of the unit's part in CTA c: a CTA's first part is slot 0.
__device__ __forceinline__ int64_t part_row(const KvAttendParams& p, int64_t total, int32_t n, int32_t c, int32_t first_tile) {
  const int slot = part_slot(tile_range(total, n, c).first, first_tile);
  return (static_cast<int64_t>(c) * 2 + slot) * p.rows_per_unit;
}

// Base-2 lse of query head `hr` of a unit.
__device__ __forceinline__ float unit_lse2(const KvAttendParams& p, int64_t total, int32_t n, int32_t first_tile,
                                           int32_t tiles, int64_t unit_row, int32_t hr) {
  const Parts parts = parts_of(total, n, first_tile, tiles);
  if (parts.first == parts.last) return p.unit_lse[unit_row + hr];
  float m = kNegInf, l = 0.0f;
  for (int32_t c = parts.first; c <= parts.last; c++) {
    const float2 o = p.part_ml[part_row(p, total, n, c, first_tile) + hr];
    const float top = fmaxf(m, o.x);
    const float base = top == kNegInf ? 0.0f : top;
    l = l * exp2f(m - base) + o.y * exp2f(o.x - base);
    m = top;
  }
  return l == 0.0f ? kNegInf : m + log2f(l);
}

__global__ void __launch_bounds__(kThreads) join_kernel(const KvAttendParams p, int32_t join_blocks, int32_t weight_blocks) {
  __shared__ int64_t s_sum[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units = p.cache.heads * p.chunks;
  const int me_x = static_cast<int>(blockIdx.x);
  const int my_b = me_x < join_blocks ? me_x / p.q_heads : -1;

  // tiles of all sequences, and of those before this block's
  int64_t all = 0, before = 0;
  for (int b = tid; b < p.table.sequences; b += kThreads) {
    const int nt = tiles_of(kv_length(p.table, b, nullptr));
    all += nt;
    if (b < my_b) before += nt;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) s_sum[warp] = all;
  __syncthreads();
  const int64_t sum_tiles = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  __syncthreads();
  if (lane == 0) s_sum[warp] = before;
  __syncthreads();
  const int64_t before_tiles = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  const int64_t total = sum_tiles * units;
  if (total == 0) return;
  const int32_t n = static_cast<int32_t>(min(static_cast<int64_t>(p.ctas), total));

  if (my_b >= 0) {
    // ---- join of one query head
    const int q_head = me_x - my_b * p.q_heads;
    const int head = q_head / p.group, in_group = q_head - head * p.group;
    const int chunk = in_group / p.chunk, hr = in_group - chunk * p.chunk;
    const int tiles = tiles_of(kv_length(p.table, my_b, nullptr));
    if (tiles == 0) return;
    const int32_t first_tile = static_cast<int32_t>(before_tiles * units) + (head * p.chunks + chunk) * tiles;
    const Parts parts = parts_of(total, n, first_tile, tiles);
    if (parts.first == parts.last) return;                  // done by the CTA that had it alone
    __shared__ float s_max[4], s_l[4], s_acc[4][256];
    // warps take the parts in turn, each with its own maximum
    float m = kNegInf;
    for (int32_t c = parts.first + tid; c <= parts.last; c += kThreads)
      m = fmaxf(m, p.part_ml[part_row(p, total, n, c, first_tile) + hr].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_max[warp] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    const float base = m == kNegInf ? 0.0f : m;
    float acc[8] = {};
    float l = 0.0f;
    const int width = p.cache.width;
    for (int32_t c = parts.first + warp; c <= parts.last; c += 4) {
      const int64_t row = part_row(p, total, n, c, first_tile) + hr;
      const float2 o = p.part_ml[row];
      const float f = exp2f(o.x - base);
      l += o.y * f;
#pragma unroll
      for (int x = 0; x < 8; x++) {
        const int d = x * 32 + lane;
        if (d < width) acc[x] += p.part_acc[row * width + d] * f;
      }
    }
#pragma unroll
    for (int x = 0; x < 8; x++) s_acc[warp][x * 32 + lane] = acc[x];
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    l = s_l[0] + s_l[1] + s_l[2] + s_l[3];
    const float v_scale = p.cache.value_scale != nullptr ? __ldg(p.cache.value_scale + head) : 1.0f;
    const float inv = l == 0.0f ? 0.0f : v_scale / l;
    for (int d = tid; d < width; d += kThreads) {
      const float v = (s_acc[0][d] + s_acc[1][d] + s_acc[2][d] + s_acc[3][d]) * inv;
      uint8_t* const to = p.out + my_b * p.out_seq + q_head * p.out_head + d * 2;
      if (p.q_bf16) *reinterpret_cast<__nv_bfloat16*>(to) = __float2bfloat16_rn(v);
      else *reinterpret_cast<__half*>(to) = __float2half_rn(v);
    }
    if (tid == 0 && p.lse != nullptr) {
      p.lse[static_cast<int64_t>(my_b) * p.q_heads + q_head] = l == 0.0f ? kNegInf : (m + log2f(l)) * 0.69314718055994530942f;
    }
    return;
  }

  // ---- weights: runs of (sequence, key head, tile), one per warp
  const int64_t w_total = sum_tiles * p.cache.heads;
  const int32_t warps = weight_blocks * 4, me = (me_x - join_blocks) * 4 + warp;
  const TileRange range = tile_range(w_total, warps, me);
  if (range.first == range.last) return;
  TileCursor at{0, 0, 0, 0, 0};
  int32_t seq_tile = 0;                                      // tiles of the sequences before at.b
  {
    int64_t seen = 0;
    for (int b = 0; b < p.table.sequences; b += 32) {
      const int mine = b + lane;
      const int nt = mine < p.table.sequences ? tiles_of(kv_length(p.table, mine, nullptr)) : 0;
      int64_t incl = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const int64_t off = range.first - (seen + incl - nt) * p.cache.heads;
      const bool found = off >= 0 && off < static_cast<int64_t>(nt) * p.cache.heads;
      const uint32_t who = __ballot_sync(0xffffffffu, found);
      if (who != 0) {
        const int src = __ffs(who) - 1;
        const int32_t o32 = __shfl_sync(0xffffffffu, static_cast<int32_t>(off), src);
        at.b = b + src;
        at.tiles = __shfl_sync(0xffffffffu, nt, src);
        at.unit = o32 / at.tiles;
        at.j = o32 % at.tiles;
        seq_tile = static_cast<int32_t>(__shfl_sync(0xffffffffu, seen + incl - nt, src));
        break;
      }
      seen += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  at.length = kv_length(p.table, at.b, nullptr);
  float lse[2] = {};                                         // of query heads lane, lane + 32 of the chunk in use
  int lse_b = -1, lse_unit = -1;
  for (int32_t t = range.first; t < range.last; t++) {
    const int row0 = at.j * kKvTile + lane * 2;
    float w[2] = {0.0f, 0.0f};
    for (int chunk = 0; chunk < p.chunks; chunk++) {
      const int unit = at.unit * p.chunks + chunk;
      const int32_t first_tile = seq_tile * units + unit * at.tiles;
      const int heads = min(p.chunk, p.group - chunk * p.chunk);
      if (lse_b != at.b || lse_unit != unit) {
        const int64_t unit_row = (static_cast<int64_t>(at.b) * units + unit) * p.rows_per_unit;
#pragma unroll
        for (int x = 0; x < 2; x++)
          if (lane + 32 * x < heads) lse[x] = unit_lse2(p, total, n, first_tile, at.tiles, unit_row, lane + 32 * x);
        lse_b = at.b;
        lse_unit = unit;
      }
      const float* const s = p.scores + (static_cast<int64_t>(first_tile) + at.j) * p.chunk * kKvTile + lane * 2;
      for (int g = 0; g < heads; g++) {
        const float e = __shfl_sync(0xffffffffu, g < 32 ? lse[0] : lse[1], g & 31);
        if (row0 < at.length && e != kNegInf) {
          const float2 x = *reinterpret_cast<const float2*>(s + g * kKvTile);
          w[0] += exp2f(x.x - e);
          w[1] += exp2f(x.y - e);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
      if (row0 + x < at.length) {
        int32_t slot;
        const int32_t page = kv_locate(p.cache, p.table.pages, p.table.stride, at.b, row0 + x, &slot);
        if (page >= 0) p.cache.weights[kv_weight_index(p.cache, page, at.unit, slot)] += w[x];
      }
    }
    if (at.j + 1 == at.tiles && at.unit + 1 == p.cache.heads) seq_tile += at.tiles;
    at.advance(p.table, p.cache.heads);
  }
}

}  // namespace

void launch_kv_join(const KvAttendParams& p, int sms, cudaStream_t stream) {
  const int32_t join_blocks = p.table.sequences * p.q_heads;
  const int32_t weight_blocks = p.scores != nullptr ? sms * 8 : 0;
  join_kernel<<<join_blocks + weight_blocks, kThreads, 0, stream>>>(p, join_blocks, weight_blocks);
  NVE_B200_CUDA(cudaGetLastError());
}

int kv_attend_resident(nve_data_type_t cache_dtype, int width, int rows_per_unit) {
  switch (cache_dtype) {
    case NVE_DTYPE_BFLOAT16: return KvAttendVariant<__nv_bfloat16>::resident(width, rows_per_unit);
    case NVE_DTYPE_FLOAT16: return KvAttendVariant<__half>::resident(width, rows_per_unit);
    default: return KvAttendVariant<__nv_fp8_e4m3>::resident(width, rows_per_unit);
  }
}

void launch_kv_attend(const KvAttendParams& p, nve_data_type_t cache_dtype, cudaStream_t stream) {
  switch (cache_dtype) {
    case NVE_DTYPE_BFLOAT16: KvAttendVariant<__nv_bfloat16>::launch(p, stream); break;
    case NVE_DTYPE_FLOAT16: KvAttendVariant<__half>::launch(p, stream); break;
    default: KvAttendVariant<__nv_fp8_e4m3>::launch(p, stream); break;
  }
}

}  // namespace nve_b200
