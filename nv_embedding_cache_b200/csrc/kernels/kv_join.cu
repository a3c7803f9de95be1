// Second launch of the attention over the paged cache: joins the units that several CTAs shared, and turns the scores
// into the weight every row drew.
//
// Join: out = sum_c 2^(m_c - M) acc_c / sum_c 2^(m_c - M) l_c over the CTAs c that had a part of the unit, M the
// largest m_c; added up in a fixed order, so the result is the same on every run.  A block takes 1, 2, 4 or 8 query
// heads of a unit, 8, 4, 2 or 1 warps each: one head where units are few and their parts many, eight where it is the
// other way round.
// Weights: row j of key head h grows by sum_g 2^(x_gj - lse_g).  A block takes a slice of the rows of a (sequence, key
// head), four rows a thread and step.  The scores were written by the first launch moments ago and come from L2 as
// far as they fit (4 bytes per query head and row, against 2 width values of the cache: 6 % of its bytes for eight
// heads on bf16 rows of 128); read as the first to leave it, so that what does not fit costs no more than itself (131 MB
// of scores: 34 -> 29 us).  What a block does before its first score (tiles before its sequence, the lse of its
// heads) is a chain of waits, so slices are as long as filling the GPU allows.
// What needs only the lengths is done before the wait for the first launch.
#include <algorithm>

#include "../common.hpp"
#include "kv_attend.hpp"
#include "kv_launch.cuh"

namespace nve_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kStep = kThreads * 4;    // rows a weight block takes at once
constexpr int kMaxChunk = 64;          // query heads of a unit
constexpr float kNegInf = -__builtin_huge_valf();

// relative error 2^-22; a probability below 2^-126 is 0
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The CTAs that had a part of the unit that begins at tile `first_tile`, and where their parts are in the scratch: a
// CTA's first part is slot 0, and only the first CTA of a unit can have it second.
struct Parts {
  int32_t first, last;
  int32_t first_slot;
  __device__ __forceinline__ int64_t row(const KvAttendParams& p, int32_t c) const {
    return (static_cast<int64_t>(c) * 2 + (c == first ? first_slot : 0)) * p.rows_per_unit;
  }
};
__device__ __forceinline__ Parts parts_of(TileSplit split, int32_t first_tile, int32_t tiles) {
  Parts r;
  r.first = cta_of_tile(split, first_tile);
  r.last = cta_of_tile(split, first_tile + tiles - 1);
  r.first_slot = part_slot(run_first(split, r.first), first_tile);
  return r;
}

// (maximum, sum) of two runs together
__device__ __forceinline__ float2 join_ml(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), base = m == kNegInf ? 0.0f : m;
  return make_float2(m, a.y * exp2f(a.x - base) + b.y * exp2f(b.x - base));
}

__device__ __forceinline__ void first_launch_done() {
  grid_wait();
  grid_release();
}

struct JoinPlan {
  int32_t weight_blocks;             // the first blocks: slices of rows
  int32_t slices;                    // of a (sequence, key head)
  int32_t slice_rows;                // a multiple of kStep
  int32_t heads;                     // query heads of a join block: 1, 2, 4 or 8
  int32_t per_unit;                  // join blocks of a unit
};

// kAtOnce: query heads whose scores a thread has under way together.  Eight take 80 registers, three blocks per SM; a
// unit of four heads or fewer runs four blocks (64 sequences of 3000 rows, four heads: 14.0 us against 18.5; with eight
// heads in two rounds of four it is the other way round, 48.7 against 38.8).
template <int kAtOnce>
__global__ void __launch_bounds__(kThreads, kAtOnce == 4 ? 4 : 3) join_kernel(const KvAttendParams p, const JoinPlan plan) {
  __shared__ int32_t s_sum[kWarps][2];
  __shared__ float s_lse[kMaxChunk];
  __shared__ float s_l[kWarps], s_acc[kWarps][256];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units = p.cache.heads * p.chunks;
  const int block = static_cast<int>(blockIdx.x);
  const bool weights = block < plan.weight_blocks;
  const int list = weights ? block / plan.slices : (block - plan.weight_blocks) / plan.per_unit;   // (sequence, key head), or (sequence, unit)
  const int b = list / (weights ? p.cache.heads : units);

  const int length = kv_length(p.table, b, nullptr);
  const int tiles = tiles_of(length, p.tile_rows);
  const int row0 = weights ? (block - list * plan.slices) * plan.slice_rows : 0;
  if (row0 >= length) {
    first_launch_done();
    return;
  }
  // tiles of all sequences, and of those before b
  int32_t all = 0, before = 0;
  for (int x = tid; x < p.table.sequences; x += kThreads) {
    const int nt = tiles_of(kv_length(p.table, x, nullptr), p.tile_rows);
    all += nt;
    if (x < b) before += nt;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) {
    s_sum[warp][0] = all;
    s_sum[warp][1] = before;
  }
  __syncthreads();
  all = before = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    all += s_sum[w][0];
    before += s_sum[w][1];
  }
  const int32_t total = all * units;                        // below 2^31, as the host has seen to
  const TileSplit split = tile_split(total, min(p.ctas, total));
  const int32_t seq_tile = before * units;

  if (!weights) {
    // ---- join of some query heads of a unit
    const int unit = list - b * units;
    const Parts parts = parts_of(split, seq_tile + unit * tiles, tiles);
    first_launch_done();
    if (parts.first == parts.last) return;                  // done by the CTA that had it alone
    const int head = unit / p.chunks, chunk = unit - head * p.chunks;
    const int shares = kWarps / plan.heads;                 // warps of a query head
    const int share = warp % shares;
    const int hr = (block - plan.weight_blocks - list * plan.per_unit) * plan.heads + warp / shares;
    const bool mine = hr < min(p.chunk, p.group - chunk * p.chunk);
    const int width = p.cache.width;
    float m = kNegInf, l = 0.0f;
    if (mine) {
      for (int32_t c = parts.first + lane; c <= parts.last; c += 32) m = fmaxf(m, p.part_ml[parts.row(p, c) + hr].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float base = m == kNegInf ? 0.0f : m;
      float acc[8] = {};
      for (int32_t c = parts.first + share; c <= parts.last; c += shares) {
        const int64_t row = parts.row(p, c) + hr;
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
    }
    __syncthreads();
    if (!mine) return;
    l = 0.0f;
    for (int w = 0; w < shares; w++) l += s_l[warp - share + w];
    const float v_scale = p.cache.value_scale != nullptr ? __ldg(p.cache.value_scale + head) : 1.0f;
    const float inv = l == 0.0f ? 0.0f : v_scale / l;
    const int q_head = head * p.group + chunk * p.chunk + hr;
    for (int d = share * 32 + lane; d < width; d += shares * 32) {
      float v = 0.0f;
      for (int w = 0; w < shares; w++) v += s_acc[warp - share + w][d];
      uint8_t* const to = p.out + b * p.out_seq + q_head * p.out_head + d * 2;
      if (p.q_bf16) *reinterpret_cast<__nv_bfloat16*>(to) = __float2bfloat16_rn(v * inv);
      else *reinterpret_cast<__half*>(to) = __float2half_rn(v * inv);
    }
    if (share == 0 && lane == 0 && p.lse != nullptr) {
      p.lse[static_cast<int64_t>(b) * p.q_heads + q_head] = l == 0.0f ? kNegInf : (m + log2f(l)) * 0.69314718055994530942f;
    }
    return;
  }

  // ---- weights of a slice of rows
  const int head = list - b * p.cache.heads;
  const int slice_end = min(row0 + plan.slice_rows, length);
  // four rows of one page are one piece of memory where pages hold fours
  const bool four = p.cache.page_size % 4 == 0 && reinterpret_cast<uint64_t>(p.cache.weights) % 16 == 0;
  // pages and slots of the four rows from `row` on (with `four`, of the first); page -1: not there
  auto find = [&](int row, int32_t (&page)[4], int32_t (&slot)[4]) {
#pragma unroll
    for (int x = 0; x < 4; x++) {
      page[x] = -1;
      if (row + x < slice_end && (x == 0 || !four)) {
        page[x] = kv_locate(p.cache, p.table.pages, p.table.stride, b, row + x, &slot[x]);
      }
    }
  };
  int32_t page[4], slot[4];
  find(row0 + tid * 4, page, slot);
  first_launch_done();
  for (int chunk = 0; chunk < p.chunks; chunk++) {
    const int unit = head * p.chunks + chunk;
    const int32_t first_tile = seq_tile + unit * tiles;
    const int heads = min(p.chunk, p.group - chunk * p.chunk);
    const Parts parts = parts_of(split, first_tile, tiles);
    if (chunk > 0) __syncthreads();
    if (parts.first == parts.last) {
      if (tid < heads) s_lse[tid] = p.unit_lse[(static_cast<int64_t>(b) * units + unit) * p.rows_per_unit + tid];
    } else {
      // eight lanes a head
      for (int g0 = warp * 4; g0 < heads; g0 += kWarps * 4) {
        const int g = g0 + (lane >> 3);
        float2 ml = make_float2(kNegInf, 0.0f);
        if (g < heads) {
          for (int32_t c = parts.first + (lane & 7); c <= parts.last; c += 8) ml = join_ml(ml, p.part_ml[parts.row(p, c) + g]);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
          const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, ml.x, o), __shfl_xor_sync(0xffffffffu, ml.y, o));
          ml = join_ml(ml, other);
        }
        if ((lane & 7) == 0 && g < heads) s_lse[g] = ml.y == 0.0f ? kNegInf : ml.x + log2f(ml.y);
      }
    }
    __syncthreads();
    if (chunk > 0) find(row0 + tid * 4, page, slot);
    for (int row = row0 + tid * 4; row < slice_end; row += kStep) {
      // in this order, so that nothing waits before everything is under way: scores, weights, the pages of the next step
      const int tile = row / p.tile_rows, in_tile = row % p.tile_rows;
      const float* const s = p.scores + (static_cast<int64_t>(first_tile) + tile) * p.chunk * p.tile_rows + in_tile;
      float4 x[kAtOnce];
#pragma unroll
      for (int g = 0; g < kAtOnce; g++)
        if (g < heads) x[g] = __ldcs(reinterpret_cast<const float4*>(s + g * p.tile_rows));
      float w[4] = {};
      float* at[4];
      const bool piece = four && row + 3 < slice_end && page[0] >= 0;
      if (piece) {
        at[0] = p.cache.weights + kv_weight_index(p.cache, page[0], head, slot[0]);
        const float4 old = *reinterpret_cast<const float4*>(at[0]);
        w[0] = old.x;
        w[1] = old.y;
        w[2] = old.z;
        w[3] = old.w;
      } else {
#pragma unroll
        for (int y = 0; y < 4; y++) {
          at[y] = nullptr;
          const int from = four ? 0 : y;
          if (row + y < slice_end && page[from] >= 0) {
            at[y] = p.cache.weights + kv_weight_index(p.cache, page[from], head, slot[from]) + (four ? y : 0);
            w[y] = *at[y];
          }
        }
      }
      find(row + kStep, page, slot);
      float sum[4] = {};
      for (int g0 = 0; g0 < heads; g0 += kAtOnce) {
#pragma unroll
        for (int g = 0; g < kAtOnce; g++) {
          if (g0 + g >= heads) break;
          if (g0 > 0) x[g] = __ldcs(reinterpret_cast<const float4*>(s + (g0 + g) * p.tile_rows));
          const float e = s_lse[g0 + g];
          if (e != kNegInf) {
            sum[0] += exp2_fast(x[g].x - e);
            sum[1] += exp2_fast(x[g].y - e);
            sum[2] += exp2_fast(x[g].z - e);
            sum[3] += exp2_fast(x[g].w - e);
          }
        }
      }
      if (piece) {
        *reinterpret_cast<float4*>(at[0]) = make_float4(w[0] + sum[0], w[1] + sum[1], w[2] + sum[2], w[3] + sum[3]);
      } else {
#pragma unroll
        for (int y = 0; y < 4; y++)
          if (at[y] != nullptr) *at[y] = w[y] + sum[y];
      }
    }
  }
}

}  // namespace

void launch_kv_join(const KvAttendParams& p, int sms, cudaStream_t stream) {
  const int64_t lists = static_cast<int64_t>(p.table.sequences) * p.cache.heads;
  const int64_t unit_count = lists * p.chunks;
  JoinPlan plan{};
  // slices: three blocks per SM (as many as run at once) if the rows are enough for that; at most six steps, so that
  // lists of different lengths do not wait for the longest (128 sequences of 4000 to 12000 rows: 34 us against 39)
  const int64_t most = std::max<int64_t>(1, ceil_div(p.table.capacity, kStep));
  const int64_t wanted = std::min<int64_t>(most, std::max<int64_t>(ceil_div(most, 6), int64_t{3} * sms / lists));
  plan.slice_rows = static_cast<int32_t>(ceil_div(most, wanted) * kStep);
  plan.slices = static_cast<int32_t>(std::max<int64_t>(1, ceil_div(p.table.capacity, plan.slice_rows)));
  plan.weight_blocks = p.scores != nullptr ? static_cast<int32_t>(lists * plan.slices) : 0;
  plan.heads = 1;
  while (plan.heads < kWarps && plan.heads < p.chunk && unit_count * ceil_div(p.chunk, plan.heads) > sms) plan.heads *= 2;
  plan.per_unit = static_cast<int32_t>(ceil_div(p.chunk, plan.heads));
  launch_overlapped(p.chunk <= 4 ? join_kernel<4> : join_kernel<8>, plan.weight_blocks + unit_count * plan.per_unit, kThreads,
                    0, 1, stream, p, plan);
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
