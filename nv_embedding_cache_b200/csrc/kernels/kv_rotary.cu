// Rotary positions with several axes, alone and as the write into the paged cache.
//
// (a, b) -> (a cos - b sin, b cos + a sin) with angle = positions[axis of the pair][token] * inv_freq[pair].
// Every value is read once and written once and meets three flops, so memory bounds it.  The angles are shared by
// all heads of a token: a block takes a few whole tokens and computes their cosines and sines once into shared memory.
// A thread then keeps those of one item (a 16-byte vector of the row, or two for the split pairing: the vector of
// the a's and that of the b's) in registers and walks over the rows of several heads, the next row's load always under
// way; the first one's starts before the angles.  The queries, keys and values of a token go through one launch.
// Held at 64 registers, four blocks per SM: 65 us for 16 384 tokens of 40 heads of 128 in bf16 (5.2 TB/s; three blocks 69,
// five, which spill, 97), 73 us for the append of 13 391 tokens of 48 heads into E4M3 rows (4.1 TB/s).
//
// The angle is the product of a 32-bit integer and an fp32 number: exact in 64 bits up to its last two bits.  It is
// reduced there (in turns, so that the reduction is a subtraction of an integer) and only the remainder is
// rounded to fp32, so far positions are as exact as near ones.
#include <algorithm>

#include "../common.hpp"
#include "kv_launch.cuh"
#include "kv_rotary.cuh"

namespace nve_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokensPerBlock = 32;

template <typename T>
struct Wide;  // fp32 <-> stored value
template <>
struct Wide<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <>
struct Wide<__half> {
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <>
struct Wide<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(uint8_t* p, const float (&x)[VEC]) {
  Vec<T, VEC> u;
#pragma unroll
  for (int i = 0; i < VEC; i++) u.v[i] = Wide<T>::down(x[i]);
  *reinterpret_cast<Vec<T, VEC>*>(p) = u;
}

// Stored value of an E4M3 cache: x / scale, rounded to nearest even, saturated to the largest finite value.  One
// division per row: x (1 / scale) rounds once more, 2^-24, against the 2^-4 of the stored value.
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&x)[VEC], float inverse) {
  Vec<uint8_t, VEC> u;
  if constexpr (VEC == 1) {
    u.v[0] = __nv_cvt_float_to_fp8(x[0] * inverse, __NV_SATFINITE, __NV_E4M3);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(x[i] * inverse, x[i + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
      u.v[i] = static_cast<uint8_t>(two & 0xff);
      u.v[i + 1] = static_cast<uint8_t>(two >> 8);
    }
  }
  *reinterpret_cast<Vec<uint8_t, VEC>*>(p) = u;
}

struct TokenPlace {
  int64_t key, value;               // byte offsets of the token's row in the pools, head 0
  int64_t weight;                   // index of its weight, head 0
  bool stored;                      // has a place in the cache
  bool padding;                     // belongs to no sequence: nothing of it is written
};

// Which sequence token t belongs to and where its row goes; found by a whole warp, 32 offsets a step.
__device__ __forceinline__ TokenPlace place_token(const RotaryParams& p, int32_t t) {
  TokenPlace r{0, 0, 0, false, true};
  const int lane = threadIdx.x & 31;
  int32_t b, first;
  if (p.offsets != nullptr) {
    // lo: the last sequence that begins at or before t.  Offsets that do not ascend give some sequence; the row is
    // checked below whatever it is.
    const int32_t n = p.table.sequences;
    if (t < __ldg(p.offsets) || t >= __ldg(p.offsets + n)) return r;
    int32_t lo = 0, span = n;
    while (span > 1) {
      const int32_t stride = (span + 31) / 32;
      const int32_t at = lo + lane * stride;
      const bool before = lane * stride < span && __ldg(p.offsets + at) <= t;
      const int32_t steps = 31 - __clz(__ballot_sync(0xffffffffu, before) | 1u);
      lo += steps * stride;
      span = min(stride, span - steps * stride);
    }
    b = lo;
    first = __ldg(p.offsets + lo);
  } else {
    b = t / p.per_sequence;
    first = b * p.per_sequence;
  }
  r.padding = false;
  const int64_t row = static_cast<int64_t>(kv_length(p.table, b, p.cache.status)) + t - first;
  if (row < 0 || row >= p.table.capacity) {
    kv_flag(p.cache.status, NVE_B200_KV_BAD_LENGTH);
    return r;
  }
  int32_t slot;
  const int32_t page = kv_locate(p.cache, p.table.pages, p.table.stride, b, static_cast<int32_t>(row), &slot);
  if (page < 0) return r;
  r.key = page * p.cache.k_page + slot * p.cache.k_slot;
  r.value = page * p.cache.v_page + slot * p.cache.v_slot;
  r.weight = kv_weight_index(p.cache, page, 0, slot);
  r.stored = true;
  return r;
}

// VEC: values of one vector (16 bytes of T, or 1 where alignment or an odd pair count asks for it).
template <typename T, int VEC, bool INTERLEAVED, bool TO_CACHE, bool E4M3>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 turn[];                       // [tokens of the block][pairs] (cos, sin)
  __shared__ TokenPlace place[TO_CACHE ? kMaxTokensPerBlock : 1];
  constexpr bool kTwo = !INTERLEAVED || VEC == 1;        // the a's and the b's of a turned item are two vectors
  constexpr int kPairs = kTwo ? VEC : VEC / 2;           // pairs of an item
  using V = Vec<T, VEC>;
  const int32_t t0 = blockIdx.x * p.tokens_per_block;
  const int32_t nt = min(p.tokens_per_block, p.tokens - t0);

  // this thread: item `item` of the rows r0, r0 + row_lanes, .. of the tokens t, t + token_lanes, ..
  const int32_t group = threadIdx.x / p.lanes, t_first = group / p.row_lanes, r_first = group - t_first * p.row_lanes;
  int32_t item = threadIdx.x - group * p.lanes;
  int32_t t = t_first, r = r_first;
  bool pair_item, two;
  int32_t first;
  const int32_t gap = INTERLEAVED ? 1 : p.pairs;         // from the a's to the b's
  V a, b;
  auto set_item = [&]() {
    pair_item = item < p.turned_items;
    two = kTwo && pair_item;
    first = pair_item ? (INTERLEAVED && VEC == 1 ? 2 * item : item * VEC) : 2 * p.pairs + (item - p.turned_items) * VEC;
  };
  // group of rows r belongs to: 0 queries, 1 keys, 2 values; r becomes the head
  auto split_row = [&](int32_t& head) -> int {
    if (head < p.g[0].heads) return 0;
    head -= p.g[0].heads;
    if (head < p.g[1].heads) return 1;
    head -= p.g[1].heads;
    return 2;
  };
  auto load = [&](int32_t token, int32_t head, V& x, V& y) {
    const int which = split_row(head);
    const RowGroup& g = which == 0 ? p.g[0] : (which == 1 ? p.g[1] : p.g[2]);
    const uint8_t* const src = g.in + (t0 + token) * g.in_token + head * g.in_head + first * static_cast<int64_t>(sizeof(T));
    x = *reinterpret_cast<const V*>(src);
    if (two) y = *reinterpret_cast<const V*>(src + gap * static_cast<int64_t>(sizeof(T)));
  };
  set_item();
  grid_wait();
  grid_release();
  const int32_t token_lanes = kThreads / p.lanes / p.row_lanes;
  const bool works = t < min(nt, token_lanes) && item < p.items;   // threads that fill no whole token lane are idle
  if (works) load(t, r, a, b);

  if constexpr (TO_CACHE) {
    for (int32_t s = blockIdx.x * kThreads + threadIdx.x; s < p.table.sequences; s += gridDim.x * kThreads) {
      const int64_t more = p.offsets != nullptr ? static_cast<int64_t>(__ldg(p.offsets + s + 1)) - __ldg(p.offsets + s) : p.per_sequence;
      const int64_t n = kv_length(p.table, s, p.cache.status) + max(more, int64_t{0});
      p.new_lengths[s] = static_cast<int32_t>(min(n, static_cast<int64_t>(p.table.capacity)));
    }
    for (int32_t i = threadIdx.x >> 5; i < nt; i += kThreads / 32) {
      const TokenPlace at = place_token(p, t0 + i);
      if ((threadIdx.x & 31) == 0) place[i] = at;
    }
  }
  for (int32_t i = threadIdx.x; i < nt * p.pairs; i += kThreads) {
    const int32_t token = i / p.pairs, k = i - token * p.pairs;
    const int32_t axis = p.pair_axis != nullptr ? __ldg(p.pair_axis + k) : 0;
    float2 cs = make_float2(1.0f, 0.0f);
    if (static_cast<uint32_t>(axis) < static_cast<uint32_t>(p.axes)) {
      const int32_t pos = __ldg(p.positions + axis * p.axis_stride + (t0 + token) * p.token_stride);
      const double half_turns = static_cast<double>(pos) * static_cast<double>(__ldg(p.inv_freq + k)) *
                                0.31830988618379067153776752674503;     // 1 / pi
      const double rest = half_turns - 2.0 * rint(0.5 * half_turns);     // in [-1, 1]
      sincospif(static_cast<float>(rest), &cs.y, &cs.x);
      cs.y *= p.sign;
    } else {
      kv_flag(p.status, NVE_B200_KV_BAD_AXIS);
    }
    turn[i] = cs;
  }
  __syncthreads();

  auto finish = [&](int32_t token, int32_t head, const float2 (&cs)[kPairs], V x_raw, V y_raw) {
    const int which = split_row(head);
    bool as_is = which == 2 || !pair_item;
    uint8_t* dst;
    if (TO_CACHE && which > 0) {
      const TokenPlace& at = place[token];
      if (!at.stored) return;
      dst = which == 2 ? p.cache.values + at.value + head * p.cache.v_head : p.cache.keys + at.key + head * p.cache.k_head;
    } else {
      const RowGroup& g = which == 0 ? p.g[0] : p.g[1];
      dst = g.out + (t0 + token) * g.out_token + head * g.out_head;
      if (TO_CACHE && place[token].padding) {
        if (!p.zero_padding) return;
        x_raw = y_raw = V{};
        as_is = true;
      }
    }
    const bool to_e4m3 = E4M3 && which > 0;
    if (as_is && !to_e4m3) {
      *reinterpret_cast<V*>(dst + first * sizeof(T)) = x_raw;
      if (two) *reinterpret_cast<V*>(dst + (first + gap) * sizeof(T)) = y_raw;
      return;
    }
    float x[VEC], y[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      x[i] = Wide<T>::up(x_raw.v[i]);
      if (kTwo) y[i] = two ? Wide<T>::up(y_raw.v[i]) : 0.0f;
    }
    if (!as_is) {
#pragma unroll
      for (int i = 0; i < kPairs; i++) {
        float& xa = kTwo ? x[i] : x[2 * i];
        float& xb = kTwo ? y[i] : x[2 * i + 1];
        const float u0 = xa;
        xa = u0 * cs[i].x - xb * cs[i].y;
        xb = xb * cs[i].x + u0 * cs[i].y;
      }
    }
    if (to_e4m3) {
      const float* const s = which == 2 ? p.cache.value_scale : p.cache.key_scale;
      const float inverse = s != nullptr ? 1.0f / __ldg(s + head) : 1.0f;
      store_e4m3<VEC>(dst + first, x, inverse);
      if (two) store_e4m3<VEC>(dst + first + gap, y, inverse);
    } else {
      store_vec<T, VEC>(dst + first * sizeof(T), x);
      if (two) store_vec<T, VEC>(dst + (first + gap) * sizeof(T), y);
    }
  };

  if (works) {
    float2 cs[kPairs];
    int32_t cs_token = -1, cs_item = -1;
    for (;;) {
      // the row after this one: next row, next token, next item
      int32_t r_next = r + p.row_lanes, t_next = t, item_next = item;
      if (r_next >= p.rows) {
        r_next = r_first;
        t_next += token_lanes;
        if (t_next >= nt) {
          t_next = t_first;
          item_next += p.lanes;
        }
      }
      const bool more = item_next < p.items, same_item = item_next == item;
      V a_next, b_next;
      if (more && same_item) load(t_next, r_next, a_next, b_next);
      if (cs_token != t || cs_item != item) {
#pragma unroll
        for (int i = 0; i < kPairs; i++) cs[i] = pair_item ? turn[t * p.pairs + item * kPairs + i] : make_float2(1.0f, 0.0f);
        cs_token = t;
        cs_item = item;
      }
      finish(t, r, cs, a, b);
      if (!more) break;
      r = r_next;
      t = t_next;
      if (same_item) {
        a = a_next;
        b = b_next;
      } else {
        item = item_next;
        set_item();
        load(t, r, a, b);
      }
    }
  }
  if constexpr (TO_CACHE) {
    if (p.cache.weights != nullptr) {
      for (int32_t i = threadIdx.x; i < nt * p.cache.heads; i += kThreads) {
        const int32_t t = i / p.cache.heads, h = i - t * p.cache.heads;
        if (place[t].stored) p.cache.weights[place[t].weight + static_cast<int64_t>(h) * p.cache.page_size] = 0.0f;
      }
    }
  }
}

template <typename T, int VEC, bool INTERLEAVED, bool TO_CACHE, bool E4M3>
void launch_one(const RotaryParams& p, cudaStream_t stream) {
  launch_overlapped(rotary_kernel<T, VEC, INTERLEAVED, TO_CACHE, E4M3>,
                    std::max<int64_t>(1, ceil_div(p.tokens, p.tokens_per_block)), kThreads,
                    size_t(p.tokens_per_block) * p.pairs * sizeof(float2), 1, stream, p);
}

template <typename T, int VEC, bool INTERLEAVED>
void launch_dest(const RotaryParams& p, bool e4m3, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (p.to_cache && e4m3) return launch_one<T, VEC, INTERLEAVED, true, true>(p, stream);
    if (p.to_cache) return launch_one<T, VEC, INTERLEAVED, true, false>(p, stream);
  }
  launch_one<T, VEC, INTERLEAVED, false, false>(p, stream);
}

template <typename T>
void launch_type(RotaryParams& p, bool e4m3, bool interleaved, int sms, cudaStream_t stream) {
  constexpr int W = 16 / sizeof(T);
  // 16-byte vectors where every address, stride and the vector of b's allow them; single values otherwise
  uint64_t all = 0;
  for (const RowGroup& g : p.g) {
    if (g.heads == 0) continue;
    all |= reinterpret_cast<uint64_t>(g.in) | static_cast<uint64_t>(g.in_token) | static_cast<uint64_t>(g.in_head);
    if (g.out != nullptr) {
      all |= reinterpret_cast<uint64_t>(g.out) | static_cast<uint64_t>(g.out_token) | static_cast<uint64_t>(g.out_head);
    }
  }
  const bool wide = all % 16 == 0 && p.width % W == 0 && (interleaved ? 2 * p.pairs : p.pairs) % W == 0;
  const int vec = wide ? W : 1;
  p.turned_items = interleaved && wide ? 2 * p.pairs / vec : p.pairs / vec;
  p.items = p.turned_items + (p.width - 2 * p.pairs) / vec;
  // Threads of a block: `lanes` along the items of a row, then `row_lanes` along the rows of a token, then tokens.  Where
  // tokens are few, a block is one token and as many rows at once as fit; else a thread walks over about five rows of
  // a token, and of two tokens where that leaves every SM its blocks twice.
  p.lanes = std::min(p.items, kThreads);
  const int32_t groups = kThreads / p.lanes;
  const bool few = p.tokens < static_cast<int64_t>(sms) * 8;
  p.row_lanes = std::min({groups, p.rows, few ? groups : static_cast<int32_t>(ceil_div(p.rows, 5))});
  p.tokens_per_block = few ? 1 : std::min(groups / p.row_lanes, kMaxTokensPerBlock / 2);
  if (p.tokens / (p.tokens_per_block * 2) >= static_cast<int64_t>(sms) * 8) p.tokens_per_block *= 2;
  if (wide) {
    if (interleaved) launch_dest<T, W, true>(p, e4m3, stream);
    else launch_dest<T, W, false>(p, e4m3, stream);
  } else {
    if (interleaved) launch_dest<T, 1, true>(p, e4m3, stream);
    else launch_dest<T, 1, false>(p, e4m3, stream);
  }
}

}  // namespace

void launch_rotary(RotaryParams p, nve_data_type_t dtype, nve_data_type_t cache_dtype, bool interleaved, int sms,
                   cudaStream_t stream) {
  const bool e4m3 = p.to_cache && cache_dtype == NVE_DTYPE_E4M3;
  switch (dtype) {
    case NVE_DTYPE_FLOAT32: launch_type<float>(p, e4m3, interleaved, sms, stream); break;
    case NVE_DTYPE_FLOAT16: launch_type<__half>(p, e4m3, interleaved, sms, stream); break;
    default: launch_type<__nv_bfloat16>(p, e4m3, interleaved, sms, stream); break;
  }
}

}  // namespace nve_b200
