// Rotary positions with several axes, alone and as the write into the paged cache.
//
// (a, b) -> (a cos - b sin, b cos + a sin) with angle = positions[axis of the pair][token] * inv_freq[pair].
// Every value is read once and written once and meets three flops, so memory bounds it.  The angles are shared by
// all heads of a token: a block takes a few whole tokens, computes their cosines and sines once into shared memory
// and then streams the rows of every head past them, one 16-byte vector (two for the split pairing: the vector of
// the a's and that of the b's) per thread and step.  The queries, keys and values of a token go through one launch.
//
// The angle is the product of a 32-bit integer and an fp32 number: exact in 64 bits up to its last two bits.  It is
// reduced there (in turns, so that the reduction is a subtraction of an integer) and only the remainder is
// rounded to fp32, so far positions are as exact as near ones.
#include <algorithm>

#include "../common.hpp"
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

// Stored value of an E4M3 cache: x / scale, rounded to nearest even, saturated to the largest finite value.
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&x)[VEC], float scale) {
  Vec<uint8_t, VEC> u;
#pragma unroll
  for (int i = 0; i < VEC; i++) u.v[i] = __nv_cvt_float_to_fp8(x[i] / scale, __NV_SATFINITE, __NV_E4M3);
  *reinterpret_cast<Vec<uint8_t, VEC>*>(p) = u;
}

struct TokenPlace {
  int64_t key, value;               // byte offsets of the token's row in the pools, head 0
  int64_t weight;                   // index of its weight, head 0
  bool stored;                      // has a place in the cache
  bool padding;                     // belongs to no sequence: nothing of it is written
};

// Which sequence a token belongs to and where its row goes.
__device__ __forceinline__ TokenPlace place_token(const RotaryParams& p, int32_t t) {
  TokenPlace r{0, 0, 0, false, true};
  int32_t b, first;
  if (p.offsets != nullptr) {
    const int32_t n = p.table.sequences;
    if (t < __ldg(p.offsets) || t >= __ldg(p.offsets + n)) return r;
    int32_t lo = 0, hi = n;         // offsets[lo] <= t < offsets[hi]
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (__ldg(p.offsets + mid) <= t) lo = mid;
      else hi = mid;
    }
    b = lo;
    first = __ldg(p.offsets + lo);
  } else {
    b = t / p.per_sequence;
    first = b * p.per_sequence;
  }
  r.padding = false;
  const int64_t row = static_cast<int64_t>(kv_length(p.table, b, p.cache.status)) + (t - first);
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
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 turn[];                       // [tokens of the block][pairs] (cos, sin)
  __shared__ TokenPlace place[TO_CACHE ? kMaxTokensPerBlock : 1];
  const int32_t t0 = blockIdx.x * p.tokens_per_block;
  const int32_t nt = min(p.tokens_per_block, p.tokens - t0);

  if constexpr (TO_CACHE) {
    for (int32_t b = blockIdx.x * kThreads + threadIdx.x; b < p.table.sequences; b += gridDim.x * kThreads) {
      const int32_t more = p.offsets != nullptr ? __ldg(p.offsets + b + 1) - __ldg(p.offsets + b) : p.per_sequence;
      const int64_t n = static_cast<int64_t>(kv_length(p.table, b, p.cache.status)) + max(more, 0);
      p.new_lengths[b] = static_cast<int32_t>(min(n, static_cast<int64_t>(p.table.capacity)));
    }
    if (static_cast<int32_t>(threadIdx.x) < nt) place[threadIdx.x] = place_token(p, t0 + threadIdx.x);
  }
  for (int32_t i = threadIdx.x; i < nt * p.pairs; i += kThreads) {
    const int32_t t = i / p.pairs, k = i - t * p.pairs;
    const int32_t axis = p.pair_axis != nullptr ? __ldg(p.pair_axis + k) : 0;
    float2 cs = make_float2(1.0f, 0.0f);
    if (static_cast<uint32_t>(axis) < static_cast<uint32_t>(p.axes)) {
      const int32_t pos = __ldg(p.positions + axis * p.axis_stride + (t0 + t) * p.token_stride);
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

  constexpr bool kTwo = !INTERLEAVED || VEC == 1;        // the a's and the b's of a turned item are two vectors
  constexpr int U = 2;                                   // items in flight per thread
  using V = Vec<T, VEC>;
  const int32_t work = nt * p.rows * p.items;
  for (int32_t w0 = threadIdx.x; w0 < work; w0 += kThreads * U) {
    V a[U], b[U];
    uint8_t* dst[U];
    int32_t first[U], cs_at[U];                          // cs_at < 0: copied
    float scale[U];
    int to[U];                                           // 0: nothing, 1: rows of T, 2: E4M3 rows
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int32_t w = w0 + u * kThreads;
      to[u] = 0;
      if (w >= work) continue;
      const int32_t tr = static_cast<int32_t>(fast_div(w, p.item_div));
      const int32_t item = w - tr * p.items;
      const int32_t t = static_cast<int32_t>(fast_div(tr, p.row_div));
      int32_t head = tr - t * p.rows;
      const bool is_q = head < p.g[0].heads;
      if (!is_q) head -= p.g[0].heads;
      const bool is_v = !is_q && head >= p.g[1].heads;
      if (is_v) head -= p.g[1].heads;
      const RowGroup& g = is_q ? p.g[0] : (is_v ? p.g[2] : p.g[1]);
      const bool pair_item = item < p.turned_items;
      first[u] = pair_item ? (INTERLEAVED && VEC == 1 ? 2 * item : item * VEC)
                           : 2 * p.pairs + (item - p.turned_items) * VEC;
      const int64_t src = (t0 + t) * g.in_token + head * g.in_head + first[u] * static_cast<int64_t>(sizeof(T));
      if (TO_CACHE && !is_q) {
        const TokenPlace& at = place[t];
        if (!at.stored) continue;
        dst[u] = is_v ? p.cache.values + at.value + head * p.cache.v_head : p.cache.keys + at.key + head * p.cache.k_head;
        to[u] = E4M3 ? 2 : 1;
        if constexpr (E4M3) {
          const float* s = is_v ? p.cache.value_scale : p.cache.key_scale;
          scale[u] = s != nullptr ? __ldg(s + head) : 1.0f;
        }
      } else {
        dst[u] = g.out + (t0 + t) * g.out_token + head * g.out_head;
        to[u] = 1;
        if (TO_CACHE && place[t].padding) {
          if (!p.zero_padding) {
            to[u] = 0;
            continue;
          }
          a[u] = b[u] = V{};
          cs_at[u] = pair_item ? -2 : -1;
          continue;
        }
      }
      cs_at[u] = pair_item ? (is_v ? -2 : t * p.pairs + (kTwo ? item * VEC : item * (VEC / 2))) : -1;
      a[u] = *reinterpret_cast<const V*>(g.in + src);
      if (kTwo && pair_item) {
        b[u] = *reinterpret_cast<const V*>(g.in + src + (INTERLEAVED ? 1 : p.pairs) * static_cast<int64_t>(sizeof(T)));
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (to[u] == 0) continue;
      const bool two = kTwo && cs_at[u] != -1;
      const int32_t second = first[u] + (INTERLEAVED ? 1 : p.pairs);
      if (cs_at[u] < 0 && to[u] == 1) {                  // bytes as they are
        *reinterpret_cast<V*>(dst[u] + first[u] * sizeof(T)) = a[u];
        if (two) *reinterpret_cast<V*>(dst[u] + second * sizeof(T)) = b[u];
        continue;
      }
      float x[VEC], y[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        x[i] = Wide<T>::up(a[u].v[i]);
        if (kTwo) y[i] = two ? Wide<T>::up(b[u].v[i]) : 0.0f;
      }
      if (cs_at[u] >= 0) {
        if constexpr (kTwo) {
#pragma unroll
          for (int i = 0; i < VEC; i++) {
            const float2 cs = turn[cs_at[u] + i];
            const float xa = x[i];
            x[i] = xa * cs.x - y[i] * cs.y;
            y[i] = y[i] * cs.x + xa * cs.y;
          }
        } else {
#pragma unroll
          for (int i = 0; i < VEC / 2; i++) {
            const float2 cs = turn[cs_at[u] + i];
            const float xa = x[2 * i];
            x[2 * i] = xa * cs.x - x[2 * i + 1] * cs.y;
            x[2 * i + 1] = x[2 * i + 1] * cs.x + xa * cs.y;
          }
        }
      }
      if (E4M3 && to[u] == 2) {
        store_e4m3<VEC>(dst[u] + first[u], x, scale[u]);
        if (two) store_e4m3<VEC>(dst[u] + second, y, scale[u]);
      } else {
        store_vec<T, VEC>(dst[u] + first[u] * sizeof(T), x);
        if (two) store_vec<T, VEC>(dst[u] + second * sizeof(T), y);
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
  const int64_t token_blocks = ceil_div(p.tokens, p.tokens_per_block);
  const unsigned grid = static_cast<unsigned>(std::max<int64_t>(token_blocks, 1));
  rotary_kernel<T, VEC, INTERLEAVED, TO_CACHE, E4M3>
      <<<grid, kThreads, size_t(p.tokens_per_block) * p.pairs * sizeof(float2), stream>>>(p);
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
  p.item_div = make_fast_div(static_cast<uint32_t>(p.items));
  p.row_div = make_fast_div(static_cast<uint32_t>(p.rows));
  // one token per block until every SM has its eight blocks, then several, so that a block's angles are one step
  // of all its threads
  const int64_t fill = static_cast<int64_t>(sms) * 8;
  p.tokens_per_block = static_cast<int32_t>(std::min<int64_t>(4, std::max<int64_t>(1, p.tokens / fill)));
  if (wide) {
    if (interleaved) launch_dest<T, W, true>(p, e4m3, stream);
    else launch_dest<T, W, false>(p, e4m3, stream);
  } else {
    if (interleaved) launch_dest<T, 1, true>(p, e4m3, stream);
    else launch_dest<T, 1, false>(p, e4m3, stream);
  }
  NVE_B200_CUDA(cudaGetLastError());
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
