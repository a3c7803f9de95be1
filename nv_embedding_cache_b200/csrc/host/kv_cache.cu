// C ABI of the paged key/value cache (include/nve_b200_kv.h): argument checks, parameter packing, scratch layout.
#include <algorithm>
#include <cmath>

#include "../common.hpp"
#include "../kernels/kv_attend.hpp"
#include "../kernels/kv_evict.hpp"
#include "../kernels/kv_rotary.cuh"

namespace nve_b200 {

namespace {

constexpr int64_t kIntMax = 0x7fffffff;
constexpr int64_t kMaxWidth = 256;         // of cache rows
constexpr int32_t kMaxTurnedWidth = 1024;  // of rows that are only turned

int64_t value_bytes(nve_data_type_t t) {
  switch (t) {
    case NVE_DTYPE_FLOAT32: return 4;
    case NVE_DTYPE_FLOAT16:
    case NVE_DTYPE_BFLOAT16: return 2;
    default: return 1;
  }
}

uint64_t bits(const void* p) { return reinterpret_cast<uint64_t>(p); }

KvView view_of(const nve_b200_kv_cache_t* c, const char* who) {
  NVE_B200_ARG(c != nullptr, who, ": cache is NULL");
  NVE_B200_ARG(c->keys != nullptr && c->values != nullptr, who, ": the cache has no keys or no values");
  NVE_B200_ARG(c->dtype == NVE_DTYPE_FLOAT16 || c->dtype == NVE_DTYPE_BFLOAT16 || c->dtype == NVE_DTYPE_E4M3, who,
               ": cache rows must be FLOAT16, BFLOAT16 or E4M3");
  NVE_B200_ARG(c->num_pages > 0 && c->num_pages <= kIntMax, who, ": num_pages must be in [1, 2^31)");
  NVE_B200_ARG(c->page_size > 0 && c->num_heads > 0, who, ": page_size and num_heads must be positive");
  NVE_B200_ARG(c->head_width > 0 && c->head_width <= kMaxWidth, who, ": head_width must be in [1, 256]");
  NVE_B200_ARG(c->head_width * value_bytes(c->dtype) % 16 == 0, who, ": rows must be a multiple of 16 bytes");
  uint64_t all = bits(c->keys) | bits(c->values);
  for (int i = 0; i < 3; i++) {
    NVE_B200_ARG(c->key_strides[i] >= 0 && c->value_strides[i] >= 0, who, ": negative cache strides");
    all |= static_cast<uint64_t>(c->key_strides[i]) | static_cast<uint64_t>(c->value_strides[i]);
  }
  NVE_B200_ARG(all % 16 == 0, who, ": addresses and strides of the cache must be multiples of 16 bytes");
  NVE_B200_ARG(c->dtype == NVE_DTYPE_E4M3 || (c->key_scale == nullptr && c->value_scale == nullptr), who,
               ": scales belong to E4M3 caches");
  KvView v{};
  v.keys = static_cast<uint8_t*>(c->keys);
  v.values = static_cast<uint8_t*>(c->values);
  v.k_page = c->key_strides[0];
  v.k_slot = c->key_strides[1];
  v.k_head = c->key_strides[2];
  v.v_page = c->value_strides[0];
  v.v_slot = c->value_strides[1];
  v.v_head = c->value_strides[2];
  v.weights = c->weights;
  v.key_scale = c->key_scale;
  v.value_scale = c->value_scale;
  v.status = c->status;
  v.num_pages = static_cast<uint32_t>(c->num_pages);
  v.page_size = c->page_size;
  v.heads = c->num_heads;
  v.width = c->head_width;
  v.page_div = make_fast_div(static_cast<uint32_t>(c->page_size));
  return v;
}

// A page table of `sequences` rows; capacity: rows a sequence may have (bounded by max_length when that is >= 0).
KvTable table_of(const nve_b200_kv_cache_t* c, const int32_t* pages, int64_t stride, int32_t per_sequence,
                 const int32_t* lengths, int32_t sequences, int32_t max_length, const char* who) {
  NVE_B200_ARG(sequences >= 0, who, ": negative number of sequences");
  NVE_B200_ARG(per_sequence >= 0 && static_cast<int64_t>(per_sequence) * c->page_size <= kIntMax, who,
               ": pages_per_sequence * page_size must be in [0, 2^31)");
  NVE_B200_ARG(sequences == 0 || (lengths != nullptr && (pages != nullptr || per_sequence == 0)), who,
               ": page_table or lengths is NULL");
  NVE_B200_ARG(stride >= per_sequence || sequences <= 1, who, ": rows of the page table overlap");
  KvTable t{};
  t.pages = pages;
  t.stride = stride;
  t.lengths = lengths;
  t.sequences = sequences;
  t.capacity = per_sequence * c->page_size;
  if (max_length >= 0) {
    NVE_B200_ARG(max_length <= t.capacity, who, ": max_length is above pages_per_sequence * page_size");
    t.capacity = max_length;
  }
  return t;
}

RowGroup group_of(const nve_b200_head_rows_t& r, int64_t elem, bool with_out, const char* who) {
  NVE_B200_ARG(r.num_heads >= 0, who, ": negative number of heads");
  NVE_B200_ARG(r.in != nullptr && (!with_out || r.out != nullptr), who, ": NULL rows");
  uint64_t all = bits(r.in) | static_cast<uint64_t>(r.in_token_stride) | static_cast<uint64_t>(r.in_head_stride);
  if (with_out) {
    all |= bits(r.out) | static_cast<uint64_t>(r.out_token_stride) | static_cast<uint64_t>(r.out_head_stride);
  }
  NVE_B200_ARG(all % static_cast<uint64_t>(elem) == 0, who, ": addresses and strides must be multiples of the value size");
  RowGroup g{};
  g.in = static_cast<const uint8_t*>(r.in);
  g.in_token = r.in_token_stride;
  g.in_head = r.in_head_stride;
  g.out = with_out ? static_cast<uint8_t*>(r.out) : nullptr;
  g.out_token = with_out ? r.out_token_stride : 0;
  g.out_head = with_out ? r.out_head_stride : 0;
  g.heads = r.num_heads;
  return g;
}

void pack_rotary(const nve_b200_rotary_t* r, int32_t width, int64_t tokens, RotaryParams& p, const char* who) {
  p.width = width;
  p.sign = 1.0f;
  if (r == nullptr) return;
  NVE_B200_ARG(r->num_pairs >= 0 && static_cast<int64_t>(r->num_pairs) * 2 <= width, who,
               ": 2 * num_pairs must be in [0, head width]");
  NVE_B200_ARG(r->num_axes > 0, who, ": num_axes must be positive");
  NVE_B200_ARG(r->num_pairs == 0 || tokens == 0 || (r->positions != nullptr && r->inv_freq != nullptr), who,
               ": positions or inv_freq is NULL");
  p.positions = r->positions;
  p.axis_stride = r->axis_stride;
  p.token_stride = r->token_stride;
  p.axes = r->num_axes;
  p.inv_freq = r->inv_freq;
  p.pair_axis = r->pair_axis;
  p.pairs = r->num_pairs;
  p.status = r->status;
}

void rotary(const nve_b200_rotary_t* r, nve_data_type_t dtype, int32_t width, int64_t tokens,
            const nve_b200_head_rows_t* groups, int32_t num_groups, bool backward, cudaStream_t stream) {
  const char* who = "rotary";
  NVE_B200_ARG(r != nullptr, who, ": rotary is NULL");
  NVE_B200_ARG(dtype == NVE_DTYPE_FLOAT32 || dtype == NVE_DTYPE_FLOAT16 || dtype == NVE_DTYPE_BFLOAT16, who,
               ": values must be FLOAT32, FLOAT16 or BFLOAT16");
  NVE_B200_ARG(width > 0 && width <= kMaxTurnedWidth, who, ": head width must be in [1, 1024]");
  NVE_B200_ARG(tokens >= 0 && tokens <= kIntMax, who, ": number of tokens must be in [0, 2^31)");
  NVE_B200_ARG(num_groups >= 1 && num_groups <= 2 && groups != nullptr, who, ": one or two groups of rows");
  RotaryParams p{};
  pack_rotary(r, width, tokens, p, who);
  if (backward) p.sign = -1.0f;
  p.tokens = static_cast<int32_t>(tokens);
  if (tokens == 0) return;
  for (int i = 0; i < num_groups; i++) {
    if (groups[i].num_heads == 0) continue;
    p.g[i] = group_of(groups[i], value_bytes(dtype), true, who);
    NVE_B200_ARG(groups[i].in != groups[i].out || (groups[i].in_token_stride == groups[i].out_token_stride &&
                                                   groups[i].in_head_stride == groups[i].out_head_stride),
                 who, ": rows turned in place need one set of strides");
    p.rows += p.g[i].heads;
  }
  if (p.rows == 0) return;
  NVE_B200_ARG(static_cast<int64_t>(p.rows) * width * 4 <= kIntMax, who, ": too many heads");
  launch_rotary(p, dtype, dtype, r->interleaved != 0, sm_count(), stream);
}

void append(const nve_b200_kv_cache_t* cache, const nve_b200_kv_append_t* a, cudaStream_t stream) {
  const char* who = "kv_append";
  RotaryParams p{};
  p.cache = view_of(cache, who);
  NVE_B200_ARG(a != nullptr, who, ": args is NULL");
  NVE_B200_ARG(a->dtype == cache->dtype ||
                   (cache->dtype == NVE_DTYPE_E4M3 && (a->dtype == NVE_DTYPE_FLOAT16 || a->dtype == NVE_DTYPE_BFLOAT16)),
               who, ": rows must have the cache's type, or be FLOAT16 or BFLOAT16 for an E4M3 cache");
  NVE_B200_ARG(a->dtype != NVE_DTYPE_E4M3, who, ": new rows must be FLOAT16 or BFLOAT16");
  NVE_B200_ARG(a->num_tokens >= 0 && a->num_tokens <= kIntMax, who, ": number of tokens must be in [0, 2^31)");
  p.table = table_of(cache, a->page_table, a->page_table_stride, a->pages_per_sequence, a->lengths, a->num_sequences,
                     -1, who);
  if (a->num_sequences == 0) {              // every token is padding
    NVE_B200_ARG(a->num_tokens == 0 || a->csr_offsets != nullptr, who, ": tokens without a sequence");
    if (a->num_tokens == 0) return;
  } else {
    NVE_B200_ARG(a->new_lengths != nullptr, who, ": new_lengths is NULL");
    NVE_B200_ARG(a->new_lengths != a->lengths, who, ": new_lengths must not be lengths");
  }
  if (a->csr_offsets == nullptr) {
    NVE_B200_ARG(a->num_tokens % a->num_sequences == 0, who, ": num_tokens is not a multiple of num_sequences");
    p.per_sequence = static_cast<int32_t>(a->num_tokens / a->num_sequences);
  }
  p.offsets = a->csr_offsets;
  p.new_lengths = a->new_lengths;
  p.zero_padding = a->zero_padding != 0;
  p.to_cache = true;
  p.tokens = static_cast<int32_t>(a->num_tokens);
  pack_rotary(a->rotary, cache->head_width, a->num_tokens, p, who);
  const int64_t elem = value_bytes(a->dtype);
  if (a->num_tokens > 0) {
    if (a->q.in != nullptr && a->q.num_heads != 0) p.g[0] = group_of(a->q, elem, true, who);
    NVE_B200_ARG(a->k.num_heads == cache->num_heads && a->v.num_heads == cache->num_heads, who,
                 ": k and v must have the cache's heads");
    p.g[1] = group_of(a->k, elem, false, who);
    p.g[2] = group_of(a->v, elem, false, who);
    NVE_B200_ARG(a->q.in == nullptr || a->q.in != a->q.out || (a->q.in_token_stride == a->q.out_token_stride &&
                                                               a->q.in_head_stride == a->q.out_head_stride),
                 who, ": queries turned in place need one set of strides");
  } else {
    p.g[1].heads = 1;                      // nothing is read: only the new lengths are written
  }
  p.rows = p.g[0].heads + p.g[1].heads + p.g[2].heads;
  NVE_B200_ARG(static_cast<int64_t>(p.rows) * p.width * 4 <= kIntMax, who, ": too many heads");
  launch_rotary(p, a->dtype, cache->dtype, a->rotary != nullptr && a->rotary->interleaved != 0, sm_count(), stream);
}

// Takes `bytes` from a scratch buffer, 256-byte steps.
template <typename T>
T* carve(uint8_t*& at, int64_t count) {
  T* const p = reinterpret_cast<T*>(at);
  at += (count * static_cast<int64_t>(sizeof(T)) + 255) / 256 * 256;
  return p;
}

void attend(const nve_b200_kv_cache_t* cache, const nve_b200_kv_attend_t* a, void* scratch, size_t* scratch_bytes,
            cudaStream_t stream) {
  const char* who = "kv_attend";
  KvAttendParams p{};
  p.cache = view_of(cache, who);
  NVE_B200_ARG(a != nullptr && scratch_bytes != nullptr, who, ": args or scratch_bytes is NULL");
  NVE_B200_ARG(a->dtype == cache->dtype ||
                   (cache->dtype == NVE_DTYPE_E4M3 && (a->dtype == NVE_DTYPE_FLOAT16 || a->dtype == NVE_DTYPE_BFLOAT16)),
               who, ": queries must have the cache's type, or be FLOAT16 or BFLOAT16 for an E4M3 cache");
  NVE_B200_ARG(a->dtype != NVE_DTYPE_E4M3, who, ": queries must be FLOAT16 or BFLOAT16");
  NVE_B200_ARG(cache->head_width % 8 == 0, who, ": head_width must be a multiple of 8");
  NVE_B200_ARG(a->num_q_heads > 0 && a->num_q_heads % cache->num_heads == 0, who,
               ": num_q_heads must be a positive multiple of the cache's heads");
  NVE_B200_ARG(a->max_length >= 0, who, ": negative max_length");
  NVE_B200_ARG(std::isfinite(a->scale), who, ": scale must be finite");
  NVE_B200_ARG(!a->accumulate_weights || cache->weights != nullptr, who, ": the cache keeps no weights");
  p.table = table_of(cache, a->page_table, a->page_table_stride, a->pages_per_sequence, a->lengths, a->num_sequences,
                     a->max_length, who);
  p.q_heads = a->num_q_heads;
  p.group = a->num_q_heads / cache->num_heads;
  p.chunks = static_cast<int32_t>(ceil_div(p.group, 64));
  p.chunk = static_cast<int32_t>(ceil_div(p.group, p.chunks));
  p.rows_per_unit = p.chunk <= 8 ? 8 : (p.chunk <= 16 ? 16 : (p.chunk <= 32 ? 32 : 64));
  const int64_t units = static_cast<int64_t>(cache->num_heads) * p.chunks;
  p.tile_rows = kv_tile_rows(cache->head_width, static_cast<int>(value_bytes(cache->dtype)));
  const int64_t tiles = a->num_sequences * units * ceil_div(p.table.capacity, p.tile_rows);
  NVE_B200_ARG(tiles < kIntMax && static_cast<int64_t>(a->num_sequences) * p.q_heads < (1 << 30) &&
                   static_cast<int64_t>(a->num_sequences) * cache->num_heads * ceil_div(p.table.capacity, 1024) < (1 << 30),
               who,
               ": too many rows for one call");
  if (a->num_sequences == 0) {
    if (scratch == nullptr) *scratch_bytes = 0;
    return;
  }
  const int resident = kv_attend_resident(cache->dtype, cache->head_width, p.rows_per_unit);
  p.ctas = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(resident, tiles)));
  auto* const begin = static_cast<uint8_t*>(scratch);
  uint8_t* at = begin;
  const int64_t part_rows = static_cast<int64_t>(p.ctas) * 2 * p.rows_per_unit;
  p.part_acc = carve<float>(at, part_rows * cache->head_width);
  p.part_ml = carve<float2>(at, part_rows);
  if (a->accumulate_weights) {
    p.unit_lse = carve<float>(at, a->num_sequences * units * p.rows_per_unit);
    p.scores = carve<float>(at, std::max<int64_t>(tiles, 1) * p.chunk * p.tile_rows);
  }
  const size_t need = static_cast<size_t>(at - begin);
  if (scratch == nullptr) {
    *scratch_bytes = need;
    return;
  }
  NVE_B200_ARG(*scratch_bytes >= need, who, ": scratch buffer too small");
  NVE_B200_ARG(bits(scratch) % 256 == 0, who, ": scratch must be 256-byte aligned");
  NVE_B200_ARG(a->q != nullptr && a->out != nullptr, who, ": q or out is NULL");
  NVE_B200_ARG((bits(a->q) | static_cast<uint64_t>(a->q_sequence_stride) | static_cast<uint64_t>(a->q_head_stride)) % 16 == 0,
               who, ": address and strides of q must be multiples of 16 bytes");
  NVE_B200_ARG((bits(a->out) | static_cast<uint64_t>(a->out_sequence_stride) | static_cast<uint64_t>(a->out_head_stride)) % 2 == 0,
               who, ": address and strides of out must be multiples of the value size");
  p.q = static_cast<const uint8_t*>(a->q);
  p.q_seq = a->q_sequence_stride;
  p.q_head = a->q_head_stride;
  p.out = static_cast<uint8_t*>(a->out);
  p.out_seq = a->out_sequence_stride;
  p.out_head = a->out_head_stride;
  p.lse = a->lse;
  p.q_bf16 = a->dtype == NVE_DTYPE_BFLOAT16;
  p.scale_log2 = a->scale * 1.44269504088896340736f;
  launch_kv_attend(p, cache->dtype, stream);
  launch_kv_join(p, sm_count(), stream);
}

void evict(const nve_b200_kv_cache_t* cache, const nve_b200_kv_evict_t* a, cudaStream_t stream) {
  const char* who = "kv_evict";
  KvEvictParams p{};
  p.cache = view_of(cache, who);
  NVE_B200_ARG(a != nullptr, who, ": args is NULL");
  NVE_B200_ARG(cache->weights != nullptr, who, ": the cache keeps no weights");
  NVE_B200_ARG(a->budget > 0 && a->sinks >= 0 && a->recent >= 0 &&
                   static_cast<int64_t>(a->sinks) + a->recent <= a->budget,
               who, ": budget must be positive and hold sinks + recent rows");
  NVE_B200_ARG(a->max_length >= 0, who, ": negative max_length");
  p.table = table_of(cache, a->page_table, a->page_table_stride, a->pages_per_sequence, a->lengths, a->num_sequences,
                     a->max_length, who);
  if (a->num_sequences == 0) return;
  const int64_t most = std::min(a->budget, a->max_length);
  NVE_B200_ARG(a->new_pages_per_sequence >= 0 &&
                   static_cast<int64_t>(a->new_pages_per_sequence) * cache->page_size >= most,
               who, ": new_page_table holds fewer than min(budget, max_length) rows");
  NVE_B200_ARG(a->new_page_table_stride >= a->new_pages_per_sequence || a->num_sequences <= 1, who,
               ": rows of the new page table overlap");
  NVE_B200_ARG(a->kept != nullptr && a->new_lengths != nullptr && (a->new_page_table != nullptr || most == 0), who,
               ": kept, new_lengths or new_page_table is NULL");
  NVE_B200_ARG(a->new_lengths != a->lengths, who, ": new_lengths must not be lengths");
  NVE_B200_ARG(static_cast<int64_t>(a->num_sequences) * cache->num_heads * std::max<int64_t>(8, ceil_div(most, 32)) < kIntMax,
               who, ": too many rows for one call");
  p.new_pages = a->new_page_table;
  p.new_stride = a->new_page_table_stride;
  p.budget = a->budget;
  p.sinks = a->sinks;
  p.recent = a->recent;
  p.kept = a->kept;
  p.new_lengths = a->new_lengths;
  p.row_bytes = static_cast<int32_t>(cache->head_width * value_bytes(cache->dtype));
  launch_kv_evict(p, sm_count(), stream);
}

}  // namespace
}  // namespace nve_b200

extern "C" {

nve_status_t nve_b200_rotary(const nve_b200_rotary_t* rotary, nve_data_type_t dtype, int32_t head_width,
                             int64_t num_tokens, const nve_b200_head_rows_t* groups, int32_t num_groups,
                             int32_t backward, void* stream) {
  return nve_b200::guarded([&] {
    NVE_B200_RANGE();
    nve_b200::rotary(rotary, dtype, head_width, num_tokens, groups, num_groups, backward != 0,
                     static_cast<cudaStream_t>(stream));
  });
}

nve_status_t nve_b200_kv_append(const nve_b200_kv_cache_t* cache, const nve_b200_kv_append_t* args, void* stream) {
  return nve_b200::guarded([&] {
    NVE_B200_RANGE();
    nve_b200::append(cache, args, static_cast<cudaStream_t>(stream));
  });
}

nve_status_t nve_b200_kv_attend(const nve_b200_kv_cache_t* cache, const nve_b200_kv_attend_t* args, void* scratch,
                                size_t* scratch_bytes, void* stream) {
  return nve_b200::guarded([&] {
    NVE_B200_RANGE();
    nve_b200::attend(cache, args, scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
  });
}

nve_status_t nve_b200_kv_evict(const nve_b200_kv_cache_t* cache, const nve_b200_kv_evict_t* args, void* stream) {
  return nve_b200::guarded([&] {
    NVE_B200_RANGE();
    nve_b200::evict(cache, args, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
