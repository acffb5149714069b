// C++ API (include/kvbridge/attention_common.h, attention_ext.h) as a thin
// layer over the extern "C" entry points.  Status codes become the
// reference's exception types: KVB_EINVAL -> std::invalid_argument,
// KVB_ERUNTIME -> std::runtime_error (reference src/attention_launch_checks.h:8-27).
#include <stdexcept>

#include "kvbridge/attention_ext.h"
#include "kvbridge_c.h"

namespace kvbridge {
namespace {

kvb_shape c_shape(const Shape& s) {
  return kvb_shape{s.rows, s.q_heads, s.kv_heads, s.dim, s.page_tokens, s.pages,
                   s.tokens, s.begin, s.end, s.scale, s.int8 ? 1u : 0u};
}

kvb_device_input c_input(const DeviceInput& in) {
  return kvb_device_input{in.q, in.q_positions, in.k_positions, in.page_table,
                          in.k, in.v, in.k_scales, in.v_scales};
}

void check(int rc) {
  if (rc == KVB_OK) return;
  if (rc == KVB_EINVAL) throw std::invalid_argument(kvb_last_error());
  throw std::runtime_error(kvb_last_error());
}

kvb_append_shape c_append(const AppendShape& a) {
  return kvb_append_shape{a.tokens,   a.kv_heads, a.dim,      a.page_tokens,
                          a.pages,    a.k_stride, a.v_stride, uint32_t(a.src_type)};
}

kvb_read_shape c_read(const ReadShape& r) {
  return kvb_read_shape{r.tokens, r.kv_heads, r.dim, r.page_tokens, r.pages, r.kv_bits, uint32_t(r.out_type)};
}

kvb_scored_shape c_scored(const ScoredShape& s) {
  return kvb_scored_shape{s.batch,      s.rows,         s.q_heads,       s.kv_heads,     s.dim,     s.page_tokens,
                          s.pages,      s.max_tokens,   s.total_tokens,  s.table_entries, s.split_tokens, s.kv_bits,
                          uint32_t(s.q_type), s.q_stride, s.window,      s.scale,        s.cap};
}

kvb_scored_input c_scored_input(const ScoredInput& in) {
  return kvb_scored_input{in.q, in.q_positions, in.seq_starts, in.page_offsets, in.k_positions, in.page_table,
                          in.k, in.v,           in.k_scales,   in.v_scales,     in.slopes,      in.prefix};
}

kvb_evict_shape c_evict(const EvictShape& e) {
  return kvb_evict_shape{e.batch,         e.kv_heads,    e.dim,  e.page_tokens, e.pages,  e.max_tokens, e.total_tokens,
                         e.table_entries, e.dst_entries, e.keep, e.sink,        e.recent, e.kv_bits};
}

kvb_evict_input c_evict_input(const EvictInput& in) {
  return kvb_evict_input{in.seq_starts, in.page_offsets, in.page_table, in.k_positions};
}

}  // namespace

hipError_t preload_attention_kernels() { return hipError_t(kvb_preload_attention_kernels()); }
hipError_t preload_attention_reference_kernels() {
  return hipError_t(kvb_preload_attention_reference_kernels());
}
hipError_t preload_attention_mma_kernels() { return hipError_t(kvb_preload_attention_mma_kernels()); }

void launch_attention(const Shape& s, const DeviceInput& in, float* scratch, float* m, float* l,
                      float* n, hipStream_t stream) {
  const kvb_shape cs = c_shape(s);
  const kvb_device_input ci = c_input(in);
  check(kvb_launch_attention(&cs, &ci, scratch, m, l, n, stream));
}

void launch_attention_mma(const Shape& s, const DeviceInput& in, float* scratch, float* m,
                          float* l, float* n, hipStream_t stream) {
  const kvb_shape cs = c_shape(s);
  const kvb_device_input ci = c_input(in);
  check(kvb_launch_attention_mma(&cs, &ci, scratch, m, l, n, stream));
}

void merge_attention(const Shape& s, const float* scratch, unsigned splits, float* m, float* l,
                     float* n, hipStream_t stream) {
  const kvb_shape cs = c_shape(s);
  check(kvb_merge_attention(&cs, scratch, splits, m, l, n, stream));
}

void launch_split_attention(const Shape& s, const DeviceInput& in, unsigned split_tokens,
                            float* scratch, hipStream_t stream) {
  const kvb_shape cs = c_shape(s);
  const kvb_device_input ci = c_input(in);
  check(kvb_split_attention(&cs, &ci, split_tokens, scratch, stream));
}

void merge_finalize_attention(const Shape& s, const float* scratch, unsigned splits, float* m,
                              float* l, float* n, void* out, OutputType out_type,
                              hipStream_t stream) {
  const kvb_shape cs = c_shape(s);
  check(kvb_merge_finalize(&cs, scratch, splits, m, l, n, out, int(out_type), stream));
}

void decode_attention(const Shape& s, const DeviceInput& in, unsigned split_tokens,
                      float* scratch, float* m, float* l, float* n, void* out,
                      OutputType out_type, hipStream_t stream) {
  const kvb_shape cs = c_shape(s);
  const kvb_device_input ci = c_input(in);
  check(kvb_decode_attention(&cs, &ci, split_tokens, scratch, m, l, n, out, int(out_type), stream));
}

void decode_attention_batched(const BatchShape& b, const BatchInput& in, float* scratch, uint32_t* counters,
                              float* m, float* l, float* n, void* out, OutputType out_type, hipStream_t stream) {
  const kvb_batch_shape cs{b.batch,      b.rows,         b.q_heads,      b.kv_heads,     b.dim,
                           b.page_tokens, b.pages,        b.max_tokens,   b.total_tokens, b.table_entries,
                           b.split_tokens, b.scale,       b.int8 ? 1u : 0u};
  const kvb_batch_input ci{in.q,          in.q_positions, in.seq_starts, in.page_offsets, in.k_positions,
                           in.page_table, in.k,           in.v,          in.k_scales,     in.v_scales};
  check(kvb_decode_attention_batched(&cs, &ci, scratch, counters, m, l, n, out, int(out_type), stream));
}

void append_kv(const AppendShape& a, const void* k_new, const void* v_new, const uint32_t* slots, int8_t* k,
               int8_t* v, float* k_scales, float* v_scales, hipStream_t stream) {
  const kvb_append_shape cs = c_append(a);
  const kvb_append_io io{k_new, v_new, slots, k, v, k_scales, v_scales};
  check(kvb_append_kv(&cs, &io, stream));
}

const char* append_i4_error(const AppendShape& a) noexcept {
  const kvb_append_shape cs = c_append(a);
  return kvb_append_i4_shape_error(&cs);
}

void append_kv_i4(const AppendShape& a, const void* k_new, const void* v_new, const uint32_t* slots, uint8_t* k,
                  uint8_t* v, uint32_t* k_scales, uint32_t* v_scales, hipStream_t stream) {
  const kvb_append_shape cs = c_append(a);
  const kvb_append_i4_io io{k_new, v_new, slots, k, v, k_scales, v_scales};
  check(kvb_append_kv_i4(&cs, &io, stream));
}

const char* read_shape_error(const ReadShape& r) noexcept {
  const kvb_read_shape cs = c_read(r);
  return kvb_read_shape_error(&cs);
}

void read_kv(const ReadShape& r, const uint32_t* slots, const void* k, const void* v, const void* k_scales,
             const void* v_scales, void* k_out, void* v_out, hipStream_t stream) {
  const kvb_read_shape cs = c_read(r);
  const kvb_read_io io{slots, k, v, k_scales, v_scales, k_out, v_out};
  check(kvb_read_kv(&cs, &io, stream));
}

const char* scored_shape_error(const ScoredShape& s) noexcept {
  const kvb_scored_shape cs = c_scored(s);
  return kvb_scored_shape_error(&cs);
}

unsigned scored_item_count(const ScoredShape& s) {
  const kvb_scored_shape cs = c_scored(s);
  uint32_t items = 0;
  check(kvb_scored_item_count(&cs, &items));
  return items;
}

size_t scored_scratch_elements(const ScoredShape& s) {
  const kvb_scored_shape cs = c_scored(s);
  size_t n = 0;
  check(kvb_scored_scratch_elements(&cs, &n));
  return n;
}

size_t scored_counter_elements(const ScoredShape& s) {
  const kvb_scored_shape cs = c_scored(s);
  size_t n = 0;
  check(kvb_scored_counter_elements(&cs, &n));
  return n;
}

void decode_attention_scored(const ScoredShape& s, const ScoredInput& in, float* scratch, uint32_t* counters, float* m,
                             float* l, void* out, OutputType out_type, hipStream_t stream) {
  const kvb_scored_shape cs = c_scored(s);
  const kvb_scored_input ci = c_scored_input(in);
  check(kvb_decode_attention_scored(&cs, &ci, scratch, counters, m, l, out, int(out_type), stream));
}

void accumulate_weights(const ScoredShape& s, const ScoredInput& in, const float* m, const float* l, unsigned fresh,
                        float* weights, hipStream_t stream) {
  const kvb_scored_shape cs = c_scored(s);
  const kvb_scored_input ci = c_scored_input(in);
  check(kvb_accumulate_weights(&cs, &ci, m, l, fresh, weights, stream));
}

const char* evict_shape_error(const EvictShape& e) noexcept {
  const kvb_evict_shape cs = c_evict(e);
  return kvb_evict_shape_error(&cs);
}

size_t evict_scratch_elements(const EvictShape& e) {
  const kvb_evict_shape cs = c_evict(e);
  size_t n = 0;
  check(kvb_evict_scratch_elements(&cs, &n));
  return n;
}

void evict_select(const EvictShape& e, const EvictInput& in, const float* weights, uint32_t* scratch, uint32_t* kept,
                  uint32_t* kept_starts, hipStream_t stream) {
  const kvb_evict_shape cs = c_evict(e);
  const kvb_evict_input ci = c_evict_input(in);
  check(kvb_evict_select(&cs, &ci, weights, scratch, kept, kept_starts, stream));
}

void evict_move(const EvictShape& e, const EvictInput& in, const EvictCache& c, const uint32_t* kept,
                const uint32_t* kept_starts, hipStream_t stream) {
  const kvb_evict_shape cs = c_evict(e);
  const kvb_evict_input ci = c_evict_input(in);
  const kvb_evict_cache cc{c.k, c.v, c.k_scales, c.v_scales, c.weights, c.dst_offsets, c.dst_table, c.positions};
  check(kvb_evict_move(&cs, &ci, &cc, kept, kept_starts, stream));
}

}  // namespace kvbridge
