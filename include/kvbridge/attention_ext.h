#pragma once
// Additive extensions to the reference API (no counterpart in the reference's
// include/kvbridge): a caller-chosen split size, a fused merge + normalize
// step with fp16/fp32 output, and a single decode-attention call.  The
// reference entry points in attention_common.h are unchanged; these exist
// because the decode workloads ask for split counts other than
// end-begin / kSplitTokens and for a normalized fp16 output.
#include "kvbridge/attention_common.h"

namespace kvbridge {

// Output element type of the normalize step.
enum class OutputType : int { none = 0, f32 = 1, f16 = 2, bf16 = 3 };  // bf16: the calls on a 4- or 8-bit cache below

// Splits over [begin, end) when each split covers split_tokens tokens
// (max(1, ceil((end - begin) / split_tokens))).  Validates the shape first;
// throws std::invalid_argument for an invalid shape, split_tokens == 0 or more
// than 65535 splits.
unsigned split_count(const Shape&, unsigned split_tokens);
size_t scratch_elements(const Shape&, unsigned split_tokens);

// Split partials only (same scratch layout as launch_attention, with
// split_count(s, split_tokens) splits).
void launch_split_attention(const Shape&, const DeviceInput&, unsigned split_tokens,
                            float* scratch, hipStream_t stream);

// LSE merge of `splits` partials into m/l/n, and when out_type != none also
// out[rh * dim + d] = l > 0 ? n / l : 0 as fp32 or fp16 (the normalized
// attention output; the zero row is the empty-row convention).
void merge_finalize_attention(const Shape&, const float* scratch, unsigned splits,
                              float* m, float* l, float* n, void* out,
                              OutputType out_type, hipStream_t stream);

// launch_split_attention followed by merge_finalize_attention on one stream.
void decode_attention(const Shape&, const DeviceInput&, unsigned split_tokens,
                      float* scratch, float* m, float* l, float* n, void* out,
                      OutputType out_type, hipStream_t stream);

// ---- batched ragged decode: many independent sequences over one paged pool.
// Sequence b has `rows` query rows (q_heads heads each, sharing its KV) that
// attend to its own tokens [0, T_b): T_b = seq_starts[b+1] - seq_starts[b],
// its key positions are k_positions[seq_starts[b] ..], and its logical page
// p is physical page page_table[page_offsets[b] + p] of the shared pool.
// Each sequence runs max(1, ceil(T_b / split_tokens)) splits; the partial
// stride per sequence is batch_split_count (the split count of max_tokens),
// and splits past a sequence's own count hold empty partials (two-launch
// path; the single launch leaves them untouched and packs its own partials
// in an internal layout of the same size).  The device
// metadata is read by the kernels (the call is graph-capturable with
// changing lengths); indices are clamped to total_tokens / table_entries and
// T_b to max_tokens, so a malformed batch cannot read out of bounds.
struct BatchShape {
  unsigned batch, rows, q_heads, kv_heads, dim, page_tokens, pages;
  unsigned max_tokens;     // bound on every T_b: sizes the grid and the scratch
  unsigned total_tokens;   // k_positions entries
  unsigned table_entries;  // page_table entries
  unsigned split_tokens;   // tokens per split
  float scale;
  bool int8;
};

struct BatchInput {
  const float* q;               // [batch][rows][q_heads][dim]
  const int64_t* q_positions;   // [batch][rows]
  const uint32_t* seq_starts;   // [batch + 1], nondecreasing
  const uint32_t* page_offsets; // [batch]
  const int64_t* k_positions;   // [total_tokens], nondecreasing within a sequence
  const uint32_t* page_table;   // [table_entries]
  const void* k;                // shared pool, layouts as DeviceInput
  const void* v;
  const float* k_scales;
  const float* v_scales;
};

// nullptr when valid, else the first failed rule (never throws).
const char* batch_shape_error(const BatchShape&) noexcept;
// Partial stride per sequence (split count of max_tokens); validates.
unsigned batch_split_count(const BatchShape&);
// batch * rows * q_heads * batch_split_count * (dim + 2) floats; validates.
size_t batch_scratch_elements(const BatchShape&);
// batch * rows * q_heads (m, l); times dim for n and out; validates.
size_t batch_output_scalar_elements(const BatchShape&);

// Split partials + LSE merge (+ normalized output) of every sequence.  With
// counters (batch * kv_heads uint32, zero before the first call and left
// zero) the int8-MFMA kernel serves the whole call in one launch where it
// supports the shape; with counters == nullptr, or otherwise, split and merge
// run as two launches.
void decode_attention_batched(const BatchShape&, const BatchInput&, float* scratch,
                              uint32_t* counters, float* m, float* l, float* n, void* out,
                              OutputType out_type, hipStream_t stream);

// ---- paged INT8 KV append: the write side of the cache layout.
// New token t, kv head h: the rows k_new / v_new[t * stride + h * dim + d]
// (fp32, fp16 or bf16) are quantized with scale = absmax / 127 (1 for an
// all-zero row) and code = clamp(rint(x / scale), -127, 127) in IEEE fp32,
// and stored at physical slot slots[t] (page = slot / page_tokens): K
// token-major, V dim-major, scales per (page, kv head, slot).  slots is a
// device array; ids >= pages * page_tokens are skipped.
enum class SourceType : int { f32 = 1, f16 = 2, bf16 = 3 };

struct AppendShape {
  unsigned tokens, kv_heads, dim, page_tokens, pages;
  unsigned k_stride, v_stride;  // elements between consecutive new tokens (>= kv_heads * dim)
  SourceType src_type;
};

// Throws std::invalid_argument for an invalid shape or null buffers,
// std::runtime_error for a launch failure.  Asynchronous on `stream`.
void append_kv(const AppendShape&, const void* k_new, const void* v_new, const uint32_t* slots, int8_t* k,
               int8_t* v, float* k_scales, float* v_scales, hipStream_t stream);

// ---- 4-bit cache, score forms and eviction.  Formats, formulas, buffers and
// what the calls may share: include/kvbridge_c.h.  Every call throws
// std::invalid_argument for an invalid shape or buffer before anything is
// enqueued, std::runtime_error for a launch failure, and is asynchronous on
// `stream`; the *_error functions return nullptr when valid and never throw.

// Quantizes new tokens' rows into their slots of a 4-bit pool (blocks of 32
// dims, bfloat16 step and least value).  The shape is append_kv's.
const char* append_i4_error(const AppendShape&) noexcept;
void append_kv_i4(const AppendShape&, const void* k_new, const void* v_new, const uint32_t* slots, uint8_t* k,
                  uint8_t* v, uint32_t* k_scales, uint32_t* v_scales, hipStream_t stream);

// The rows of `slots` as values, k_out / v_out[(t * kv_heads + kv) * dim + d].
struct ReadShape {
  unsigned tokens, kv_heads, dim, page_tokens, pages;
  unsigned kv_bits;  // 4 or 8
  OutputType out_type;
};
const char* read_shape_error(const ReadShape&) noexcept;
void read_kv(const ReadShape&, const uint32_t* slots, const void* k, const void* v, const void* k_scales,
             const void* v_scales, void* k_out, void* v_out, hipStream_t stream);

// Ragged decode attention under score forms: tanh cap, bias by distance, window,
// prefix.
struct ScoredShape {
  unsigned batch, rows, q_heads, kv_heads, dim, page_tokens, pages;
  unsigned max_tokens, total_tokens, table_entries;  // as BatchShape
  unsigned split_tokens;  // a multiple of 32, or 0: the library's choice
  unsigned kv_bits;       // 4 or 8
  SourceType q_type;
  unsigned q_stride;      // elements from one query row to the next
  unsigned window;        // 0: none
  float scale, cap;       // cap 0: none
};
struct ScoredInput {
  const void* q;                // [batch][rows][q_stride]
  const int64_t* q_positions;   // [batch][rows]
  const uint32_t* seq_starts;   // [batch + 1]
  const uint32_t* page_offsets; // [batch]
  const int64_t* k_positions;   // [total_tokens]
  const uint32_t* page_table;   // [table_entries]
  const void* k;
  const void* v;
  const void* k_scales;
  const void* v_scales;
  const float* slopes;          // [q_heads] or nullptr
  const int64_t* prefix;        // [batch] or nullptr
};
const char* scored_shape_error(const ScoredShape&) noexcept;
unsigned scored_item_count(const ScoredShape&);       // validate
size_t scored_scratch_elements(const ScoredShape&);   // floats
size_t scored_counter_elements(const ScoredShape&);   // uint32, zero before the first call and left zero
void decode_attention_scored(const ScoredShape&, const ScoredInput&, float* scratch, uint32_t* counters, float* m,
                             float* l, void* out, OutputType out_type, hipStream_t stream);

// weights[(page * kv_heads + kv) * page_tokens + slot] += the token's share of
// the attention with these m and l; the last `fresh` tokens are set.
void accumulate_weights(const ScoredShape&, const ScoredInput&, const float* m, const float* l, unsigned fresh,
                        float* weights, hipStream_t stream);

// Which tokens stay (select), and packing them into other pages (move).
struct EvictShape {
  unsigned batch, kv_heads, dim, page_tokens, pages;
  unsigned max_tokens, total_tokens, table_entries, dst_entries;
  unsigned keep, sink, recent, kv_bits;
};
struct EvictInput {
  const uint32_t* seq_starts;
  const uint32_t* page_offsets;
  const uint32_t* page_table;
  const int64_t* k_positions;  // nullptr where no positions are moved
};
struct EvictCache {
  void* k;
  void* v;
  void* k_scales;
  void* v_scales;
  float* weights;               // or nullptr
  const uint32_t* dst_offsets;  // [batch]
  const uint32_t* dst_table;    // [dst_entries]
  int64_t* positions;           // [batch * keep] or nullptr
};
const char* evict_shape_error(const EvictShape&) noexcept;
size_t evict_scratch_elements(const EvictShape&);  // uint32
void evict_select(const EvictShape&, const EvictInput&, const float* weights, uint32_t* scratch, uint32_t* kept,
                  uint32_t* kept_starts, hipStream_t stream);
void evict_move(const EvictShape&, const EvictInput&, const EvictCache&, const uint32_t* kept,
                const uint32_t* kept_starts, hipStream_t stream);

}  // namespace kvbridge
