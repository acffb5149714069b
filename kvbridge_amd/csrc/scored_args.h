// Arguments of the scored attention, weight and eviction launchers, shared by
// the entry points (scored_capi.cpp) and the kernels.  Shapes reaching the
// launchers are already validated.
#pragma once
#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace kvb {

struct ScoredArgs {
  const void* q;
  const int64_t* q_positions;
  const uint32_t* seq_starts;
  const uint32_t* page_offsets;
  const int64_t* k_positions;
  const uint32_t* page_table;
  const void* k;
  const void* v;
  const void* ks;
  const void* vs;
  const float* slopes;
  const int64_t* prefix;
  float* scratch;
  uint32_t* counters;
  float* m;
  float* l;
  void* out;
  uint32_t batch, rows, q_heads, kv_heads, group, head_rows, blocks;  // blocks of 16 head-rows per kv head
  uint32_t dim, page_tokens, pages, max_tokens, total_tokens, table_entries;
  uint32_t items, splits, split_tiles;  // work items per kv head and block, items per sequence (0: shared out), least tiles of one
  uint32_t alone_tiles;  // up to so many tiles a sequence is not split
  uint32_t waves;  // of an attention work-group, at most (4, or all that a CU holds)
  uint32_t q_stride, q_type, out_type, window, kv_bits;
  float scale, cap;
  float* weights;
  uint32_t fresh;
};

// Load the code objects of all these calls.
hipError_t preload_scored();
hipError_t preload_scored_weights();
hipError_t preload_cache4();
hipError_t preload_evict();

hipError_t launch_scored_attend(const ScoredArgs& a, hipStream_t stream);
hipError_t launch_scored_weights(const ScoredArgs& a, hipStream_t stream);

struct Append4Args {
  const void* k_new;
  const void* v_new;
  const uint32_t* slots;
  uint8_t* k;
  uint8_t* v;
  uint32_t* k_scales;
  uint32_t* v_scales;
  uint32_t tokens, kv_heads, dim, page_tokens, pages, k_stride, v_stride, src_type;
};
hipError_t launch_append4(const Append4Args& a, hipStream_t stream);

struct ReadArgs {
  const uint32_t* slots;
  const void* k;
  const void* v;
  const void* k_scales;
  const void* v_scales;
  void* k_out;
  void* v_out;
  uint32_t tokens, kv_heads, dim, page_tokens, pages, kv_bits, out_type;
};
hipError_t launch_read(const ReadArgs& a, hipStream_t stream);

struct EvictArgs {
  const uint32_t* seq_starts;
  const uint32_t* page_offsets;
  const uint32_t* page_table;
  const int64_t* k_positions;
  const float* weights_in;
  uint32_t* scratch;
  uint32_t* kept;
  uint32_t* kept_starts;
  void* k;
  void* v;
  void* k_scales;
  void* v_scales;
  float* weights;
  const uint32_t* dst_offsets;
  const uint32_t* dst_table;
  int64_t* positions;
  uint32_t batch, kv_heads, dim, page_tokens, pages, max_tokens, total_tokens, table_entries, dst_entries;
  uint32_t keep, sink, recent, kv_bits;
  uint32_t scratch_stride;  // keys of a sequence, a multiple of 4
};
hipError_t launch_evict_select(const EvictArgs& a, hipStream_t stream);
hipError_t launch_evict_move(const EvictArgs& a, hipStream_t stream);

}  // namespace kvb
