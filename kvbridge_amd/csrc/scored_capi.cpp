// extern "C" entry points of the calls on a 4- or 8-bit cache
// (include/kvbridge_c.h): argument checks, sizes and launches.  As in capi.cpp
// no exception crosses the boundary and nothing is enqueued before every check
// has passed.
#include <hip/hip_runtime.h>

#include <exception>
#include <string>

#include "kernels.h"
#include "kvbridge_c.h"
#include "scored_args.h"
#include "scored_shape.h"

namespace {

template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return kvb::set_error(KVB_ERUNTIME, e.what());
  } catch (...) {
    return kvb::set_error(KVB_ERUNTIME, "unknown error");
  }
}

int invalid(const char* msg) { return kvb::set_error(KVB_EINVAL, msg); }

int status(hipError_t e, const char* op) {
  return e == hipSuccess ? KVB_OK : kvb::set_error(KVB_ERUNTIME, std::string(op) + ": " + hipGetErrorString(e));
}

bool off16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }
uintptr_t source_bytes(uint32_t type) { return type == KVB_SRC_F32 ? 4 : 2; }

// Cache buffers: every row is a whole number of 8- or 16-byte pieces from the
// pool's start (int8 scales: single floats).
const char* cache_buffers_error(const void* k, const void* v, const void* ks, const void* vs, uint32_t bits) {
  if (!k || !v || !ks || !vs) return "cache buffers must be non-null";
  if (off16(k) || off16(v)) return "cache K and V buffers must be 16-byte aligned";
  const uintptr_t al = bits == 4 ? 16 : 4;
  if (reinterpret_cast<uintptr_t>(ks) % al || reinterpret_cast<uintptr_t>(vs) % al)
    return "cache scales must be aligned to 16 bytes (4-bit) or 4 bytes (8-bit)";
  return nullptr;
}

const char* scored_input_error(const kvb_scored_shape& s, const kvb_scored_input& in, bool values) {
  if (!in.q || !in.q_positions || !in.seq_starts || !in.page_offsets || !in.k_positions || !in.page_table)
    return "attention input device buffers must be non-null";
  if (reinterpret_cast<uintptr_t>(in.q) % source_bytes(s.q_type)) return "query rows must be aligned to their element size";
  return cache_buffers_error(in.k, values ? in.v : in.k, in.k_scales, values ? in.v_scales : in.k_scales, s.kv_bits);
}

kvb::ScoredArgs scored_args(const kvb_scored_shape& s, const kvb_scored_input& in) {
  kvb::ScoredArgs a{};
  a.q = in.q;
  a.q_positions = in.q_positions;
  a.seq_starts = in.seq_starts;
  a.page_offsets = in.page_offsets;
  a.k_positions = in.k_positions;
  a.page_table = in.page_table;
  a.k = in.k;
  a.v = in.v;
  a.ks = in.k_scales;
  a.vs = in.v_scales;
  a.slopes = in.slopes;
  a.prefix = in.prefix;
  a.batch = s.batch;
  a.rows = s.rows;
  a.q_heads = s.q_heads;
  a.kv_heads = s.kv_heads;
  a.group = s.q_heads / s.kv_heads;
  a.head_rows = s.rows * a.group;
  a.blocks = kvb::scored_blocks(s);
  a.dim = s.dim;
  a.page_tokens = s.page_tokens;
  a.pages = s.pages;
  a.max_tokens = s.max_tokens;
  a.total_tokens = s.total_tokens;
  a.table_entries = s.table_entries;
  a.q_stride = s.q_stride;
  a.q_type = s.q_type;
  a.window = s.window;
  a.kv_bits = s.kv_bits;
  a.scale = s.scale;
  a.cap = s.cap;
  return a;
}

template <class T, class F>
int sized(const kvb_scored_shape* s, T* out, F&& f) {
  return guarded([&]() -> int {
    if (!s || !out) return invalid("shape and output pointers must be non-null");
    if (const char* e = kvb::scored_error(*s)) return invalid(e);
    *out = f(*s);
    return KVB_OK;
  });
}

const char* kNullShape = "shape pointer must be non-null";

uint32_t key_stride(const kvb_evict_shape& s) { return (s.max_tokens + 3) / 4 * 4; }

kvb::EvictArgs evict_args(const kvb_evict_shape& s, const kvb_evict_input& in) {
  kvb::EvictArgs a{};
  a.seq_starts = in.seq_starts;
  a.page_offsets = in.page_offsets;
  a.page_table = in.page_table;
  a.k_positions = in.k_positions;
  a.batch = s.batch;
  a.kv_heads = s.kv_heads;
  a.dim = s.dim;
  a.page_tokens = s.page_tokens;
  a.pages = s.pages;
  a.max_tokens = s.max_tokens;
  a.total_tokens = s.total_tokens;
  a.table_entries = s.table_entries;
  a.dst_entries = s.dst_entries;
  a.keep = s.keep;
  a.sink = s.sink;
  a.recent = s.recent;
  a.kv_bits = s.kv_bits;
  a.scratch_stride = key_stride(s);
  return a;
}

}  // namespace

extern "C" {

const char* kvb_append_i4_shape_error(const kvb_append_shape* s) { return s ? kvb::append4_error(*s) : kNullShape; }

int kvb_append_kv_i4(const kvb_append_shape* s, const kvb_append_i4_io* io, void* stream) {
  return guarded([&]() -> int {
    if (!s || !io) return invalid("shape and buffer descriptors must be non-null");
    if (const char* e = kvb::append4_error(*s)) return invalid(e);
    if (s->tokens == 0) return KVB_OK;
    if (!io->k_new || !io->v_new || !io->slots) return invalid("append buffers must be non-null");
    if (const char* e = cache_buffers_error(io->k, io->v, io->k_scales, io->v_scales, 4)) return invalid(e);
    const uintptr_t el = source_bytes(s->src_type);
    if (reinterpret_cast<uintptr_t>(io->k_new) % el || reinterpret_cast<uintptr_t>(io->v_new) % el)
      return invalid("source rows must be aligned to their element size");
    const kvb::Append4Args a{io->k_new,    io->v_new,   io->slots, io->k,          io->v,    io->k_scales,
                             io->v_scales, s->tokens,   s->kv_heads, s->dim,       s->page_tokens,
                             s->pages,     s->k_stride, s->v_stride, s->src_type};
    return status(kvb::launch_append4(a, static_cast<hipStream_t>(stream)), "4-bit kv append launch");
  });
}

const char* kvb_read_shape_error(const kvb_read_shape* s) { return s ? kvb::read_error(*s) : kNullShape; }

int kvb_read_kv(const kvb_read_shape* s, const kvb_read_io* io, void* stream) {
  return guarded([&]() -> int {
    if (!s || !io) return invalid("shape and buffer descriptors must be non-null");
    if (const char* e = kvb::read_error(*s)) return invalid(e);
    if (s->tokens == 0) return KVB_OK;
    if (!io->slots || !io->k_out || !io->v_out) return invalid("read buffers must be non-null");
    if (const char* e = cache_buffers_error(io->k, io->v, io->k_scales, io->v_scales, s->kv_bits)) return invalid(e);
    if (off16(io->k_out) || off16(io->v_out)) return invalid("output rows must be 16-byte aligned");
    const kvb::ReadArgs a{io->slots, io->k,      io->v,       io->k_scales, io->v_scales,   io->k_out, io->v_out,
                          s->tokens, s->kv_heads, s->dim,     s->page_tokens, s->pages,     s->kv_bits, s->out_type};
    return status(kvb::launch_read(a, static_cast<hipStream_t>(stream)), "kv read launch");
  });
}

const char* kvb_scored_shape_error(const kvb_scored_shape* s) { return s ? kvb::scored_error(*s) : kNullShape; }

int kvb_scored_item_count(const kvb_scored_shape* s, uint32_t* items) {
  return sized(s, items, [](const kvb_scored_shape& x) { return kvb::scored_splits(x).items; });
}

int kvb_scored_scratch_elements(const kvb_scored_shape* s, size_t* elements) {
  return sized(s, elements, [](const kvb_scored_shape& x) {
    return size_t(kvb::scored_splits(x).items) * x.rows * x.q_heads * (size_t(x.dim) + 2);
  });
}

int kvb_scored_counter_elements(const kvb_scored_shape* s, size_t* elements) {
  return sized(s, elements, [](const kvb_scored_shape& x) { return size_t(x.batch) * x.kv_heads * kvb::scored_blocks(x); });
}

int kvb_decode_attention_scored(const kvb_scored_shape* s, const kvb_scored_input* in, float* scratch,
                                uint32_t* counters, float* m, float* l, void* out, int out_type, void* stream) {
  return guarded([&]() -> int {
    if (!s || !in) return invalid("shape and input descriptors must be non-null");
    if (const char* e = kvb::scored_error(*s)) return invalid(e);
    if (!scratch || !m || !l || !out) return invalid("scratch, m, l and out must be non-null device buffers");
    if (const char* e = scored_input_error(*s, *in, true)) return invalid(e);
    if (out_type != KVB_OUT_F32 && out_type != KVB_OUT_F16 && out_type != KVB_OUT_BF16) return invalid("unknown output type");
    if (off16(out) || off16(scratch)) return invalid("scratch and out must be 16-byte aligned");
    kvb::ScoredArgs a = scored_args(*s, *in);
    const kvb::ScoredSplits p = kvb::scored_splits(*s);
    a.items = p.items;
    a.splits = p.splits;
    a.split_tiles = p.tiles;
    a.alone_tiles = p.alone;
    a.waves = p.waves;
    a.scratch = scratch;
    a.counters = kvb::scored_one_launch(*s, p) ? counters : nullptr;
    a.m = m;
    a.l = l;
    a.out = out;
    a.out_type = uint32_t(out_type);
    return status(kvb::launch_scored_attend(a, static_cast<hipStream_t>(stream)), "scored attention launch");
  });
}

int kvb_accumulate_weights(const kvb_scored_shape* s, const kvb_scored_input* in, const float* m, const float* l,
                           uint32_t fresh, float* weights, void* stream) {
  return guarded([&]() -> int {
    if (!s || !in) return invalid("shape and input descriptors must be non-null");
    if (const char* e = kvb::scored_error(*s)) return invalid(e);
    if (!m || !l || !weights) return invalid("m, l and weights must be non-null device buffers");
    if (const char* e = scored_input_error(*s, *in, false)) return invalid(e);
    kvb::ScoredArgs a = scored_args(*s, *in);
    const kvb::ScoredSplits p = kvb::weight_splits(*s);
    a.items = p.items;
    a.splits = p.splits;
    a.split_tiles = p.tiles;
    a.waves = p.waves;
    a.m = const_cast<float*>(m);
    a.l = const_cast<float*>(l);
    a.weights = weights;
    a.fresh = fresh;
    return status(kvb::launch_scored_weights(a, static_cast<hipStream_t>(stream)), "weight accumulation launch");
  });
}

const char* kvb_evict_shape_error(const kvb_evict_shape* s) { return s ? kvb::evict_error(*s) : kNullShape; }

int kvb_evict_scratch_elements(const kvb_evict_shape* s, size_t* elements) {
  return guarded([&]() -> int {
    if (!s || !elements) return invalid("shape and output pointers must be non-null");
    if (const char* e = kvb::evict_error(*s)) return invalid(e);
    *elements = size_t(s->batch) * key_stride(*s);
    return KVB_OK;
  });
}

int kvb_evict_select(const kvb_evict_shape* s, const kvb_evict_input* in, const float* weights, uint32_t* scratch,
                     uint32_t* kept, uint32_t* kept_starts, void* stream) {
  return guarded([&]() -> int {
    if (!s || !in) return invalid("shape and input descriptors must be non-null");
    if (const char* e = kvb::evict_error(*s)) return invalid(e);
    if (!in->seq_starts || !in->page_offsets || !in->page_table || !weights || !scratch || !kept || !kept_starts)
      return invalid("eviction buffers must be non-null");
    if (off16(scratch)) return invalid("eviction scratch must be 16-byte aligned");
    kvb::EvictArgs a = evict_args(*s, *in);
    a.weights_in = weights;
    a.scratch = scratch;
    a.kept = kept;
    a.kept_starts = kept_starts;
    return status(kvb::launch_evict_select(a, static_cast<hipStream_t>(stream)), "eviction selection launch");
  });
}

int kvb_evict_move(const kvb_evict_shape* s, const kvb_evict_input* in, const kvb_evict_cache* c, const uint32_t* kept,
                   const uint32_t* kept_starts, void* stream) {
  return guarded([&]() -> int {
    if (!s || !in || !c) return invalid("shape, input and cache descriptors must be non-null");
    if (const char* e = kvb::evict_error(*s)) return invalid(e);
    if (!in->seq_starts || !in->page_offsets || !in->page_table || !kept || !kept_starts || !c->dst_offsets || !c->dst_table)
      return invalid("eviction buffers must be non-null");
    if (c->positions && !in->k_positions) return invalid("positions need k_positions");
    if (const char* e = cache_buffers_error(c->k, c->v, c->k_scales, c->v_scales, s->kv_bits)) return invalid(e);
    kvb::EvictArgs a = evict_args(*s, *in);
    a.kept = const_cast<uint32_t*>(kept);
    a.kept_starts = const_cast<uint32_t*>(kept_starts);
    a.k = c->k;
    a.v = c->v;
    a.k_scales = c->k_scales;
    a.v_scales = c->v_scales;
    a.weights = c->weights;
    a.dst_offsets = c->dst_offsets;
    a.dst_table = c->dst_table;
    a.positions = c->positions;
    return status(kvb::launch_evict_move(a, static_cast<hipStream_t>(stream)), "eviction move launch");
  });
}

}  // extern "C"
