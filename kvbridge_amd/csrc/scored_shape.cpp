// Validation and sizing of the calls on a 4- or 8-bit cache (host only, no
// HIP): the writer and reader, the scored attention and weights, eviction.
#include "scored_shape.h"

#include <cmath>
#include <limits>

namespace kvb {
namespace {

// Threads of a grid dimension are counted in 32 bits; work-groups of 256 threads.
constexpr uint64_t kMaxGroups = (uint64_t(1) << 24) - 1;

const char* cache_error(uint32_t kv_heads, uint32_t dim, uint32_t page_tokens, uint32_t pages, uint32_t kv_bits) {
  if (kv_bits != 4 && kv_bits != 8) return "kv_bits must be 4 or 8";
  if (dim != 64 && dim != 128 && dim != 256) return "dim must be 64, 128 or 256";
  if (page_tokens == 0 || page_tokens % 8 != 0) return "page_tokens must be a positive multiple of 8";
  if (pages == 0) return "pages must be positive";
  if (kv_heads == 0 || kv_heads > 65535) return "kv_heads must be in [1,65535]";
  if (uint64_t(pages) * kv_heads > 0xffffffffull) return "page and kv head product exceeds 32 bits";
  return nullptr;
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

}  // namespace

const char* append4_error(const kvb_append_shape& s) {
  if (const char* e = cache_error(s.kv_heads, s.dim, s.page_tokens, s.pages, 4)) return e;
  if (s.src_type != KVB_SRC_F32 && s.src_type != KVB_SRC_F16 && s.src_type != KVB_SRC_BF16)
    return "unknown source element type";
  if (uint64_t(s.k_stride) < uint64_t(s.kv_heads) * s.dim || uint64_t(s.v_stride) < uint64_t(s.kv_heads) * s.dim)
    return "token stride must cover kv_heads * dim elements";
  if ((uint64_t(s.tokens) * s.kv_heads + 63) / 64 > kMaxGroups) return "token and kv head product exceeds the grid limit";
  return nullptr;
}

const char* read_error(const kvb_read_shape& s) {
  if (const char* e = cache_error(s.kv_heads, s.dim, s.page_tokens, s.pages, s.kv_bits)) return e;
  if (s.out_type != KVB_OUT_F32 && s.out_type != KVB_OUT_F16 && s.out_type != KVB_OUT_BF16) return "unknown output type";
  if ((uint64_t(s.tokens) * s.kv_heads + 63) / 64 > kMaxGroups) return "token and kv head product exceeds the grid limit";
  return nullptr;
}

uint32_t scored_blocks(const kvb_scored_shape& s) { return ceil_div(uint64_t(s.rows) * (s.q_heads / s.kv_heads), 16); }

namespace {

constexpr uint64_t kCus = 256;

// Waves of the attention kernel that a CU holds (kAttendOccupancy in
// scored_attend.h).  One more wave per SIMD with spills inside the tile loop cost
// a third to a half (16 ragged sequences 78 -> 160 us, four of 128K 186 -> 266).
uint32_t resident_waves(const kvb_scored_shape& s) {
  const uint64_t head_rows = uint64_t(s.rows) * (s.q_heads / s.kv_heads), blocks = s.dim / 32;
  const bool half = s.kv_bits == 4 && s.dim > 128 && head_rows > 16 / blocks && head_rows <= 32 / blocks;
  return s.dim == 256 || half || (s.kv_bits == 8 && s.page_tokens % 32 != 0) ? 8 : 12;
}

// Work items; others: kv heads times blocks.  Where the caller names no split size, there are as many as fit
// the GPU at once and the kernel shares them out over the sequences by length
// (scored.h, item_of): every work-group then has about the same number of tiles
// and pays for its start and end once.  An item is a whole CU's unless the
// sequences are so many that rounding to whole items would idle over a
// sixteenth of them; then work-groups have four waves.
ScoredSplits split_items(const kvb_scored_shape& s, uint64_t others, uint32_t split_tokens) {
  const uint64_t seen = s.window == 0 ? s.max_tokens
                                      : std::min<uint64_t>(s.max_tokens, uint64_t(s.window) + s.rows + 32);
  const uint64_t tiles = (seen + 31) / 32;
  const uint32_t all = resident_waves(s);
  const uint32_t waves = s.batch * 8 <= std::max<uint64_t>(8, kCus / others) ? all : 4;
  const uint64_t resident = kCus * (all / waves);
  if (split_tokens != 0 || s.batch > 256) {
    uint64_t per = split_tokens / 32;
    if (per == 0) {
      const uint64_t splits = std::max<uint64_t>(1, resident * 2 / (others * s.batch));
      per = std::max<uint64_t>(16, (tiles + splits - 1) / splits);
    }
    const uint64_t splits = std::max<uint64_t>(1, (tiles + per - 1) / per);
    return ScoredSplits{uint32_t(std::min<uint64_t>(s.batch * splits, 0xffffffffu)), uint32_t(std::min<uint64_t>(splits, 0xffffffffu)),
                        uint32_t(per), per < all ? 4u : waves, 0};
  }
  // A tile costs a SIMD 0.8 us at dim 64 and 128 (twice that at 256), so a CU
  // four of them; joining several parts costs about 3 us.
  const uint64_t least = s.dim == 256 ? 4 : 8, useful = s.batch * ((tiles + least - 1) / least);
  const uint64_t items = std::max<uint64_t>(s.batch, std::min(useful, resident / others));
  return ScoredSplits{uint32_t(items), s.batch == 1 ? uint32_t(items) : 0, uint32_t(least), waves, s.dim == 256 ? 10u : 20u};
}

}  // namespace

ScoredSplits scored_splits(const kvb_scored_shape& s) {
  return split_items(s, uint64_t(s.kv_heads) * scored_blocks(s), s.split_tokens);
}

// One work-group's merge reads the partials of its head-rows past its L2, a
// second launch spreads that over a work-group per head-row.  Measured (us, one
// launch against two) by the sets of four dims that a thread of the first has to
// add: 1 (int8, window, 32 sequences) 111 / 114, 3 (16 ragged ones) 78.7 / 79.6, 3
// (four of 128K, 64 heads) 115.5 / 115.3, 5 (one of 64K) 27.7 / 24.8, 21 (24 heads
// of 256 over 8 rows) 38.1 / 34.2.
bool scored_one_launch(const kvb_scored_shape& s, const ScoredSplits& p) {
  const uint64_t head_rows = std::min<uint64_t>(16, uint64_t(s.rows) * (s.q_heads / s.kv_heads));
  return p.items / s.batch * head_rows * (s.dim / 4) <= 3 * 64 * p.waves;
}

const char* scored_error(const kvb_scored_shape& s) {
  if (s.batch == 0 || s.batch > 65535) return "batch must be in [1,65535]";
  if (s.rows == 0 || s.q_heads == 0 || s.kv_heads == 0) return "rows and head counts must be positive";
  if (s.q_heads % s.kv_heads != 0) return "q_heads must be divisible by kv_heads";
  if (const char* e = cache_error(s.kv_heads, s.dim, s.page_tokens, s.pages, s.kv_bits)) return e;
  if (s.max_tokens == 0 || s.max_tokens > 0x7fffffffu) return "max_tokens must be in [1,2^31-1]";
  if (uint64_t(s.max_tokens) > uint64_t(s.pages) * s.page_tokens) return "tokens exceed allocated page capacity";
  if (s.total_tokens == 0 || s.table_entries == 0) return "total_tokens and table_entries must be positive";
  if (s.split_tokens % 32 != 0) return "split_tokens must be a multiple of 32";
  if (s.q_type != KVB_SRC_F32 && s.q_type != KVB_SRC_F16 && s.q_type != KVB_SRC_BF16) return "unknown query element type";
  if (uint64_t(s.q_stride) < uint64_t(s.q_heads) * s.dim) return "row stride must cover q_heads * dim elements";
  if (!std::isfinite(s.scale)) return "score scale must be finite";
  if (!std::isfinite(s.cap) || s.cap < 0.f) return "score cap must be finite and not negative";
  if (uint64_t(s.rows) * s.q_heads > kMaxGroups || uint64_t(s.batch) * s.rows * s.q_heads > kMaxGroups)
    return "batch row/head product exceeds the grid limit";
  const ScoredSplits p = scored_splits(s);
  if (p.splits > 65535) return "split count exceeds 65535";
  if (uint64_t(s.kv_heads) * scored_blocks(s) * p.items * 64 * p.waves > 0xffffffffull)
    return "split and head product exceeds the grid limit";
  return nullptr;
}

const char* evict_error(const kvb_evict_shape& s) {
  if (s.batch == 0 || s.batch > 65535) return "batch must be in [1,65535]";
  if (const char* e = cache_error(s.kv_heads, s.dim, s.page_tokens, s.pages, s.kv_bits)) return e;
  if (s.max_tokens == 0 || s.max_tokens > 0x7fffffffu) return "max_tokens must be in [1,2^31-1]";
  if (s.total_tokens == 0 || s.table_entries == 0 || s.dst_entries == 0)
    return "total_tokens, table_entries and dst_entries must be positive";
  if (s.keep == 0 || s.keep > (1u << 30)) return "keep must be in [1,2^30]";
  if (uint64_t(s.sink) + s.recent > s.keep) return "sink and recent exceed keep";
  if (uint64_t(s.batch) * s.keep > 0xffffffffull) return "batch and keep product exceeds 32 bits";
  // Work-groups of the two launches: 1,024 tokens, and 64 kept tokens of a kv head.
  const uint64_t most = std::min(s.keep, s.max_tokens);
  if (uint64_t(s.batch) * ceil_div(s.max_tokens, 1024) > 0x7fffffffull ||
      uint64_t(s.batch) * s.kv_heads * ceil_div(most, 64) > 0x7fffffffull)
    return "batch, tokens and heads exceed the grid limit";
  return nullptr;
}

ScoredSplits weight_splits(const kvb_scored_shape& s) {
  ScoredSplits p = split_items(s, s.kv_heads, 0);
  if (p.waves > 4) p.waves = 16;  // all that its work-group can have
  return p;
}

}  // namespace kvb
