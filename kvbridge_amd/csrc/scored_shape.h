// Validation and sizing of the calls on a 4- or 8-bit cache; host only.
#pragma once
#include <algorithm>
#include <cstdint>

#include "kvbridge_c.h"

namespace kvb {

// nullptr when valid, else the first failed rule's message.
const char* append4_error(const kvb_append_shape& s);
const char* read_error(const kvb_read_shape& s);
const char* scored_error(const kvb_scored_shape& s);
const char* evict_error(const kvb_evict_shape& s);

uint32_t scored_blocks(const kvb_scored_shape& s);  // blocks of 16 head-rows per kv head

struct ScoredSplits {
  uint32_t items;   // (sequence, split) work items of a kv head and block, each with its partials
  uint32_t splits;  // items of every sequence; 0: the kernel shares them out by the sequences' lengths
  uint32_t tiles;   // least tiles of an item
  uint32_t waves;   // of a work-group
  uint32_t alone;   // up to so many tiles a sequence is not split
};
ScoredSplits scored_splits(const kvb_scored_shape& s);
// Whether the last work-group of a block merges its splits itself.
bool scored_one_launch(const kvb_scored_shape& s, const ScoredSplits& p);

// The same for the weights, whose work-groups take all blocks of a kv head.
ScoredSplits weight_splits(const kvb_scored_shape& s);

}  // namespace kvb
