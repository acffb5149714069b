// Shared parts of the kernels that read a 4- or 8-bit cache under score forms
// (scored_attend.h, scored_weights.hip): a sequence's extent and the tokens
// its query rows see, the page lookups of a wave's tiles, and a tile's scores.
//
// A tile is 32 tokens, head-rows (query row x query head of one kv head) go in
// blocks of 16.  Scores are S^T = K Q^T by v_mfma_f32_16x16x32_f16: two
// products (A, B) of 16 tokens by 16 head-rows for each 32 dims.  The C layout
// leaves lane (r = l % 16, kg = l / 16) four tokens of A and four of B for
// head-row r; which tokens those are is the choice of the rows loaded, and is
// made such that the lane's eight scores are the eight k indices that it has
// to supply as B operand of O^T = V^T P^T: P never changes lanes.
//
// 4 bits, K: a code c in the low bits of a half-word is the fp16 subnormal c *
// 2^-24, in bits 4..7 it is 16 c * 2^-24, and the products of subnormals are
// exact here, so a code is unpacked by one mask: two v_perm_b32 and four
// v_and_b32 give eight of them.  The 2^24 goes into the score's factor, the 16
// into Q.  A block of 32 dims is one product, so its step multiplies the
// product's result and its least value the sum of Q over the block: score =
// sum_g step_g D_g + least_g Qs_g, in fp32.  The codes are not negative and the
// two terms cancel, and the products' sums are truncated, not rounded, which
// cost 2e-6 of m and 7e-6 of l; therefore Q's first digit is an integer of 11
// bits and a sign, with which the sum of 32 products is an exact integer below
// 2^20, and a second digit holds the rest.
// 4 bits, V: the same cancellation over a whole context would cost 2e-5 of an
// output, so codes enter as c - 8 (one v_and_or_b32 and half a v_pk_add_f16 more
// per two codes) and the block's value at code 8 replaces the least.
// With few head-rows most of the 16 columns would be idle while every lane
// multiplies all G parameters of its tokens.  Instead column r * F + f holds
// head-row r's Q of the blocks f * H .. f * H + H - 1 (G = F H) and zeros
// elsewhere: the products of all blocks then accumulate in H results, a lane
// applies the parameters of its H blocks only (loaded by itself), and a sum over
// F neighbouring lanes makes the score; likewise the weights times the steps
// and the values at code 8.  That was 592 -> 350 vector instructions per tile
// at dim 128 and four head-rows (F = 4).  F = 1 (more head-rows): the parameters
// of a lane's tokens lie in the 16 lanes of its row and are read by DPP row
// broadcasts inside the multiply-adds.
// 8 bits: codes are converted exactly (i8x8_to_f16), the per-token scale
// multiplies the sum.
//
// Q is scaled by a power of two per head-row such that its largest magnitude
// lies in [2^13, 2^14).  One digit (8 bits, 16-bit q) then holds it exactly down
// to 2^-28 of the row's maximum, two within 2^-24 of that maximum.
#pragma once
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cstdint>

#include "batch.h"
#include "device_common.h"
#include "scored_args.h"

namespace kvb {

typedef uint32_t u32x2_s __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_s __attribute__((ext_vector_type(4)));

constexpr uint32_t kTileTokens = 32;

// Lane J of each 16-lane row.  Every lane must be active where it is called:
// outside of selects and branches.
template <int J>
__device__ __forceinline__ float bc(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x150 + J, 0xF, 0xF, true));
}
template <int J>
__device__ __forceinline__ int bci(int x) {
  return __builtin_amdgcn_mov_dpp(x, 0x150 + J, 0xF, 0xF, true);
}

// For a lane group's eight tokens, whose parameters of one block lie in lanes L,
// L + 2, .. of its row: x[j] += step_j d_j + least_j sum, d_j products of the
// matrix unit.  The compiler gives every broadcast into a fused multiply-add a
// v_mov_b32 of its own (with weigh_block 1,114 -> 858 vector instructions per
// tile at dim 256, f32; two sequences of 32K under 16 head-rows of dim 128 38.2
// -> 35.3 us).  The waits inside are the author's: 2 states from a write to a
// DPP read, 19 from the longest matrix product to a read of its result (2 + 8 +
// 12 here).
template <int L>
__device__ __forceinline__ void add_block(float (&x)[8], float step, float least, const f32x4& da, const f32x4& db, float sum) {
  asm("s_nop 1\n\t"
      "v_fmac_f32_dpp %0, %9, %10 row_newbcast:%c19 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %1, %9, %10 row_newbcast:%c20 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %2, %9, %10 row_newbcast:%c21 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %3, %9, %10 row_newbcast:%c22 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %4, %9, %10 row_newbcast:%c23 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %5, %9, %10 row_newbcast:%c24 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %6, %9, %10 row_newbcast:%c25 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %7, %9, %10 row_newbcast:%c26 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 11\n\t"
      "v_fmac_f32_dpp %0, %8, %11 row_newbcast:%c19 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %1, %8, %12 row_newbcast:%c20 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %2, %8, %13 row_newbcast:%c21 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %3, %8, %14 row_newbcast:%c22 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %4, %8, %15 row_newbcast:%c23 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %5, %8, %16 row_newbcast:%c24 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %6, %8, %17 row_newbcast:%c25 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %7, %8, %18 row_newbcast:%c26 row_mask:0xf bank_mask:0xf"
      : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7])
      : "v"(step), "v"(least), "v"(sum), "v"(da[0]), "v"(da[1]), "v"(da[2]), "v"(da[3]), "v"(db[0]), "v"(db[1]), "v"(db[2]),
        "v"(db[3]), "n"(L), "n"(L + 2), "n"(L + 4), "n"(L + 6), "n"(L + 8), "n"(L + 10), "n"(L + 12), "n"(L + 14));
}
// The same for weights p: w[j] = step_j p_j, mid += at8_j p_j.
template <int L>
__device__ __forceinline__ void weigh_block(float (&w)[8], float& mid, float step, float at8, const float (&p)[8]) {
  asm("s_nop 1\n\t"
      "v_mul_f32_dpp %0, %9, %11 row_newbcast:%c19 row_mask:0xf bank_mask:0xf\n\t"
      "v_mul_f32_dpp %1, %9, %12 row_newbcast:%c20 row_mask:0xf bank_mask:0xf\n\t"
      "v_mul_f32_dpp %2, %9, %13 row_newbcast:%c21 row_mask:0xf bank_mask:0xf\n\t"
      "v_mul_f32_dpp %3, %9, %14 row_newbcast:%c22 row_mask:0xf bank_mask:0xf\n\t"
      "v_mul_f32_dpp %4, %9, %15 row_newbcast:%c23 row_mask:0xf bank_mask:0xf\n\t"
      "v_mul_f32_dpp %5, %9, %16 row_newbcast:%c24 row_mask:0xf bank_mask:0xf\n\t"
      "v_mul_f32_dpp %6, %9, %17 row_newbcast:%c25 row_mask:0xf bank_mask:0xf\n\t"
      "v_mul_f32_dpp %7, %9, %18 row_newbcast:%c26 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %8, %10, %11 row_newbcast:%c19 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %8, %10, %12 row_newbcast:%c20 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %8, %10, %13 row_newbcast:%c21 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %8, %10, %14 row_newbcast:%c22 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %8, %10, %15 row_newbcast:%c23 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %8, %10, %16 row_newbcast:%c24 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %8, %10, %17 row_newbcast:%c25 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %8, %10, %18 row_newbcast:%c26 row_mask:0xf bank_mask:0xf"
      : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7]), "+v"(mid)
      : "v"(step), "v"(at8), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]), "n"(L),
        "n"(L + 2), "n"(L + 4), "n"(L + 6), "n"(L + 8), "n"(L + 10), "n"(L + 12), "n"(L + 14));
}

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return uint32_t(__builtin_amdgcn_readfirstlane(int(x))); }

template <int I, int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<I + 1, N>(f);
  }
}

// Sequence b's metadata, every index clamped to the declared sizes.
struct ScoredSeq {
  uint32_t start, tokens, table_off;
};
__device__ __forceinline__ ScoredSeq clamp_seq(uint32_t s0, uint32_t s1, uint32_t off, uint32_t total, uint32_t entries,
                                               uint32_t page_tokens, uint32_t max_tokens) {
  s0 = s0 < total ? s0 : total;
  s1 = s1 < s0 ? s0 : (s1 < total ? s1 : total);
  uint32_t t = s1 - s0 < max_tokens ? s1 - s0 : max_tokens;
  off = off < entries ? off : entries;
  const uint64_t room = uint64_t(entries - off) * page_tokens;
  if (t > room) t = uint32_t(room);
  return ScoredSeq{s0, t, off};
}

// A work-group's part of the batch: split `split` of the `count` that sequence
// `seq` has, whose items begin at `first`.
struct WorkItem {
  uint32_t seq, split, count, first;
  ScoredSeq e;
};
__device__ __forceinline__ ScoredSeq load_seq(const ScoredArgs& a, uint32_t b) {
  return clamp_seq(a.seq_starts[b], a.seq_starts[b + 1u], a.page_offsets[b], a.total_tokens, a.table_entries, a.page_tokens,
                   a.max_tokens);
}

// How many items each sequence gets where the host leaves that open (at most
// 256 sequences, four per lane): one, and of its tiles a share that is the same
// for all and as large as the number of items allows.  Every wave of the call,
// and of the merge, derives the same numbers from the same metadata.
struct ItemShares {
  uint32_t count[4];
};
__device__ __forceinline__ ItemShares item_shares(const ScoredArgs& a) {
  const uint32_t lane = threadIdx.x & 63u;
  ItemShares s;
  float tiles[4], total = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = 64u * i + lane;
    tiles[i] = 0.f;
    if (64u * i < a.batch && b < a.batch) {
      const uint32_t t = load_seq(a, b).tokens;
      const uint64_t seen = uint64_t(a.window) + a.rows + 31u;
      uint32_t n = (a.window != 0u && seen < t ? uint32_t(seen) : t) / kTileTokens + 1u;
      if (a.prefix != nullptr && a.window != 0u) {
        const int64_t p = a.prefix[b];
        n += p <= 0 ? 0u : (p < int64_t(t) ? uint32_t(p) : t) / kTileTokens + 1u;
      }
      tiles[i] = float(n);
    }
    total += tiles[i];
  }
  total = wave_sum(total);
  float per = fminf(1.f / float(a.split_tiles), float(a.items) / total);  // items per tile
  for (int round = 0; round < 24; ++round) {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = 64u * i + lane;
      const uint32_t c = uint32_t(fmaf(tiles[i], per, 0.9990234375f));  // one rounding in every kernel
      s.count[i] = b < a.batch ? (c > 1u ? c : 1u) : 0u;
      n += s.count[i];
    }
    n = uint32_t(__builtin_amdgcn_readlane(int(wave_scan(n)), 63));
    if (n <= a.items) return s;
    per = round < 22 ? per * (0.999f * float(a.items) / float(n)) : 0.f;  // at last one item each
  }
  return s;
}

// Item w's sequence and split; false past the last item.
__device__ __forceinline__ bool item_of(const ScoredArgs& a, uint32_t w, WorkItem& it) {
  if (a.splits != 0u) {
    it.seq = w / a.splits;
    it.split = w - it.seq * a.splits;
    it.count = a.splits;
    it.first = w - it.split;
    it.e = load_seq(a, it.seq);
    return true;
  }
  const ItemShares s = item_shares(a);
  uint32_t base = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (64u * i >= a.batch) break;
    const uint32_t upto = base + wave_scan(s.count[i]);
    const uint64_t hit = __ballot(upto > w);
    if (hit != 0u) {
      const int l = __builtin_ctzll(hit);
      it.seq = 64u * i + uint32_t(l);
      it.count = uint32_t(__builtin_amdgcn_readlane(int(s.count[i]), l));
      it.first = uint32_t(__builtin_amdgcn_readlane(int(upto), l)) - it.count;
      it.split = w - it.first;
      it.e = load_seq(a, it.seq);
      return true;
    }
    base = uint32_t(__builtin_amdgcn_readlane(int(upto), 63));
  }
  return false;
}
// The items of sequence b: first and count.
__device__ __forceinline__ WorkItem items_of(const ScoredArgs& a, uint32_t b) {
  WorkItem it;
  it.seq = b;
  it.split = 0u;
  it.count = a.splits;
  it.first = b * a.splits;
  if (a.splits != 0u) return it;
  const ItemShares s = item_shares(a);
  uint32_t base = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t upto = base + wave_scan(s.count[i]);
    if (b / 64u == uint32_t(i)) {
      it.count = uint32_t(__builtin_amdgcn_readlane(int(s.count[i]), int(b % 64u)));
      it.first = uint32_t(__builtin_amdgcn_readlane(int(upto), int(b % 64u))) - it.count;
    }
    base = uint32_t(__builtin_amdgcn_readlane(int(upto), 63));
  }
  return it;
}

// First t in [0, n) with kpos[t] > x, else n (kpos nondecreasing), by every
// lane for its own x.  The first guess is that positions count up from 0: its
// two neighbours are requested beside the last position, before any of them is
// waited for.  Next the place that the last position implies if they count up
// by one, then a search.
struct Above {
  int64_t x, above, below;
  uint32_t g;
};
__device__ __forceinline__ Above ask_above(const int64_t* __restrict__ kpos, uint32_t n, int64_t x) {
  Above q;
  q.x = x;
  q.g = x < 0 ? 0u : (uint64_t(x) + 1u < n ? uint32_t(x) + 1u : (n > 0u ? n - 1u : 0u));
  q.above = n > 0u ? kpos[q.g] : 0;
  q.below = n > 0u && q.g > 0u ? kpos[q.g - 1u] : INT64_MIN;
  return q;
}
__device__ __forceinline__ uint32_t find_above(const int64_t* __restrict__ kpos, uint32_t n, int64_t last, const Above& q) {
  const int64_t x = q.x;
  if (n == 0u || last <= x) return n;
  if (q.above > x && (q.g == 0u || q.below <= x)) return q.g;
  const uint64_t back = uint64_t(last) - uint64_t(x);  // positive
  const uint32_t g = back < n ? n - uint32_t(back) : 0u;
  const int64_t above = kpos[g], below = g > 0u ? kpos[g - 1u] : INT64_MIN;
  uint32_t lo = 0, hi = n - 1u;  // kpos[hi] > x
  if (above > x && (g == 0u || below <= x)) return g;
  if (above > x) hi = g < hi ? g : hi;
  else lo = g + 1u;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2u;
    if (kpos[mid] > x) hi = mid;
    else lo = mid + 1u;
  }
  return lo;
}

__device__ __forceinline__ uint32_t row_min16(uint32_t v) {
  unrolled<0, 4>([&](auto i) {
    const uint32_t o = uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x120 + (1 << i), 0xF, 0xF, false));
    v = o < v ? o : v;
  });
  return v;
}
__device__ __forceinline__ uint32_t row_max16(uint32_t v) { return ~row_min16(~v); }

// The tokens that head-row r of a block sees: [lo, hi) and [0, pre); and over
// the block's rows (wave-uniform) the least lo, the largest hi, and the tokens
// that all of them see: [all_lo, all_hi) or [0, pre).
struct Visible {
  uint32_t lo, hi;
  uint32_t pre, min_lo, max_hi, all_lo, all_hi;
};
// What visible_tokens has to look up, requested early.
struct Sight {
  int64_t last;
  Above hi, lo, pre;
  bool has_lo, has_pre;
};
__device__ __forceinline__ Sight ask_visible(const ScoredArgs& a, const ScoredSeq& e, int64_t qpos, int64_t prefix) {
  const int64_t* kpos = a.k_positions + e.start;
  Sight s;
  s.last = e.tokens > 0u ? kpos[e.tokens - 1u] : 0;
  s.hi = ask_above(kpos, e.tokens, qpos);
  const int64_t w = int64_t(a.window);
  s.has_lo = a.window != 0u && qpos >= INT64_MIN + w;  // qpos - kpos < window  <=>  kpos > qpos - window
  s.has_pre = a.prefix != nullptr && prefix > INT64_MIN;
  s.lo = s.pre = s.hi;
  if (a.window != 0u) s.lo = ask_above(kpos, e.tokens, s.has_lo ? qpos - w : INT64_MIN);
  if (a.prefix != nullptr) s.pre = ask_above(kpos, e.tokens, s.has_pre ? prefix - 1 : INT64_MIN);
  return s;
}
__device__ __forceinline__ Visible visible_tokens(const ScoredArgs& a, const ScoredSeq& e, bool valid, const Sight& s) {
  Visible v;
  const int64_t* kpos = a.k_positions + e.start;
  v.hi = find_above(kpos, e.tokens, s.last, s.hi);
  v.lo = s.has_lo ? find_above(kpos, e.tokens, s.last, s.lo) : 0u;
  v.pre = s.has_pre ? find_above(kpos, e.tokens, s.last, s.pre) : 0u;
  if (v.lo > v.hi) v.lo = v.hi;
  if (!valid) v.lo = v.hi = 0u;
  const bool sees = v.lo < v.hi;
  v.pre = uint32_t(__builtin_amdgcn_readfirstlane(int(v.pre)));
  v.min_lo = uint32_t(__builtin_amdgcn_readfirstlane(int(row_min16(sees ? v.lo : 0xffffffffu))));
  v.max_hi = uint32_t(__builtin_amdgcn_readfirstlane(int(row_max16(sees ? v.hi : 0u))));
  // A head-row past the last one is never written out: it counts as seeing all.
  v.all_lo = uint32_t(__builtin_amdgcn_readfirstlane(int(row_max16(valid ? v.lo : 0u))));
  v.all_hi = uint32_t(__builtin_amdgcn_readfirstlane(int(row_min16(valid ? v.hi : 0xffffffffu))));
  if (v.max_hi == 0u) v.min_lo = 0u;
  return v;
}

// The live tiles of a block: [0, pre_tiles) of the prefix and [first, first +
// n - pre_tiles) of the rows' windows, numbered 0 .. n - 1.
struct LiveTiles {
  uint32_t pre_tiles, first, n;
  __device__ __forceinline__ bool same(const LiveTiles& o) const {
    return pre_tiles == o.pre_tiles && first == o.first && n == o.n;
  }
  __device__ __forceinline__ uint32_t tile(uint32_t i) const { return i < pre_tiles ? i : i - pre_tiles + first; }
};
__device__ __forceinline__ LiveTiles live_tiles(uint32_t pre, uint32_t lo, uint32_t hi) {
  LiveTiles t;
  t.pre_tiles = pre / kTileTokens + (pre % kTileTokens != 0u ? 1u : 0u);
  t.first = lo / kTileTokens;
  const uint32_t end = hi / kTileTokens + (hi % kTileTokens != 0u ? 1u : 0u);
  if (t.first < t.pre_tiles) t.first = t.pre_tiles;
  t.n = t.pre_tiles + (end > t.first ? end - t.first : 0u);
  return t;
}

// Page and slot of the four runs of 8 tokens of 16 of a wave's tiles: lane l
// holds run l % 4 of the wave's tile i0 + l / 4 (tile numbers by `tile_of`).
// Runs past the sequence's end repeat its last one, page ids past the pool the
// last page, so that every address formed from them lies inside.
struct TilePages {
  uint32_t page, slot;
};
template <typename F>
__device__ __forceinline__ TilePages tile_pages(const ScoredArgs& a, const ScoredSeq& e, F tile_of, uint32_t i0,
                                                uint32_t lane) {
  const uint32_t last = (e.tokens - 1u) / 8u;
  const uint64_t run64 = uint64_t(tile_of(i0 + lane / 4u)) * 4u + lane % 4u;
  const uint32_t run = run64 < last ? uint32_t(run64) : last;
  const uint32_t per = a.page_tokens / 8u;
  const uint32_t lp = run / per;
  const uint32_t page = a.page_table[e.table_off + lp];
  return TilePages{page < a.pages ? page : a.pages - 1u, (run - lp * per) * 8u};
}

// A tile's runs, wave-uniform: page and kv head in one number, first slot, and
// the row number (page, kv head, slot).  ONE: pages hold whole tiles, so that
// the four runs follow each other and only the first is kept.
template <bool ONE>
struct TileRows {
  static constexpr int kRuns = ONE ? 1 : 4;
  uint32_t slab[kRuns], slot[kRuns];
  __device__ __forceinline__ uint64_t row(int i, uint32_t page_tokens) const {
    return uint64_t(slab[ONE ? 0 : i]) * page_tokens + slot[ONE ? 0 : i] + (ONE ? 8u * uint32_t(i) : 0u);
  }
};
template <bool ONE>
__device__ __forceinline__ TileRows<ONE> tile_rows(const ScoredArgs& a, const TilePages& p, uint32_t i, uint32_t kv) {
  TileRows<ONE> t;
#pragma unroll
  for (int r = 0; r < TileRows<ONE>::kRuns; ++r) {
    const uint32_t page = uint32_t(__builtin_amdgcn_readlane(int(p.page), int((i % 16u) * 4u + r)));
    t.slot[r] = uint32_t(__builtin_amdgcn_readlane(int(p.slot), int((i % 16u) * 4u + r)));
    t.slab[r] = page * a.kv_heads + kv;
  }
  return t;
}

// One of four wave-uniform values by the lane's index (values, so that nothing
// is kept in memory to be indexed).
template <typename T>
__device__ __forceinline__ T pick(uint32_t i, T a, T b, T c, T d) {
  const T lo = (i & 1u) != 0u ? b : a, hi = (i & 1u) != 0u ? d : c;
  return (i & 2u) != 0u ? hi : lo;
}

template <int N>
struct Words {
  uint32_t w[N];
};
// N dwords from p (aligned to them): one load of 4, 8 or 16 bytes, or two.
template <int N>
__device__ __forceinline__ Words<N> load_words(const uint8_t* p) {
  Words<N> r;
  if constexpr (N == 1) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const u32x2_s v = *reinterpret_cast<const u32x2_s*>(p);
    r.w[0] = v[0];
    r.w[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4_s v = reinterpret_cast<const u32x4_s*>(p)[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) r.w[4 * i + k] = v[k];
    }
  }
  return r;
}

__device__ __forceinline__ f16x8 as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(f16x8, (u32x4_s{a, b, c, d}));
}

struct QPlace {
  uint32_t block, kg, j;
  bool odd;
};

// Sum over the F lanes of a head-row, in every one of them.
template <int F>
__device__ __forceinline__ float lanes_sum(float x) {
  if constexpr (F >= 2) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xF, 0xF, true));   // lane ^ 1
  if constexpr (F >= 4) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xF, 0xF, true));   // lane ^ 2
  if constexpr (F >= 8) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xF, 0xF, true));  // lane 7 - l of 8
  return x;
}

// ---- cache formats: loads and operands of a tile, DIM = 32 G ------------------
// token(kg, j): the tile's token of index j (0..7) of lane group kg.

template <int G, int F>
struct Cache4 {
  static constexpr int kGroups = G;
  static constexpr int kF = F;
  static constexpr int kH = G / F;  // blocks of a lane
  static constexpr int kBits = 4;
  static constexpr int kVWords = G >= 4 ? G / 4 : 1;
  // Parameter words of a lane.  F = 1: word w of a lane group's 8 G lies in lane
  // w / kPWords; else the lane's own blocks of its eight tokens.
  static constexpr int kPWords = F == 1 ? G / 2 : 8 * kH;
  struct K {
    Words<G> a, b;
    Words<kPWords> p;
  };
  struct V {
    Words<kVWords> v[8];
    Words<kPWords> p;
  };
  static __device__ __forceinline__ uint32_t token(uint32_t kg, uint32_t j) { return 4u * j + kg; }

  template <bool ONE>
  static __device__ __forceinline__ Words<kPWords> params(const void* base, const TileRows<ONE>& t, uint32_t P, uint32_t r,
                                                          uint32_t kg, uint32_t left) {
    const uint8_t* b = static_cast<const uint8_t*>(base);
    Words<kPWords> p;
    if constexpr (F == 1) {  // token j = r / 2 of the lane group, blocks (r % 2) * G / 2 ..
      const uint32_t tok = token(kg, r / 2u), in = (r % 2u) * (2u * G);
      if constexpr (ONE) p = load_words<kPWords>(b + t.row(0, P) * (4u * G) + (tok * (4u * G) + in));
      else p = load_words<kPWords>(b + (pick(r / 4u, t.row(0, P), t.row(1, P), t.row(2, P), t.row(3, P)) + tok % 8u) * (4u * G) + in);
      if (tok >= left) {  // slots behind the sequence hold anything
#pragma unroll
        for (int i = 0; i < kPWords; ++i) p.w[i] = 0u;
      }
    } else {
      const uint32_t at = kg * (4u * G) + r % F * (4u * kH);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint8_t* run = b + t.row(ONE ? 0 : j / 2, P) * (4u * G);
        const Words<kH> w = load_words<kH>(run + (at + 4u * uint32_t(ONE ? j : j % 2) * (4u * G)));
#pragma unroll
        for (int h = 0; h < kH; ++h) p.w[j * kH + h] = w.w[h];
      }
      if (left < kTileTokens) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int h = 0; h < kH; ++h) p.w[j * kH + h] = token(kg, j) < left ? p.w[j * kH + h] : 0u;
      }
    }
    return p;
  }
  // The parameters as floats, and those of token j and the lane's block h.
  struct Params {
    float step[kPWords], other[kPWords];
    template <int j, int h>
    __device__ __forceinline__ float step_of() const {
      if constexpr (F == 1) return bc<2 * j + h / kPWords>(step[h % kPWords]);
      else return step[j * kH + h];
    }
    template <int j, int h>
    __device__ __forceinline__ float other_of() const {
      if constexpr (F == 1) return bc<2 * j + h / kPWords>(other[h % kPWords]);
      else return other[j * kH + h];
    }
  };
  // AT8: the value at code 8 in place of the least.
  template <bool AT8>
  static __device__ __forceinline__ Params unpack(const Words<kPWords>& w) {
    Params p;
#pragma unroll
    for (int i = 0; i < kPWords; ++i) {
      p.step[i] = __uint_as_float(w.w[i] & 0xffff0000u);
      p.other[i] = __uint_as_float(w.w[i] << 16);
      if constexpr (AT8) p.other[i] = fmaf(p.step[i], 8.f, p.other[i]);
    }
    return p;
  }
  // A rows m: tokens 4 (m % 4) + m / 4 of the first 16, B those of the last 16.
  template <bool ONE>
  static __device__ __forceinline__ K load_k(const ScoredArgs& a, const TileRows<ONE>& t, uint32_t r, uint32_t kg,
                                             uint32_t left) {
    const uint32_t P = a.page_tokens, tok = 4u * (r % 4u) + r / 4u;
    const uint8_t* base = static_cast<const uint8_t*>(a.k);
    K k;
    if constexpr (ONE) {
      const uint8_t* first = base + t.row(0, P) * (16u * G);
      const uint32_t at = tok * (16u * G) + kg * (4u * G);
      k.a = load_words<G>(first + at);
      k.b = load_words<G>(first + (at + 16u * (16u * G)));
    } else {
      const uint32_t in = (tok % 8u) * (16u * G) + kg * (4u * G);
      const uint32_t second = r / 2u % 2u;
      k.a = load_words<G>(base + pick<uint64_t>(second, t.row(0, P), t.row(1, P), 0u, 0u) * (16u * G) + in);
      k.b = load_words<G>(base + pick<uint64_t>(second, t.row(2, P), t.row(3, P), 0u, 0u) * (16u * G) + in);
    }
    k.p = params<ONE>(a.ks, t, P, r, kg, left);
    return k;
  }
  template <bool ONE>
  static __device__ __forceinline__ V load_v(const ScoredArgs& a, const TileRows<ONE>& t, uint32_t r, uint32_t kg,
                                             uint32_t left) {
    const uint32_t P = a.page_tokens, at = kg * (16u * G) + r * G;
    V v;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint8_t* run = static_cast<const uint8_t*>(a.v) + t.row(ONE ? 0 : j / 2, P) * (16u * G);
      const uint8_t* p = run + (at + 4u * uint32_t(ONE ? j : j % 2) * (16u * G));
      if constexpr (G == 2) v.v[j].w[0] = *reinterpret_cast<const uint16_t*>(p);
      else v.v[j] = load_words<kVWords>(p);
    }
    v.p = params<ONE>(a.vs, t, P, r, kg, left);
    return v;
  }
  // Eight codes of block g, dims 8 kg + (0, 2, 1, 3, 4, 6, 5, 7), the odd dims times 16.
  template <int g>
  static __device__ __forceinline__ f16x8 k_frag(const Words<G>& w) {
    constexpr uint32_t s0 = 0x0c000c00u | uint32_t(g % 4);
    uint32_t lo, hi;
    if constexpr (G == 2) {  // bytes g, 2 + g of a dword
      constexpr uint32_t s = 0x0c000c00u | uint32_t(g) | uint32_t(2 + g) << 16;
      lo = __builtin_amdgcn_perm(w.w[0], w.w[0], s);
      hi = __builtin_amdgcn_perm(w.w[1], w.w[1], s);
    } else {
      constexpr int at = g / 4, step = G / 4;
      constexpr uint32_t s = s0 | uint32_t(4 + g % 4) << 16;
      lo = __builtin_amdgcn_perm(w.w[step + at], w.w[at], s);
      hi = __builtin_amdgcn_perm(w.w[3 * step + at], w.w[2 * step + at], s);
    }
    return as_f16x8(lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u);
  }
  // Where dim d stands in Q's operands: block, lane group, element; and whether
  // its code is times 16.
  static __device__ __forceinline__ QPlace q_place(uint32_t d) {
    const uint32_t p = d % 8u;  // element order 0, 2, 1, 3, 4, 6, 5, 7
    return QPlace{d / 32u, d / 8u % 4u, (p & 4u) | (p & 1u) << 1 | (p & 2u) >> 1, (p & 1u) != 0u};
  }
};

template <int G>
struct Cache8 {
  static constexpr int kGroups = G;
  static constexpr int kF = 1, kH = G;
  static constexpr int kBits = 8;
  static constexpr int kPWords = 1;
  struct K {
    Words<2 * G> a, b;
    float p;
  };
  struct V {
    Words<2> v[2 * G];
    float p;
  };
  static __device__ __forceinline__ uint32_t token(uint32_t kg, uint32_t j) { return 8u * kg + j; }
  // Lanes r and r + 8: the scale of token r % 8 of the group.
  template <bool ONE>
  static __device__ __forceinline__ float params(const void* base, const TileRows<ONE>& t, uint32_t P, uint32_t r,
                                                 uint32_t kg, uint32_t left) {
    const float* b = static_cast<const float*>(base);
    const float p = ONE ? (b + t.row(0, P))[token(kg, r % 8u)]
                        : b[pick(kg, t.row(0, P), t.row(1, P), t.row(2, P), t.row(3, P)) + r % 8u];
    return token(kg, r % 8u) < left ? p : 0.f;
  }
  // A rows m: tokens 8 (m / 4) + m % 4, B those four later.
  template <bool ONE>
  static __device__ __forceinline__ K load_k(const ScoredArgs& a, const TileRows<ONE>& t, uint32_t r, uint32_t kg,
                                             uint32_t left) {
    const uint32_t P = a.page_tokens, D = 32u * G;
    const uint8_t* base = static_cast<const uint8_t*>(a.k);
    const uint8_t* first = ONE ? base + t.row(0, P) * D : base + pick(r / 4u, t.row(0, P), t.row(1, P), t.row(2, P), t.row(3, P)) * D;
    const uint32_t at = (ONE ? 8u * (r / 4u) + r % 4u : r % 4u) * D + kg * 16u;
    K k;
#pragma unroll
    for (int h = 0; h < G / 2; ++h) {  // 64 dims a piece: 16 bytes of each lane group
      const Words<4> x = load_words<4>(first + (at + 64u * h)), y = load_words<4>(first + (at + 64u * h + 4u * D));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k.a.w[4 * h + i] = x.w[i];
        k.b.w[4 * h + i] = y.w[i];
      }
    }
    k.p = params<ONE>(a.ks, t, P, r, kg, left);
    return k;
  }
  // Dim-major V: dim 16 f + r, the lane group's eight tokens.
  template <bool ONE>
  static __device__ __forceinline__ V load_v(const ScoredArgs& a, const TileRows<ONE>& t, uint32_t r, uint32_t kg,
                                             uint32_t left) {
    const uint32_t P = a.page_tokens, D = 32u * G;
    const uint8_t* base = static_cast<const uint8_t*>(a.v);
    V v;
    if constexpr (ONE) {
      const uint8_t* slab = base + (uint64_t(t.slab[0]) * (uint64_t(D) * P) + t.slot[0]);
      const uint64_t at = uint64_t(r) * P + 8u * kg;
#pragma unroll
      for (int f = 0; f < 2 * G; ++f) v.v[f] = load_words<2>(slab + uint64_t(16u * f) * P + at);
    } else {
      const uint32_t slab = pick(kg, t.slab[0], t.slab[1], t.slab[2], t.slab[3]);
      const uint32_t slot = pick(kg, t.slot[0], t.slot[1], t.slot[2], t.slot[3]);
      const uint8_t* first = base + uint64_t(slab) * (uint64_t(D) * P) + slot;
#pragma unroll
      for (int f = 0; f < 2 * G; ++f) v.v[f] = load_words<2>(first + uint64_t(16u * f + r) * P);
    }
    v.p = params<ONE>(a.vs, t, P, r, kg, left);
    return v;
  }
  template <int g>
  static __device__ __forceinline__ f16x8 k_frag(const Words<2 * G>& w) {
    return i8x8_to_f16(w.w[2 * g], w.w[2 * g + 1]);
  }
  static __device__ __forceinline__ QPlace q_place(uint32_t d) {
    return QPlace{d / 64u * 2u + d / 8u % 2u, d / 16u % 4u, d % 8u, false};
  }
};

// ---- Q ---------------------------------------------------------------------------

// Digits of Q: two for 4 bits, and for fp32.
template <class C, bool F32>
constexpr int kQDigits = C::kBits == 4 || F32 ? 2 : 1;

// The Q operands of a block of 16 head-rows in LDS, where every wave of the
// work-group and every tile reads them: held in registers they took 32 (dim
// 128) or 64 (dim 256) per lane and cost a third of the waves.
template <class C, int QD>
struct QBlock {
  f16x8 d[C::kGroups][QD][64];                     // fp16 digits of the scaled elements, by lane
  float sum[C::kBits == 4 ? C::kH : 1][16];        // 4 bits: sum over each 32 dims, in units of 2^-24, by column
  float factor[16];                                // score = factor * (sum of the scaled products)
};

// With F > 1 the operands are cleared first, by n threads; a barrier follows.
template <class C, int QD>
__device__ __forceinline__ void clear_q(QBlock<C, QD>& q, uint32_t tid, uint32_t n) {
  if constexpr (C::kF > 1) {
    const f16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    for (uint32_t i = tid; i < uint32_t(C::kGroups * QD * 64); i += n) (&q.d[0][0][0])[i] = zero;
  }
}
// By 256 threads (four whole waves): thread 16 r + s takes 2 G dims from 2 G s
// of head-row r, so that the maximum over a row is one over 16 lanes.  `at`:
// element index of the head-row's Q.  The caller's barrier follows.
template <class C, int QD>
__device__ __forceinline__ void stage_q(const ScoredArgs& a, uint64_t at, bool valid, QBlock<C, QD>& q, uint32_t tid) {
  constexpr int G = C::kGroups, N = 2 * G;
  constexpr int F = C::kF, H = C::kH;
  const uint32_t r = tid / 16u, s = tid % 16u, d0 = s * N;
  if (r >= 16u / F) return;
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = 0.f;
  if (valid) {
    if (a.q_type == 1u) {
      const float* p = static_cast<const float*>(a.q) + at + d0;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = p[i];
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(a.q) + at + d0;
      uint16_t u[N];
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = p[i];
#pragma unroll
      for (int i = 0; i < N; ++i)
        x[i] = a.q_type == 2u ? float(__builtin_bit_cast(_Float16, u[i])) : __uint_as_float(uint32_t(u[i]) << 16);
    }
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(x[i]));
  top = fmaxf(top, row_ror<8>(top));
  top = fmaxf(top, row_ror<4>(top));
  top = fmaxf(top, row_ror<2>(top));
  top = fmaxf(top, row_ror<1>(top));
  int up = 0;  // an infinite or NaN element: the row's result is NaN whatever the scale
  if (top > 0.f && top <= FLT_MAX) up = 14 - __builtin_amdgcn_frexp_expf(top);  // frexp: top = f * 2^e, f in [1/2, 1)
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const QPlace p = C::q_place(d0 + i);
    float y = ldexpf(x[i], up);
    sum += y;
    if (p.odd) y *= 0.0625f;
    // 4 bits: multiples of 8 up to 2^14 (odd dims: both a 16th)
    const float unit = p.odd ? 0.5f : 8.f, per = p.odd ? 2.f : 0.125f;
    const _Float16 hi = C::kBits == 4 ? _Float16(__builtin_rintf(y * per) * unit) : _Float16(y);
    const uint32_t column = r * F + p.block / H;
    reinterpret_cast<_Float16*>(&q.d[p.block][0][p.kg * 16u + (F > 1 ? column : r)])[p.j] = hi;
    if constexpr (QD == 2)
      reinterpret_cast<_Float16*>(&q.d[p.block][1][p.kg * 16u + (F > 1 ? column : r)])[p.j] = _Float16(y - float(hi));
  }
  if constexpr (C::kBits == 4) {  // 16 / G threads hold a block's 32 dims
#pragma unroll
    for (int o = 1; o < 16 / G; o <<= 1) sum += __shfl_xor(sum, o);
    const uint32_t block = s / (16u / G);
    if (s % (16u / G) == 0u) q.sum[block % H][r * F + block / H] = ldexpf(sum, -24);
  }
  if (s < uint32_t(F)) q.factor[r * F + s] = ldexpf(a.scale, (C::kBits == 4 ? 24 : 0) - up);
}

// ---- scores ------------------------------------------------------------------------

// The products of a tile: x[j] = sum of step / scale times products plus least
// value times Q sums, before the score's factor.
template <class C, int QD>
__device__ __forceinline__ void tile_scores(const typename C::K& k, const QBlock<C, QD>& q, uint32_t lane, float (&x)[8]) {
  constexpr int G = C::kGroups;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if constexpr (C::kBits == 4) {
    constexpr int H = C::kH, F = C::kF;
    const typename C::Params p = C::template unpack<false>(k.p);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
    unrolled<0, H>([&](auto hc) {
      constexpr int h = hc;
      f32x4 da = zero, db = zero;
      unrolled<0, F>([&](auto fc) {
        constexpr int g = fc * H + h;
        const f16x8 ka = C::template k_frag<g>(k.a), kb = C::template k_frag<g>(k.b);
#pragma unroll
        for (int i = 0; i < QD; ++i) {
          const f16x8 qd = q.d[g][i][lane];
          da = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qd, da, 0, 0, 0);
          db = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qd, db, 0, 0, 0);
        }
      });
      const float sum = q.sum[h][lane % 16u];
      if constexpr (F == 1) {
        constexpr int PW = C::kPWords;
        add_block<h / PW>(x, p.step[h % PW], p.other[h % PW], da, db, sum);
      } else {
        unrolled<0, 8>([&](auto jc) {
          constexpr int j = jc;
          const float d = j < 4 ? da[j % 4] : db[j % 4];
          x[j] = fmaf(p.template step_of<j, h>(), d, x[j]);
          x[j] = fmaf(p.template other_of<j, h>(), sum, x[j]);
        });
      }
    });
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = lanes_sum<F>(x[j]);
  } else {
    f32x4 da = zero, db = zero;
    unrolled<0, G>([&](auto gc) {
      constexpr int g = gc;
      const f16x8 ka = C::template k_frag<g>(k.a), kb = C::template k_frag<g>(k.b);
#pragma unroll
      for (int i = 0; i < QD; ++i) {
        const f16x8 qd = q.d[g][i][lane];
        da = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qd, da, 0, 0, 0);
        db = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qd, db, 0, 0, 0);
      }
    });
    unrolled<0, 8>([&](auto jc) {
      constexpr int j = jc;
      x[j] = bc<j>(k.p) * (j < 4 ? da[j % 4] : db[j % 4]);
    });
  }
}

// cap * tanh(s / cap).  tanh(u) as u times an odd series below 1/4
// (the next term is under 2^-26 of the value), else 1 - 2 / (e^2u + 1).
__device__ __forceinline__ float capped(float s, float cap, float inv_cap) {
  const float u = s * inv_cap, w = u * u;
  const float series = u * fmaf(w, fmaf(w, fmaf(w, fmaf(w, 0.021869488f, -0.053968254f), 0.13333333f), -0.33333333f), 1.f);
  const float e = exp_e(2.f * fabsf(u));
  const float t = copysignf(1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f), u);
  return cap * (fabsf(u) < 0.25f ? series : t);
}

// The distance k_position - q_position in two steps, both clamped to +-2^30:
// token to the sequence's first row, that row to this one.
__device__ __forceinline__ int near(int64_t d) {
  constexpr int64_t kFar = int64_t(1) << 30;
  return int(d < -kFar ? -kFar : (d > kFar ? kFar : d));
}

// Score forms on a tile's products: factor, cap, bias by distance, and -inf
// where the tile is masked and the token not visible.  Scores stay in natural
// units and are multiplied by log2(e) inside the exponent's fma: with scale and
// log2(e) in one rounded factor l of 512 tokens was off by 1.1e-6, since every
// score carried the same relative error.
struct ScoreForm {
  float factor, cap, inv_cap, slope;
  int back;  // this row's position less the first row's
};
__device__ __forceinline__ ScoreForm score_form(const ScoredArgs& a, float factor, float slope, int back) {
  return ScoreForm{factor, a.cap, a.cap > 0.f ? 1.f / a.cap : 0.f, slope, back};
}
// x: products of N of the tile's tokens, number(i) the lane's i-th one, far(i)
// its position less that of the sequence's first row.
template <int N, typename Number, typename Far>
__device__ __forceinline__ void apply_form(const ScoredArgs& a, const ScoreForm& f, bool masked, uint32_t lo, uint32_t hi,
                                           uint32_t pre, Number number, Far far, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] *= f.factor;
  if (a.cap > 0.f) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = capped(x[i], f.cap, f.inv_cap);
  }
  if (a.slopes != nullptr) {
    int d[N];
    far(d);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = fmaf(f.slope, float(d[i] - f.back), x[i]);
  }
  if (masked) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t t = number(i);
      const bool seen = (t >= lo && t < hi) || t < pre;
      x[i] = seen ? x[i] : neg_inf();
    }
  }
}

// Lane's share of a tile's key positions for the bias by distance: token
// (kg, r % 8), relative to the first row's position.
template <class C>
__device__ __forceinline__ int load_ahead(const ScoredArgs& a, const ScoredSeq& e, uint32_t t0, uint32_t r, uint32_t kg,
                                          int64_t qref) {
  if (a.slopes == nullptr) return 0;
  uint32_t t = t0 + C::token(kg, r % 8u);
  t = t < e.tokens ? t : e.tokens - 1u;
  const int64_t p = a.k_positions[e.start + t];
  return near(int64_t(uint64_t(p) - uint64_t(qref)));
}

}  // namespace kvb
