// Attention weights per cached token (kvb_accumulate_weights).
//
// With m and l of an attention call known, the weight of token t for head-row
// r is exp(s_rt - m_r) / l_r: K is read once more, V not at all.  A work-group
// of four waves takes chunk_tiles tiles of one (sequence, kv head), its waves
// every fourth tile, so that a (page, kv head, slot) of a sequence is written
// by one wave only and in one order.  The operands of as many blocks of 16
// head-rows as fit 64 KiB of LDS are staged at once and a tile's K serves all
// of them; more head-rows take another pass over the chunk.  The sum over
// the head-rows of a block is a DPP reduction over the 16 lanes of a row.
#include "scored.h"

namespace kvb {
namespace {

constexpr uint32_t kWeightWaves = 4;

__device__ __forceinline__ float row_sum16(float x) {
  x += row_ror<8>(x);
  x += row_ror<4>(x);
  x += row_ror<2>(x);
  x += row_ror<1>(x);
  return x;
}

// A block's head-rows next to their Q operands.
template <class C, int QD>
struct WeightBlock {
  QBlock<C, QD> q;
  uint32_t lo[16], hi[16];
  float m[16], per_l[16], slope[16];
  int back[16];
  uint32_t min_lo, max_hi;
};
template <class C, int QD>
constexpr uint32_t kBlocksAtOnce = 65536u / sizeof(WeightBlock<C, QD>);

template <class C, int QD, bool ONE>
__global__ __launch_bounds__(64 * kWeightWaves) void scored_weights_kernel(const ScoredArgs a) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  using Block = WeightBlock<C, QD>;
  Block* const blocks = reinterpret_cast<Block*>(lds_raw);
  const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, kg = lane >> 4;
  const uint32_t wave = uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
  uint32_t at = blockIdx.x;
  const uint32_t kv = at % a.kv_heads;
  at /= a.kv_heads;
  const uint32_t chunk = at % a.chunks, b = at / a.chunks;
  const ScoredSeq e = clamp_seq(a.seq_starts[b], a.seq_starts[b + 1u], a.page_offsets[b], a.total_tokens, a.table_entries,
                                a.page_tokens, a.max_tokens);
  const uint32_t tiles = e.tokens / kTileTokens + (e.tokens % kTileTokens != 0u ? 1u : 0u);
  const uint64_t c0 = uint64_t(chunk) * a.chunk_tiles;
  if (c0 >= tiles) return;
  const uint32_t t_begin = uint32_t(c0), t_end = tiles - t_begin > a.chunk_tiles ? t_begin + a.chunk_tiles : tiles;
  const uint32_t fresh0 = a.fresh < e.tokens ? e.tokens - a.fresh : 0u;  // tokens from here on are set
  const int64_t qref = a.q_positions[uint64_t(b) * a.rows], prefix = a.prefix ? a.prefix[b] : 0;

  for (uint32_t first = 0; first < a.blocks; first += kBlocksAtOnce<C, QD>) {
    const uint32_t count = a.blocks - first < kBlocksAtOnce<C, QD> ? a.blocks - first : kBlocksAtOnce<C, QD>;
    if (first > 0u) {
      __threadfence();  // what the first pass set is in place before it is added to
      __syncthreads();  // and every wave is done with the last pass's operands
    }
    for (uint32_t i = 0; i < count; ++i) clear_q(blocks[i].q, threadIdx.x, 64u * kWeightWaves);
    if (C::kF > 1) __syncthreads();
    for (uint32_t i = 0; i < count; ++i) {
      const uint32_t hr = (first + i) * 16u + threadIdx.x / 16u;
      stage_q<C, QD>(a, (uint64_t(b) * a.rows + hr / a.group) * a.q_stride + uint64_t(kv * a.group + hr % a.group) * a.dim,
                     hr < a.head_rows, blocks[i].q, threadIdx.x);
    }
    uint32_t pre = 0;
    for (uint32_t i = wave; i < count; i += kWeightWaves) {
      const uint32_t hr = (first + i) * 16u + r / C::kF;
      const bool valid = hr < a.head_rows;
      const uint32_t hrc = valid ? hr : a.head_rows - 1u;
      const uint32_t row = hrc / a.group, head = kv * a.group + hrc % a.group;
      const uint64_t rh = (uint64_t(b) * a.rows + row) * a.q_heads + head;
      const int64_t qpos = a.q_positions[uint64_t(b) * a.rows + row];
      const Visible vis = visible_tokens(a, e, valid, ask_visible(a, e, qpos, prefix));
      pre = vis.pre;
      const float l = a.l[rh];
      const bool counts = valid && l > 0.f;
      Block& w = blocks[i];
      if (kg == 0u) {
        w.lo[r] = vis.lo;
        w.hi[r] = vis.hi;
        w.m[r] = counts ? a.m[rh] : FLT_MAX;
        w.per_l[r] = counts && r % C::kF == 0u ? 1.f / l : 0.f;  // a head-row's F columns hold the same score
        w.slope[r] = a.slopes ? a.slopes[head] : 0.f;
        w.back[r] = near(int64_t(uint64_t(qpos) - uint64_t(qref)));
      }
      if (lane == 0u) {
        w.min_lo = vis.min_lo;
        w.max_hi = vis.max_hi;
      }
    }
    if (wave >= count && a.prefix) pre = visible_tokens(a, e, false, ask_visible(a, e, 0, prefix)).pre;  // the same for every row
    __syncthreads();
    uint32_t min_lo = 0xffffffffu, max_hi = 0u;
    for (uint32_t i = 0; i < count; ++i) {
      const uint32_t lo = blocks[i].min_lo, hi = blocks[i].max_hi;
      if (hi > 0u && lo < min_lo) min_lo = lo;
      if (hi > max_hi) max_hi = hi;
    }
    min_lo = uint32_t(__builtin_amdgcn_readfirstlane(int(min_lo)));
    max_hi = uint32_t(__builtin_amdgcn_readfirstlane(int(max_hi)));

    const auto live = [&](uint32_t t) {
      const uint32_t t0 = t * kTileTokens;
      return t0 < pre || (t0 < max_hi && t0 + kTileTokens > min_lo);
    };
    const auto next = [&](uint32_t t) {
      while (t < t_end && !live(t) && !(first == 0u && t * kTileTokens + kTileTokens > fresh0)) t += kWeightWaves;
      return t;
    };
    uint32_t t = next(t_begin + wave);
    if (t >= t_end) continue;
    // Page lookups of 16 of the wave's tiles at a time; tile t is its (t - t_begin) / 4-th.
    const auto tile_of = [&](uint32_t i) {
      const uint64_t x = uint64_t(t_begin) + wave + uint64_t(i) * kWeightWaves;
      return x < tiles ? uint32_t(x) : tiles - 1u;
    };
    const auto number = [&](uint32_t tile) { return (tile - t_begin) / kWeightWaves; };
    uint32_t window = number(t) / 16u;
    TilePages pages = tile_pages(a, e, tile_of, window * 16u, lane), pages_next = tile_pages(a, e, tile_of, window * 16u + 16u, lane);
    const auto rows_at = [&](uint32_t tile) {
      const uint32_t w = number(tile) / 16u;
      if (w != window) {
        pages = w == window + 1u ? pages_next : tile_pages(a, e, tile_of, w * 16u, lane);
        window = w;
        pages_next = tile_pages(a, e, tile_of, w * 16u + 16u, lane);
      }
      return tile_rows<ONE>(a, pages, number(tile), kv);
    };
    TileRows<ONE> rows = rows_at(t);
    int ahead = load_ahead<C>(a, e, t * kTileTokens, r, kg, qref);
    typename C::K k = C::template load_k<ONE>(a, rows, r, kg, e.tokens - t * kTileTokens);
    while (t < t_end) {
      const uint32_t t1 = next(t + kWeightWaves), tl = t1 < t_end ? t1 : t;
      const TileRows<ONE> rows1 = rows_at(tl);
      const int ahead1 = load_ahead<C>(a, e, tl * kTileTokens, r, kg, qref);
      const typename C::K k1 = C::template load_k<ONE>(a, rows1, r, kg, e.tokens - tl * kTileTokens);
      const uint32_t t0 = t * kTileTokens;
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (live(t)) {
        for (uint32_t i = 0; i < count; ++i) {
          asm volatile("" ::: "memory");  // the operands stay in LDS: not hoisted out of the loops
          const Block& w = blocks[i];
          float x[8];
          tile_scores<C, QD>(k, w.q, lane, x);
          const ScoreForm form = score_form(a, w.q.factor[r], w.slope[r], w.back[r]);
          apply_form<C>(a, form, ahead, t0, kg, true, w.lo[r], w.hi[r], pre, x);
          const float m = w.m[r], per_l = w.per_l[r];
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] = fmaf(per_l > 0.f ? exp_e(x[j] - m) : 0.f, per_l, sum[j]);
        }
      }
      float total = row_sum16(sum[0]);
      unrolled<1, 8>([&](auto jc) {
        const float s = row_sum16(sum[jc]);
        total = r == uint32_t(jc) ? s : total;
      });
      const uint32_t in = C::token(kg, r % 8u), tok = t0 + in;
      if (r < 8u && tok < e.tokens) {
        const uint32_t P = a.page_tokens;
        const uint64_t row = ONE ? rows.row(0, P) + in
                                 : pick(in / 8u, rows.row(0, P), rows.row(1, P), rows.row(2, P), rows.row(3, P)) + in % 8u;
        if (first == 0u && tok >= fresh0) a.weights[row] = total;
        else unsafeAtomicAdd(a.weights + row, total);
      }
      t = t1;
      rows = rows1;
      ahead = ahead1;
      k = k1;
    }
  }
}

template <class C, int QD>
hipError_t launch_digits(const ScoredArgs& a, hipStream_t stream) {
  const uint32_t groups = a.batch * a.chunks * a.kv_heads;
  const uint32_t bytes = uint32_t(sizeof(WeightBlock<C, QD>)) * (a.blocks < kBlocksAtOnce<C, QD> ? a.blocks : kBlocksAtOnce<C, QD>);
  if (a.page_tokens % kTileTokens == 0u) scored_weights_kernel<C, QD, true><<<groups, 64 * kWeightWaves, bytes, stream>>>(a);
  else scored_weights_kernel<C, QD, false><<<groups, 64 * kWeightWaves, bytes, stream>>>(a);
  return hipGetLastError();
}
template <class C>
hipError_t launch_cache(const ScoredArgs& a, hipStream_t stream) {
  if (a.q_type == 1u) return launch_digits<C, 2>(a, stream);
  return launch_digits<C, kQDigits<C, false>>(a, stream);
}

template <int G>
hipError_t launch_cache4(const ScoredArgs& a, hipStream_t stream) {  // as launch_attend_cache4
  if (a.head_rows <= 16u / G) return launch_cache<Cache4<G, G>>(a, stream);
  if constexpr (G > 2) {
    if (a.head_rows <= 32u / G) return launch_cache<Cache4<G, G / 2>>(a, stream);
  }
  return launch_cache<Cache4<G, 1>>(a, stream);
}

}  // namespace

hipError_t launch_scored_weights(const ScoredArgs& a, hipStream_t stream) {
  if (a.kv_bits == 4u) {
    if (a.dim == 64u) return launch_cache4<2>(a, stream);
    if (a.dim == 128u) return launch_cache4<4>(a, stream);
    return launch_cache4<8>(a, stream);
  }
  if (a.dim == 64u) return launch_cache<Cache8<2>>(a, stream);
  if (a.dim == 128u) return launch_cache<Cache8<4>>(a, stream);
  return launch_cache<Cache8<8>>(a, stream);
}

}  // namespace kvb
