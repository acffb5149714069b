// Attention weights per cached token (kvb_accumulate_weights).
//
// With m and l of an attention call known, the weight of token t for head-row
// r is exp(s_rt - m_r) / l_r: K is read once more, V not at all.  A work-group
// of four waves takes chunk_tiles tiles of one (sequence, kv head), its waves
// every fourth tile, all blocks of 16 head-rows one after the other, so that a
// (page, kv head, slot) of a sequence is written by one wave only and in one
// order.  The sum over the head-rows of a block is a DPP reduction over the 16
// lanes of a row.
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

template <class C, int QD>
__global__ __launch_bounds__(64 * kWeightWaves) void scored_weights_kernel(const ScoredArgs a) {
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
  const int64_t qref = a.q_positions[uint64_t(b) * a.rows];

  for (uint32_t block = 0; block < a.blocks; ++block) {
    if (block > 0u) __threadfence();  // what block 0 set is in place before it is added to
    const uint32_t hr = block * 16u + r;
    const bool valid = hr < a.head_rows;
    const uint32_t hrc = valid ? hr : a.head_rows - 1u;
    const uint32_t row = hrc / a.group, head = kv * a.group + hrc % a.group;
    const uint64_t rh = (uint64_t(b) * a.rows + row) * a.q_heads + head;
    const int64_t qpos = a.q_positions[uint64_t(b) * a.rows + row];
    const Visible vis = visible_tokens(a, e, b, valid, qpos);
    const float l = a.l[rh];
    const bool counts = valid && l > 0.f;
    const float m = counts ? a.m[rh] : FLT_MAX, per_l = counts ? 1.f / l : 0.f;
    const uint64_t q_at = (uint64_t(b) * a.rows + row) * a.q_stride + uint64_t(head) * a.dim;
    const QBlock<C, QD> q = load_q<C, QD>(a, q_at, valid, kg);
    const ScoreForm form = score_form(a, q.factor, a.slopes ? a.slopes[head] : 0.f, near(int64_t(uint64_t(qpos) - uint64_t(qref))));

    const auto live = [&](uint32_t t) {
      const uint32_t t0 = t * kTileTokens;
      return t0 < vis.pre || (t0 < vis.max_hi && t0 + kTileTokens > vis.min_lo);
    };
    const auto next = [&](uint32_t t) {
      while (t < t_end && !live(t) && !(block == 0u && t * kTileTokens + kTileTokens > fresh0)) t += kWeightWaves;
      return t;
    };
    uint32_t t = next(t_begin + wave);
    if (t >= t_end) continue;
    const auto load = [&](uint32_t tile, TileRows& rows, int& ahead) {
      const TilePages pages = tile_pages(a, e, [&](uint32_t) { return tile; }, 0u, lane);
      rows = tile_rows(a, pages, 0u, kv);
      ahead = load_ahead<C>(a, e, tile * kTileTokens, r, kg, qref);
      return C::load_k(a, rows, r, kg, e.tokens - tile * kTileTokens);
    };
    TileRows rows;
    int ahead;
    typename C::K k = load(t, rows, ahead);
    while (t < t_end) {
      const uint32_t t1 = next(t + kWeightWaves);
      TileRows rows1;
      int ahead1;
      const typename C::K k1 = load(t1 < t_end ? t1 : t, rows1, ahead1);
      const uint32_t t0 = t * kTileTokens;
      float x[8];
      if (live(t)) {
        tile_scores<C, QD>(k, q, x);
        apply_form<C, true>(a, form, ahead, t0, kg, vis, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = row_sum16(counts ? exp_e(x[j] - m) * per_l : 0.f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
      }
      float w = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) w = r == uint32_t(j) ? x[j] : w;
      const uint32_t in = C::token(kg, r % 8u), tok = t0 + in;
      if (r < 8u && tok < e.tokens) {
        float* p = a.weights + pick(in / 8u, rows.run[0], rows.run[1], rows.run[2], rows.run[3]) + in % 8u;
        if (block == 0u && tok >= fresh0) *p = w;
        else unsafeAtomicAdd(p, w);
      }
      t = t1;
      rows = rows1;
      ahead = ahead1;
      k = k1;
    }
  }
}

template <class C>
hipError_t launch_cache(const ScoredArgs& a, hipStream_t stream) {
  const uint32_t groups = a.batch * a.chunks * a.kv_heads;
  if (a.q_type == 1u) scored_weights_kernel<C, 2><<<groups, 64 * kWeightWaves, 0, stream>>>(a);
  else scored_weights_kernel<C, kQDigits<C, false>><<<groups, 64 * kWeightWaves, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_scored_weights(const ScoredArgs& a, hipStream_t stream) {
  if (a.kv_bits == 4u) {
    if (a.dim == 64u) return launch_cache<Cache4<2>>(a, stream);
    if (a.dim == 128u) return launch_cache<Cache4<4>>(a, stream);
    return launch_cache<Cache4<8>>(a, stream);
  }
  if (a.dim == 64u) return launch_cache<Cache8<2>>(a, stream);
  if (a.dim == 128u) return launch_cache<Cache8<4>>(a, stream);
  return launch_cache<Cache8<8>>(a, stream);
}

}  // namespace kvb
