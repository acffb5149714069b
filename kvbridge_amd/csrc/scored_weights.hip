// Attention weights per cached token (kvb_accumulate_weights).
//
// With m and l of an attention call known, the weight of token t for head-row
// r is exp(s_rt - m_r) / l_r: K is read once more, V not at all.  The items are
// those of the attention (scored.h, item_of) over the tiles that any row sees, a
// work-group's waves take an item's tiles in turn, so that a (page, kv head,
// slot) of a sequence is written by one wave only and in one order.  The
// operands of as many blocks of 16 head-rows as fit 64 KiB of LDS are staged at
// once and a tile's K serves all of them; more head-rows take another pass over
// the item.  Where a head-row has F columns, whose lanes all hold its scores,
// each of them goes on with 8 / F of the lane group's tokens; the sum over the
// head-rows of a block is then a DPP reduction over every F-th lane of a row.
//
// What bounds it: 16 ragged sequences of up to 32K tokens (32 heads over 8, dim
// 128) take 50 us, 3.7 TB/s of K and weights: 4,400 vector instructions a wave are
// 26 of them, and three waves a SIMD do not cover all waits for K.  Neither K
// requested two tiles ahead (49-50) nor plain stores in place of the atomics
// (59.3 against 60.5 at the time) changed that.  Two
// sequences of 7K under 64 head-rows of dim 64 over int8: 11 us, latency.
#include "scored.h"

namespace kvb {
namespace {

// Waves per SIMD that the registers allow (at dim 64 four: 64 head-rows over int8
// took 16 us with three, 11 with four; with a few spills outside the loop the
// dim-128 kernels gained nothing).
template <class C>
constexpr int kWeightOccupancy = C::kGroups == 8 || (C::kF > 1 && C::kH > 1) ? 2 : (C::kGroups == 2 && C::kF == 1 ? 4 : 3);

// Sum over the lanes r % F of a row.
template <int F>
__device__ __forceinline__ float rows_of_f_sum(float x) {
  x += row_ror<8>(x);
  if constexpr (F <= 4) x += row_ror<4>(x);
  if constexpr (F <= 2) x += row_ror<2>(x);
  if constexpr (F <= 1) x += row_ror<1>(x);
  return x;
}
// Of eight values the N = 8 / F from f * N on.
template <int F, typename T>
__device__ __forceinline__ void share_of(const T (&x)[8], uint32_t f, T (&y)[8 / F]) {
  constexpr int N = 8 / F;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    y[i] = x[i];
#pragma unroll
    for (int k = 1; k < F; ++k) y[i] = f == uint32_t(k) ? x[k * N + i] : y[i];
  }
}

// A block's head-rows next to their Q operands.
template <class C, int QD>
struct WeightBlock {
  QBlock<C, QD> q;
  uint32_t lo[16], hi[16];
  float m[16], per_l[16], slope[16];
  int back[16];
};
template <class C, int QD>  // 64 KiB less the static LDS
constexpr uint32_t kBlocksAtOnce = (65536u - 256u) / sizeof(WeightBlock<C, QD>);

template <class C, int QD, bool ONE>
__global__ __launch_bounds__((256 * kWeightOccupancy<C>), (kWeightOccupancy<C>)) void scored_weights_kernel(const ScoredArgs a) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  using Block = WeightBlock<C, QD>;
  Block* const blocks = reinterpret_cast<Block*>(lds_raw);
  constexpr int F = C::kF, N = 8 / F;
  __shared__ WorkItem plan_it;
  __shared__ uint32_t plan_found, plan_pre, plan_lo, plan_hi, plan_all_lo, plan_all_hi;
  const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, f = r % F, kg = lane >> 4, NW = blockDim.x >> 6;
  const uint32_t wave = uniform(threadIdx.x >> 6);
  const uint32_t kv = blockIdx.x % a.kv_heads, item = blockIdx.x / a.kv_heads;
  if (wave == 0u) {
    WorkItem w{0u, 0u, 0u, 0u, ScoredSeq{0u, 0u, 0u}};
    const bool found = item_of(a, item, w);
    if (lane == 0u) {
      plan_it = w;
      plan_found = found && w.e.tokens > 0u ? 1u : 0u;
    }
  }
  const uint32_t at_once = a.blocks < kBlocksAtOnce<C, QD> ? a.blocks : kBlocksAtOnce<C, QD>;
  for (uint32_t i = 0; i < at_once; ++i) clear_q(blocks[i].q, threadIdx.x, 64u * NW);
  __syncthreads();
  if (uniform(plan_found) == 0u) return;
  const uint32_t b = uniform(plan_it.seq), split = uniform(plan_it.split), shares = uniform(plan_it.count);
  const ScoredSeq e{uniform(plan_it.e.start), uniform(plan_it.e.tokens), uniform(plan_it.e.table_off)};
  const uint32_t tiles = (e.tokens - 1u) / kTileTokens + 1u;
  const uint32_t fresh0 = a.fresh < e.tokens ? e.tokens - a.fresh : 0u;  // tokens from here on are set
  const int64_t* q_positions = a.q_positions + uint64_t(b) * a.rows;
  const int64_t qref = q_positions[0], prefix = a.prefix ? a.prefix[b] : 0;
  const auto share = [&](uint32_t n) {
    const uint32_t per = n / shares + (n % shares != 0u ? 1u : 0u);
    return per > a.split_tiles ? per : a.split_tiles;
  };

  // The tokens that any row sees and those that all see, by the last wave: one
  // row per lane.
  if (wave == NW - 1u) {
    uint32_t lo = 0xffffffffu, hi = 0u, pre = 0u, all_lo = 0u, all_hi = 0xffffffffu;
    for (uint32_t row0 = 0; row0 < a.rows; row0 += 64u) {
      const bool valid = row0 + lane < a.rows;
      const Visible v = visible_tokens(a, e, valid, ask_visible(a, e, q_positions[valid ? row0 + lane : 0u], prefix));
      if (v.lo < v.hi) {
        lo = v.lo < lo ? v.lo : lo;
        hi = v.hi > hi ? v.hi : hi;
      }
      if (valid) {
        all_lo = v.lo > all_lo ? v.lo : all_lo;
        all_hi = v.hi < all_hi ? v.hi : all_hi;
      }
      pre = v.pre;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint32_t l3 = uint32_t(__shfl_xor(int(all_lo), o)), h3 = uint32_t(__shfl_xor(int(all_hi), o));
      all_lo = l3 > all_lo ? l3 : all_lo;
      all_hi = h3 < all_hi ? h3 : all_hi;
      const uint32_t l2 = uint32_t(__shfl_xor(int(lo), o)), h2 = uint32_t(__shfl_xor(int(hi), o));
      lo = l2 < lo ? l2 : lo;
      hi = h2 > hi ? h2 : hi;
    }
    if (lane == 0u) {
      plan_pre = pre;
      plan_lo = hi == 0u ? 0u : lo;
      plan_hi = hi;
      plan_all_lo = all_lo;
      plan_all_hi = all_hi;
    }
  }

  for (uint32_t first = 0; first < a.blocks; first += kBlocksAtOnce<C, QD>) {
    const uint32_t count = a.blocks - first < kBlocksAtOnce<C, QD> ? a.blocks - first : kBlocksAtOnce<C, QD>;
    if (first > 0u) {
      __threadfence();  // what the first pass set is in place before it is added to
      __syncthreads();  // and every wave is done with the last pass's operands
    }
    // Q by groups of four waves, what else a head-row needs by single waves.
    for (uint32_t i = wave >> 2; i < count; i += NW >> 2) {
      const uint32_t tid = threadIdx.x & 255u, hr = (first + i) * 16u + tid / 16u;
      stage_q<C, QD>(a, (uint64_t(b) * a.rows + hr / a.group) * a.q_stride + uint64_t(kv * a.group + hr % a.group) * a.dim,
                     hr < a.head_rows, blocks[i].q, tid);
    }
    for (uint32_t i = wave; i < count; i += NW) {
      const uint32_t hr = (first + i) * 16u + r / C::kF;
      const bool valid = hr < a.head_rows;
      const uint32_t hrc = valid ? hr : a.head_rows - 1u;
      const uint32_t row = hrc / a.group, head = kv * a.group + hrc % a.group;
      const uint64_t rh = (uint64_t(b) * a.rows + row) * a.q_heads + head;
      const int64_t qpos = q_positions[row];
      const float l = a.l[rh], m = a.m[rh];
      const Visible vis = visible_tokens(a, e, valid, ask_visible(a, e, qpos, prefix));
      const bool counts = valid && l > 0.f;
      Block& w = blocks[i];
      if (kg == 0u) {
        w.lo[r] = vis.lo;
        w.hi[r] = vis.hi;
        w.m[r] = counts ? m : FLT_MAX;
        w.per_l[r] = counts ? 1.f / l : 0.f;
        w.slope[r] = a.slopes ? a.slopes[head] : 0.f;
        w.back[r] = near(int64_t(uint64_t(qpos) - uint64_t(qref)));
      }
    }
    __syncthreads();
    const uint32_t pre = uniform(plan_pre), all_lo = uniform(plan_all_lo), all_hi = uniform(plan_all_hi);
    const LiveTiles live = live_tiles(pre, uniform(plan_lo), uniform(plan_hi));
    const uint32_t per = share(live.n);
    const uint32_t t_first = split * per + wave;
    const uint32_t t_end = split * per >= live.n ? 0u : (live.n - split * per > per ? split * per + per : live.n);
    const uint32_t n = t_first < t_end ? (t_end - t_first + NW - 1u) / NW : 0u;
    const auto tile_of = [&](uint32_t i) {
      const uint64_t x = uint64_t(t_first) + uint64_t(i) * NW;
      return live.tile(x < live.n ? uint32_t(x) : live.n - 1u);
    };
    if (n > 0u) {
      TilePages pages = tile_pages(a, e, tile_of, 0u, lane), ahead_pages = pages;
      TileRows<ONE> rows = tile_rows<ONE>(a, pages, 0u, kv);
      uint32_t t0 = tile_of(0u) * kTileTokens;
      typename C::K k = C::template load_k<ONE>(a, rows, r, kg, e.tokens - t0);
      int ahead = load_ahead<C>(a, e, t0, r, kg, qref);
      for (uint32_t i = 0; i < n; ++i) {
        if (i % 16u == 0u) ahead_pages = tile_pages(a, e, tile_of, i + 16u, lane);
        const uint32_t t_next = tile_of(i + 1u < n ? i + 1u : i) * kTileTokens;
        if ((i + 1u) % 16u == 0u) pages = ahead_pages;
        const TileRows<ONE> rows_next = tile_rows<ONE>(a, pages, i + 1u < n ? i + 1u : i, kv);
        const typename C::K k_next = C::template load_k<ONE>(a, rows_next, r, kg, e.tokens - t_next);
        const int ahead_next = load_ahead<C>(a, e, t_next, r, kg, qref);
        const bool whole = t0 + kTileTokens <= pre || (t0 >= all_lo && t0 + kTileTokens <= all_hi);
        float sum[N];
#pragma unroll
        for (int i2 = 0; i2 < N; ++i2) sum[i2] = 0.f;
        for (uint32_t bl = 0; bl < count; ++bl) {
          asm volatile("" ::: "memory");  // the operands stay in LDS: not hoisted out of the loops
          const Block& w = blocks[bl];
          float x[8], y[N];
          tile_scores<C, QD>(k, w.q, lane, x);
          share_of<F>(x, f, y);
          const ScoreForm form = score_form(a, w.q.factor[r], w.slope[r], w.back[r]);
          apply_form<N>(a, form, !whole, w.lo[r], w.hi[r], pre, [&](int j) { return t0 + C::token(kg, f * N + j); },
                        [&](int(&d)[N]) {
                          int all[8];
                          unrolled<0, 8>([&](auto j) { all[j] = bci<j>(ahead); });
                          share_of<F>(all, f, d);
                        },
                        y);
          const float m = w.m[r], per_l = w.per_l[r];
#pragma unroll
          for (int i2 = 0; i2 < N; ++i2) sum[i2] = fmaf(exp_e(y[i2] - m), per_l, sum[i2]);
        }
        // Lane i F + f of the row's first eight writes its lanes' token i.
        float total = rows_of_f_sum<F>(sum[0]);
        unrolled<1, N>([&](auto jc) {
          const float s = rows_of_f_sum<F>(sum[jc]);
          total = r / F == uint32_t(jc) ? s : total;
        });
        const uint32_t in = C::token(kg, f * N + r % 8u / F), tok = t0 + in;
        if (r < 8u && tok < e.tokens) {
          const uint32_t P = a.page_tokens;
          const uint64_t at = ONE ? rows.row(0, P) + in
                                  : pick(in / 8u, rows.row(0, P), rows.row(ONE ? 0 : 1, P), rows.row(ONE ? 0 : 2, P), rows.row(ONE ? 0 : 3, P)) + in % 8u;
          if (first == 0u && tok >= fresh0) a.weights[at] = total;
          else unsafeAtomicAdd(a.weights + at, total);
        }
        k = k_next;
        rows = rows_next;
        t0 = t_next;
        ahead = ahead_next;
      }
    }
    // Fresh tokens of the tiles that no row sees: 0.
    if (first == 0u) {
      const uint32_t live_end = live.first + (live.n - live.pre_tiles);
      for (uint64_t t = uint64_t(fresh0 / kTileTokens) + split * NW + wave; t < tiles; t += uint64_t(shares) * NW) {
        if (t < live.pre_tiles || (t >= live.first && t < live_end)) continue;
        const uint32_t tok = uint32_t(t) * kTileTokens + lane;
        if (lane >= kTileTokens || tok < fresh0 || tok >= e.tokens) continue;
        const uint32_t lp = tok / a.page_tokens;
        uint32_t page = a.page_table[e.table_off + lp];
        page = page < a.pages ? page : a.pages - 1u;
        a.weights[(uint64_t(page) * a.kv_heads + kv) * a.page_tokens + (tok - lp * a.page_tokens)] = 0.f;
      }
    }
  }
}

template <class C, int QD>
hipError_t launch_digits(const ScoredArgs& a, hipStream_t stream) {
  const uint32_t groups = a.items * a.kv_heads, most = 4u * uint32_t(kWeightOccupancy<C>), waves = a.waves < most ? a.waves : most;
  const uint32_t bytes = uint32_t(sizeof(WeightBlock<C, QD>)) * (a.blocks < kBlocksAtOnce<C, QD> ? a.blocks : kBlocksAtOnce<C, QD>);
  if (a.page_tokens % kTileTokens == 0u) scored_weights_kernel<C, QD, true><<<groups, 64u * waves, bytes, stream>>>(a);
  else scored_weights_kernel<C, QD, false><<<groups, 64u * waves, bytes, stream>>>(a);
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
  if constexpr (G == 8) {
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

hipError_t preload_scored_weights() {
  hipFuncAttributes attr;
  return hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&scored_weights_kernel<Cache4<2, 1>, 2, true>));
}

}  // namespace kvb
