// Eviction by accumulated weight (kvb_evict_select, kvb_evict_move).
//
// Selection: evict_keys_kernel forms each token's key, an order-preserving
// uint32 of its weight (the kv heads summed in fp64, rounded to fp32; always-
// kept tokens the largest key, NaN the least).  evict_pick_kernel, one
// work-group per sequence, finds the key of rank n by three radix passes of 11,
// 11 and 10 bits over LDS histograms, the keys of up to 32K tokens staying in
// registers, then writes the tokens in order: above the key they stay, of those
// equal to it the first ones.
// Move: one work-group per 64 kept tokens and kv head copies rows in 16-byte
// pieces (int8 V, dim-major, byte by byte gathered to dwords).
// Measured at 16 sequences of up to 32K tokens cut to 4,096, 8 kv heads of dim
// 128, 4 bits: keys 6.0 us (8.5 with a token per thread), pick 19.5 (a work-group
// per sequence; 22.5 with bounds checked at every key and six barriers a pass
// instead of three), move 50-70 (168 MB of rows; kept rows of 64 bytes share the
// memory's 128-byte lines with others: four heads to a work-group changed
// nothing).  Two sequences of 2K: 2.3, 8.2 and 6.8.
#include "device_common.h"
#include "scored.h"

namespace kvb {
namespace {

typedef uint32_t u32x4_e __attribute__((ext_vector_type(4)));

constexpr uint32_t kPickThreads = 1024, kPickWaves = kPickThreads / 64, kBins = 2048;

__device__ __forceinline__ ScoredSeq evict_seq(const EvictArgs& a, uint32_t b) {
  return clamp_seq(a.seq_starts[b], a.seq_starts[b + 1u], a.page_offsets[b], a.total_tokens, a.table_entries, a.page_tokens,
                   a.max_tokens);
}

// Four tokens a thread, which share a page (page_tokens is a multiple of 8).
template <bool VEC>
__global__ __launch_bounds__(256) void evict_keys_kernel(const EvictArgs a) {
  const uint32_t b = blockIdx.y, t = (blockIdx.x * 256u + threadIdx.x) * 4u;
  const ScoredSeq e = evict_seq(a, b);
  if (t >= e.tokens || e.tokens <= a.keep) return;  // all stay: no key is looked at
  const uint32_t lp = t / a.page_tokens, slot = t - lp * a.page_tokens;
  uint32_t page = a.page_table[e.table_off + lp];
  page = page < a.pages ? page : a.pages - 1u;
  const float* w = a.weights_in + uint64_t(page) * a.kv_heads * a.page_tokens + slot;
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  for (uint32_t h0 = 0; h0 < a.kv_heads; h0 += 8u) {  // eight heads' loads at once
    f32x4 x[8];
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
      const float* p = w + uint64_t(h0 + i) * a.page_tokens;
      x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (h0 + i >= a.kv_heads) continue;
      if constexpr (VEC) x[i] = *reinterpret_cast<const f32x4*>(p);
      else x[i] = f32x4{p[0], p[1], p[2], p[3]};
    }
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
      for (uint32_t c = 0; c < 4u; ++c) sum[c] += double(x[i][c]);
  }
  u32x4_e keys;
#pragma unroll
  for (uint32_t c = 0; c < 4u; ++c) {
    const float f = float(sum[c]) + 0.f;  // -0 becomes 0
    const uint32_t u = __float_as_uint(f), key = f != f ? 0u : ((u >> 31) != 0u ? ~u : u | 0x80000000u);
    keys[c] = t + c >= a.sink && t + c + a.recent < e.tokens ? key : 0xffffffffu;
  }
  *reinterpret_cast<u32x4_e*>(a.scratch + uint64_t(b) * a.scratch_stride + t) = keys;
}

// A thread's keys of a chunk of up to 32K tokens: 4 * rounds consecutive ones
// (rounds: as few as cover the sequence).
constexpr uint32_t kLaneKeys = 8, kChunkKeys = kPickThreads * 4 * kLaneKeys;
struct LaneKeys {
  u32x4_e k[kLaneKeys];
  uint32_t rounds, first;  // first: the thread's first token
  __device__ __forceinline__ uint32_t token(uint32_t i, uint32_t c) const { return first + i * 4u + c; }
  // All loads at once.  Past the last token, where the scratch holds anything, the
  // least key: it comes after every token of the same key and is never reached.
  __device__ __forceinline__ void load(const uint32_t* keys, uint32_t chunk, uint32_t tokens, uint32_t stride) {
    rounds = tokens >= kChunkKeys ? kLaneKeys : (tokens + kPickThreads * 4u - 1u) / (kPickThreads * 4u);
    first = chunk * kChunkKeys + threadIdx.x * (4u * rounds);
#pragma unroll
    for (uint32_t i = 0; i < kLaneKeys; ++i) {
      const uint32_t t = token(i, 0u);
      k[i] = i < rounds && t < stride ? *reinterpret_cast<const u32x4_e*>(keys + t) : u32x4_e{0u, 0u, 0u, 0u};
    }
    if (first + 4u * rounds > tokens) {
#pragma unroll
      for (uint32_t i = 0; i < kLaneKeys; ++i)
#pragma unroll
        for (uint32_t c = 0; c < 4u; ++c) k[i][c] = token(i, c) < tokens ? k[i][c] : 0u;
    }
  }
};

// The keys' sums over the threads before this one, and over all.
struct Before {
  uint32_t mine, all;
};
__device__ __forceinline__ Before sum_before(uint32_t x, uint32_t (&waves)[kPickWaves]) {
  const uint32_t upto = wave_scan(x), wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63u) == 63u) waves[wave] = upto;
  __syncthreads();
  Before r{upto - x, 0u};
#pragma unroll
  for (uint32_t w = 0; w < kPickWaves; ++w) {
    const uint32_t n = waves[w];
    r.mine += w < wave ? n : 0u;
    r.all += n;
  }
  return r;
}

__global__ __launch_bounds__(kPickThreads) void evict_pick_kernel(const EvictArgs a) {
  // The three passes' histograms beside each other, so that one barrier clears
  // all of them.  Most keys share few leading digits: neighbouring lanes count in
  // copies of their own, which begin in different banks.
  constexpr uint32_t kBinsOf[3] = {kBins, kBins, 1024u}, kCopiesOf[3] = {4u, 2u, 2u}, kShift = 8u;
  __shared__ uint32_t hist[4u * (kBins + kShift) + 2u * (kBins + kShift) + 2u * (1024u + kShift)];
  __shared__ uint32_t found[3][2], waves[3][kPickWaves], wave_gt[kPickWaves], wave_eq[kPickWaves];
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = uint32_t(__builtin_amdgcn_readfirstlane(int(tid >> 6)));
  const ScoredSeq e = evict_seq(a, b);
  const uint32_t n = e.tokens < a.keep ? e.tokens : a.keep;
  uint32_t* kept = a.kept + uint64_t(b) * a.keep;
  const uint32_t* keys = a.scratch + uint64_t(b) * a.scratch_stride;
  const uint32_t chunks = (e.tokens + kChunkKeys - 1u) / kChunkKeys;
  LaneKeys own;
  if (n < e.tokens) own.load(keys, 0u, e.tokens, a.scratch_stride);
  if (wave == 0u) {  // tokens kept before this sequence; the last one also closes the list
    uint32_t sum = 0;
    for (uint32_t i = lane; i < b; i += 64u) {
      const uint32_t t = evict_seq(a, i).tokens;
      sum += t < a.keep ? t : a.keep;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += uint32_t(__shfl_xor(int(sum), o));
    if (lane == 0u) {
      a.kept_starts[b] = sum;
      if (b + 1u == a.batch) a.kept_starts[a.batch] = sum + n;
    }
  }
  if (n == e.tokens) {
    for (uint32_t t = tid; t < n; t += kPickThreads) kept[t] = t;
    return;
  }

  // The n-th largest key: its digits from the top, `want` its rank among the
  // keys that share the digits found so far.
  for (uint32_t i = tid; i < sizeof(hist) / 4u; i += kPickThreads) hist[i] = 0u;
  __syncthreads();
  uint32_t prefix = 0, mask = 0, want = n;
  uint32_t* bins = hist;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t digits = kBinsOf[pass], copies = kCopiesOf[pass], stride = digits + kShift;
    uint32_t* const h = bins + lane % copies * stride;
    for (uint32_t chunk = 0; chunk < chunks; ++chunk) {
      if (chunks > 1u) own.load(keys, chunk, e.tokens, a.scratch_stride);
#pragma unroll
      for (uint32_t i = 0; i < kLaneKeys; ++i) {
        if (i >= own.rounds) break;
        if (own.token(i, 0u) >= e.tokens) continue;
#pragma unroll
        for (uint32_t c = 0; c < 4u; ++c)
          if (pass == 0 || (own.k[i][c] & mask) == prefix) atomicAdd(&h[(own.k[i][c] >> shift) & (digits - 1u)], 1u);
      }
    }
    __syncthreads();
    // Thread t has the bins top - 2 t and the next below (one bin in the last pass).
    const uint32_t per = digits / kPickThreads, bin = digits - 1u - tid * per;
    uint32_t c0 = 0, c1 = 0;
#pragma unroll
    for (uint32_t c = 0; c < copies; ++c) {
      c0 += bins[c * stride + bin];
      c1 += per == 2u ? bins[c * stride + bin - 1u] : 0u;
    }
    const uint32_t before = sum_before(c0 + c1, waves[pass]).mine;
    if (before < want && want <= before + c0 + c1) {
      const bool second = want > before + c0;
      found[pass][0] = second ? bin - 1u : bin;
      found[pass][1] = want - before - (second ? c0 : 0u);
    }
    __syncthreads();
    prefix |= found[pass][0] << shift;
    want = found[pass][1];
    mask |= (digits - 1u) << shift;
    bins += copies * stride;
  }

  // Chunk by chunk: a thread's first place is the number of keys before its own
  // that are above the n-th, and of those equal to it the first `want`.
  uint32_t gt0 = 0, eq0 = 0;
  for (uint32_t chunk = 0; chunk < chunks; ++chunk) {
    if (chunks > 1u) own.load(keys, chunk, e.tokens, a.scratch_stride);
    uint32_t gt = 0, eq = 0;
#pragma unroll
    for (uint32_t i = 0; i < kLaneKeys; ++i)
#pragma unroll
      for (uint32_t c = 0; c < 4u; ++c) {
        gt += own.k[i][c] > prefix ? 1u : 0u;
        eq += own.k[i][c] == prefix ? 1u : 0u;
      }
    if (chunk > 0u) __syncthreads();  // the last chunk's sums have been read
    const Before g = sum_before(gt, wave_gt), q = sum_before(eq, wave_eq);
    uint32_t rank = eq0 + q.mine, to = gt0 + g.mine + (rank < want ? rank : want);
    gt0 += g.all;
    eq0 += q.all;
#pragma unroll
    for (uint32_t i = 0; i < kLaneKeys; ++i) {
      if (i >= own.rounds) break;
#pragma unroll
      for (uint32_t c = 0; c < 4u; ++c) {
        const bool is_eq = own.k[i][c] == prefix;
        if (own.k[i][c] > prefix || (is_eq && rank < want)) kept[to++] = own.token(i, c);
        rank += is_eq ? 1u : 0u;
      }
    }
  }
}

// Rows of a destination token: where it comes from and goes to, ~0 if nowhere.
constexpr uint32_t kMoveTokens = 64;

// Pieces P of the rows of `row_bytes` at p, every thread's loads of all of them
// before any store: with a loop of load and store for each array the move of
// 65,536 tokens took 69 us.
template <typename P, uint32_t ROW_BYTES>
struct Pieces {
  static constexpr uint32_t kPer = ROW_BYTES / uint32_t(sizeof(P)), kN = (kMoveTokens * kPer + 255u) / 256u;
  P v[kN];
  template <typename F>
  __device__ __forceinline__ void load(const void* p, F row) {
#pragma unroll
    for (uint32_t k = 0; k < kN; ++k) {
      const uint32_t i = threadIdx.x + 256u * k;
      const uint64_t at = row(i / kPer);
      if (at != ~0ull) v[k] = *reinterpret_cast<const P*>(static_cast<const uint8_t*>(p) + at * ROW_BYTES + i % kPer * sizeof(P));
    }
  }
  template <typename F>
  __device__ __forceinline__ void store(void* p, F row) const {
#pragma unroll
    for (uint32_t k = 0; k < kN; ++k) {
      const uint32_t i = threadIdx.x + 256u * k;
      const uint64_t at = row(i / kPer);
      if (at != ~0ull) *reinterpret_cast<P*>(static_cast<uint8_t*>(p) + at * ROW_BYTES + i % kPer * sizeof(P)) = v[k];
    }
  }
};

template <int BITS, int G>
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictArgs a) {
  constexpr uint32_t D = 32u * G;
  __shared__ uint32_t from_page[kMoveTokens], from_slot[kMoveTokens], to_page[kMoveTokens], to_slot[kMoveTokens];
  const uint32_t b = blockIdx.z, kv = blockIdx.y, j0 = blockIdx.x * kMoveTokens, tid = threadIdx.x;
  const ScoredSeq e = evict_seq(a, b);
  const uint32_t n = e.tokens < a.keep ? e.tokens : a.keep;
  if (j0 >= n) return;
  const uint32_t count = n - j0 < kMoveTokens ? n - j0 : kMoveTokens;
  if (tid < kMoveTokens) {
    uint32_t fp = 0, fs = 0, tp = 0xffffffffu, ts = 0;
    if (tid < count) {
      const uint32_t j = j0 + tid, src = a.kept[uint64_t(b) * a.keep + j];
      const uint32_t dlp = j / a.page_tokens;
      const uint64_t entry = uint64_t(a.dst_offsets[b]) + dlp;
      if (src < e.tokens && entry < a.dst_entries) {
        const uint32_t slp = src / a.page_tokens;
        fp = a.page_table[e.table_off + slp];
        fs = src - slp * a.page_tokens;
        tp = a.dst_table[entry];
        ts = j - dlp * a.page_tokens;
        if (fp >= a.pages || tp >= a.pages) tp = 0xffffffffu;
        if (kv == 0u && a.positions) {
          const uint64_t at = uint64_t(a.kept_starts[b]) + j;
          if (at < uint64_t(a.batch) * a.keep) a.positions[at] = a.k_positions[e.start + src];
        }
      }
    }
    from_page[tid] = fp;
    from_slot[tid] = fs;
    to_page[tid] = tp;
    to_slot[tid] = ts;
  }
  __syncthreads();
  // Row numbers; ~0 past the last token and where there is no destination.
  const auto row = [&](uint32_t page, uint32_t slot) { return (uint64_t(page) * a.kv_heads + kv) * a.page_tokens + slot; };
  const auto from = [&](uint32_t t) { return t < kMoveTokens && to_page[t] != 0xffffffffu ? row(from_page[t], from_slot[t]) : ~0ull; };
  const auto to = [&](uint32_t t) { return t < kMoveTokens && to_page[t] != 0xffffffffu ? row(to_page[t], to_slot[t]) : ~0ull; };
  Pieces<float, 4> w;
  if (a.weights) w.load(a.weights, from);
  if constexpr (BITS == 4) {
    Pieces<u32x4_e, D / 2u> k, v;
    Pieces<uint64_t, 4u * G> ks, vs;
    k.load(a.k, from);
    v.load(a.v, from);
    ks.load(a.k_scales, from);
    vs.load(a.v_scales, from);
    k.store(a.k, to);
    v.store(a.v, to);
    ks.store(a.k_scales, to);
    vs.store(a.v_scales, to);
  } else {
    Pieces<u32x4_e, D> k;
    Pieces<float, 4> ks, vs;
    k.load(a.k, from);
    ks.load(a.k_scales, from);
    vs.load(a.v_scales, from);
    // V: four tokens of a dim to a dword: j0 and page_tokens are multiples of 8,
    // so the four slots are one aligned dword of one page.  The last, partial
    // four go byte by byte: the slots behind are not this call's.
    uint8_t* v = static_cast<uint8_t*>(a.v);
    const auto place = [&](uint32_t page, uint32_t slot, uint32_t d) {
      return ((uint64_t(page) * a.kv_heads + kv) * D + d) * a.page_tokens + slot;
    };
    const uint32_t qd = tid % 16u, t0 = 4u * qd;
    bool in[4], whole = true;
#pragma unroll
    for (uint32_t c = 0; c < 4u; ++c) {
      in[c] = to_page[t0 + c] != 0xffffffffu;
      whole = whole && in[c];
    }
    constexpr uint32_t kDims = D / 16u < 8u ? D / 16u : 8u;  // of a thread at once
    for (uint32_t d0 = tid / 16u; d0 < D; d0 += 16u * kDims) {
      uint8_t x[kDims][4];
#pragma unroll
      for (uint32_t i = 0; i < kDims; ++i)
#pragma unroll
        for (uint32_t c = 0; c < 4u; ++c) x[i][c] = in[c] ? v[place(from_page[t0 + c], from_slot[t0 + c], d0 + 16u * i)] : uint8_t(0);
#pragma unroll
      for (uint32_t i = 0; i < kDims; ++i) {
        if (whole) {
          *reinterpret_cast<uint32_t*>(v + place(to_page[t0], to_slot[t0], d0 + 16u * i)) =
              uint32_t(x[i][0]) | uint32_t(x[i][1]) << 8 | uint32_t(x[i][2]) << 16 | uint32_t(x[i][3]) << 24;
        } else {
#pragma unroll
          for (uint32_t c = 0; c < 4u; ++c)
            if (in[c]) v[place(to_page[t0 + c], to_slot[t0 + c], d0 + 16u * i)] = x[i][c];
        }
      }
    }
    k.store(a.k, to);
    ks.store(a.k_scales, to);
    vs.store(a.v_scales, to);
  }
  if (a.weights) w.store(a.weights, to);
}

}  // namespace

hipError_t launch_evict_select(const EvictArgs& a, hipStream_t stream) {
  const dim3 grid(a.max_tokens / 1024u + (a.max_tokens % 1024u != 0u ? 1u : 0u), a.batch);
  if (reinterpret_cast<uintptr_t>(a.weights_in) % 16u == 0u) evict_keys_kernel<true><<<grid, 256, 0, stream>>>(a);
  else evict_keys_kernel<false><<<grid, 256, 0, stream>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  evict_pick_kernel<<<a.batch, kPickThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_evict_move(const EvictArgs& a, hipStream_t stream) {
  const uint32_t most = a.keep < a.max_tokens ? a.keep : a.max_tokens;
  const dim3 grid(most / kMoveTokens + (most % kMoveTokens != 0u ? 1u : 0u), a.kv_heads, a.batch);
  if (a.kv_bits == 4u) {
    if (a.dim == 64u) evict_move_kernel<4, 2><<<grid, 256, 0, stream>>>(a);
    else if (a.dim == 128u) evict_move_kernel<4, 4><<<grid, 256, 0, stream>>>(a);
    else evict_move_kernel<4, 8><<<grid, 256, 0, stream>>>(a);
  } else {
    if (a.dim == 64u) evict_move_kernel<8, 2><<<grid, 256, 0, stream>>>(a);
    else if (a.dim == 128u) evict_move_kernel<8, 4><<<grid, 256, 0, stream>>>(a);
    else evict_move_kernel<8, 8><<<grid, 256, 0, stream>>>(a);
  }
  return hipGetLastError();
}

hipError_t preload_evict() {
  hipFuncAttributes attr;
  return hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&evict_keys_kernel<true>));
}

}  // namespace kvb
