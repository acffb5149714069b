// Eviction by accumulated weight (kvb_evict_select, kvb_evict_move).
//
// Selection: evict_keys_kernel forms each token's key, an order-preserving
// uint32 of its weight (the kv heads summed in fp64, rounded to fp32; always-
// kept tokens the largest key, NaN the least).  evict_pick_kernel, one
// work-group per sequence, finds the key of rank n by three radix passes of 11,
// 11 and 10 bits over LDS histograms, then lets every wave run over its share
// of the tokens in order: above the key they stay, of those equal to it the
// first ones.
// Move: one work-group per 64 kept tokens and kv head copies rows in 16-byte
// pieces (int8 V, dim-major, byte by byte gathered to dwords).
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

__global__ __launch_bounds__(256) void evict_keys_kernel(const EvictArgs a) {
  const uint32_t b = blockIdx.y, t = blockIdx.x * 256u + threadIdx.x;
  const ScoredSeq e = evict_seq(a, b);
  if (t >= e.tokens) return;
  uint32_t key = 0xffffffffu;
  if (t >= a.sink && e.tokens - t > a.recent) {
    const uint32_t lp = t / a.page_tokens, slot = t - lp * a.page_tokens;
    uint32_t page = a.page_table[e.table_off + lp];
    page = page < a.pages ? page : a.pages - 1u;
    const float* w = a.weights_in + uint64_t(page) * a.kv_heads * a.page_tokens + slot;
    double sum = 0.0;
    for (uint32_t h = 0; h < a.kv_heads; ++h) sum += double(w[uint64_t(h) * a.page_tokens]);
    const float f = float(sum) + 0.f;  // -0 becomes 0
    const uint32_t u = __float_as_uint(f);
    key = f != f ? 0u : ((u >> 31) != 0u ? ~u : u | 0x80000000u);
  }
  a.scratch[uint64_t(b) * a.max_tokens + t] = key;
}

__global__ __launch_bounds__(kPickThreads) void evict_pick_kernel(const EvictArgs a) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t found[2], wave_gt[kPickWaves], wave_eq[kPickWaves];
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = uint32_t(__builtin_amdgcn_readfirstlane(int(tid >> 6)));
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
      if (b + 1u == a.batch) {
        const uint32_t t = evict_seq(a, b).tokens;
        a.kept_starts[a.batch] = sum + (t < a.keep ? t : a.keep);
      }
    }
  }
  const ScoredSeq e = evict_seq(a, b);
  const uint32_t n = e.tokens < a.keep ? e.tokens : a.keep;
  uint32_t* kept = a.kept + uint64_t(b) * a.keep;
  if (n == e.tokens) {
    for (uint32_t t = tid; t < n; t += kPickThreads) kept[t] = t;
    return;
  }
  const uint32_t* keys = a.scratch + uint64_t(b) * a.max_tokens;

  // The n-th largest key: its digits from the top, `want` its rank among the
  // keys that share the digits found so far.
  uint32_t prefix = 0, mask = 0, want = n;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t digits = pass == 2 ? 1024u : kBins;
    for (uint32_t i = tid; i < kBins; i += kPickThreads) hist[i] = 0u;
    __syncthreads();
    for (uint32_t t = tid; t < e.tokens; t += kPickThreads) {
      const uint32_t key = keys[t];
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & (digits - 1u)], 1u);
    }
    __syncthreads();
    if (wave == 0u) {  // lane l: bins from the top, digits / 64 each
      const uint32_t per = digits / 64u, top = digits - 1u - lane * per;
      uint32_t sum = 0;
      for (uint32_t i = 0; i < per; ++i) sum += hist[top - i];
      uint32_t upto = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = uint32_t(__shfl_up(int(upto), o));
        if (lane >= uint32_t(o)) upto += v;
      }
      uint32_t before = upto - sum;
      if (before < want && want <= upto) {
        for (uint32_t i = 0; i < per; ++i) {
          const uint32_t c = hist[top - i];
          if (want <= before + c) {
            found[0] = top - i;
            found[1] = want - before;
            break;
          }
          before += c;
        }
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    want = found[1];
    mask |= (digits - 1u) << shift;
    __syncthreads();
  }

  // Every wave counts, then writes, its contiguous share in order.
  const uint32_t steps = (e.tokens + 63u) / 64u, per = (steps + kPickWaves - 1u) / kPickWaves;
  const uint32_t s0 = wave * per < steps ? wave * per : steps, s1 = s0 + per < steps ? s0 + per : steps;
  uint32_t gt = 0, eq = 0;
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t t = s * 64u + lane;
    const uint32_t key = t < e.tokens ? keys[t] : 0u;
    gt += uint32_t(__popcll(__ballot(t < e.tokens && key > prefix)));
    eq += uint32_t(__popcll(__ballot(t < e.tokens && key == prefix)));
  }
  if (lane == 0u) {
    wave_gt[wave] = gt;
    wave_eq[wave] = eq;
  }
  __syncthreads();
  uint32_t eq_before = 0, at = 0;
  for (uint32_t w = 0; w < wave; ++w) {
    const uint32_t room = want > eq_before ? want - eq_before : 0u;
    at += wave_gt[w] + (wave_eq[w] < room ? wave_eq[w] : room);
    eq_before += wave_eq[w];
  }
  const uint64_t below = (uint64_t(1) << lane) - 1u;
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t t = s * 64u + lane;
    const uint32_t key = t < e.tokens ? keys[t] : 0u;
    const bool is_eq = t < e.tokens && key == prefix;
    const uint64_t eqs = __ballot(is_eq);
    const bool stays = (t < e.tokens && key > prefix) || (is_eq && eq_before + uint32_t(__popcll(eqs & below)) < want);
    const uint64_t all = __ballot(stays);
    if (stays) kept[at + uint32_t(__popcll(all & below))] = t;
    at += uint32_t(__popcll(all));
    eq_before += uint32_t(__popcll(eqs));
  }
}

// Rows of a destination token: where it comes from and goes to, ~0 if nowhere.
constexpr uint32_t kMoveTokens = 64;

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
  const auto row = [&](uint32_t page, uint32_t slot) { return (uint64_t(page) * a.kv_heads + kv) * a.page_tokens + slot; };
  // Pieces of `bytes` of both K and V rows of `row_bytes`.
  const auto copy = [&](const void* p, uint32_t row_bytes, auto piece) {
    using P = decltype(piece);
    const uint32_t per = row_bytes / uint32_t(sizeof(P));
    uint8_t* base = static_cast<uint8_t*>(const_cast<void*>(p));
    for (uint32_t i = tid; i < count * per; i += 256u) {
      const uint32_t t = i / per, x = i % per;
      if (to_page[t] == 0xffffffffu) continue;
      const P v = *reinterpret_cast<const P*>(base + row(from_page[t], from_slot[t]) * row_bytes + x * sizeof(P));
      *reinterpret_cast<P*>(base + row(to_page[t], to_slot[t]) * row_bytes + x * sizeof(P)) = v;
    }
  };
  if constexpr (BITS == 4) {
    copy(a.k, D / 2u, u32x4_e{});
    copy(a.v, D / 2u, u32x4_e{});
    if constexpr (G == 2) {
      copy(a.k_scales, 8u, uint64_t{});
      copy(a.v_scales, 8u, uint64_t{});
    } else {
      copy(a.k_scales, 4u * G, u32x4_e{});
      copy(a.v_scales, 4u * G, u32x4_e{});
    }
  } else {
    copy(a.k, D, u32x4_e{});
    copy(a.k_scales, 4u, uint32_t{});
    copy(a.v_scales, 4u, uint32_t{});
    // Four tokens of a dim to a dword: j0 and page_tokens are multiples of 8,
    // so the four slots are one aligned dword of one page.  The last, partial
    // four go byte by byte: the slots behind are not this call's.
    uint8_t* v = static_cast<uint8_t*>(a.v);
    const auto place = [&](uint32_t page, uint32_t slot, uint32_t d) {
      return ((uint64_t(page) * a.kv_heads + kv) * D + d) * a.page_tokens + slot;
    };
    const uint32_t quads = (count + 3u) / 4u;
    for (uint32_t i = tid; i < 16u * D; i += 256u) {
      const uint32_t qd = i % 16u, d = i / 16u;
      if (qd >= quads || to_page[4u * qd] == 0xffffffffu) continue;
      uint8_t x[4];
      bool whole = 4u * qd + 4u <= count;
#pragma unroll
      for (uint32_t k = 0; k < 4u; ++k) {
        const uint32_t t = 4u * qd + k;
        const bool in = t < count && to_page[t] != 0xffffffffu;
        whole = whole && in;
        x[k] = in ? v[place(from_page[t], from_slot[t], d)] : uint8_t(0);
      }
      uint8_t* dst = v + place(to_page[4u * qd], to_slot[4u * qd], d);
      if (whole) {
        *reinterpret_cast<uint32_t*>(dst) = uint32_t(x[0]) | uint32_t(x[1]) << 8 | uint32_t(x[2]) << 16 | uint32_t(x[3]) << 24;
      } else {
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k)
          if (4u * qd + k < count && to_page[4u * qd + k] != 0xffffffffu) dst[k] = x[k];
      }
    }
  }
  if (a.weights) copy(a.weights, 4u, uint32_t{});
}

}  // namespace

hipError_t launch_evict_select(const EvictArgs& a, hipStream_t stream) {
  evict_keys_kernel<<<dim3(a.max_tokens / 256u + (a.max_tokens % 256u != 0u ? 1u : 0u), a.batch), 256, 0, stream>>>(a);
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

}  // namespace kvb
