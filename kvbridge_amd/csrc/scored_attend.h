// Ragged decode attention over a 4- or 8-bit cache under score forms
// (kvb_decode_attention_scored): the split kernel.
//
// A work-group takes one split of (sequence, kv head, block of 16 head-rows), its
// waves the split's 32-token tiles in turn.  It has all the waves that a CU
// holds of this kernel (12 or 8: few partials, which it can merge itself) where
// the sequences are few, and 4 where they are many and finer parts balance
// better (16 ragged sequences 78 us against 85; split_items in
// scored_shape.cpp).  One pass over the tokens with a running reference per
// head-row (not the maximum itself: it moves only when a score exceeds it by
// 5.5, so that most tiles rescale nothing), l in fp32, and the output's
// numerators in MFMA accumulators whose column is the head-row, so a rescale is
// lane-local.
//
// PV: the weight of token t for the dims of block g is p_t * step_{t,g}; times
// 2^ve it enters the product as one fp16 (PD 1: bf16 output, whose step is
// eight times coarser) or as two (PD 2).  ve is set per head-row where its
// weights are largest, and again when the reference moves or when a step times
// the largest 2^ve beside it passes 2^7, which keeps fp16 from overflowing for
// any steps.  The blocks' values at code 8 add sum_t p_t mid_{t,g} in fp32.
//
// What bounds it: long contexts the cache's bytes (16 ragged sequences of up to
// 32K tokens, 32 heads over 8 of dim 128: 76.7 us, 4.4 TB/s; four of 128K, 64
// heads: 167 us, 4.0 TB/s; int8, 32 windows of 4,096, dim 256: 110 us, 4.6 TB/s), short ones the chain of dependent loads from the item to its pages, K
// and the merge (512 tokens: 9.7 us), many head-rows of dim 256 the arithmetic of
// a tile, 4 us of a wave with two on a SIMD (48 head-rows, 8K tokens: 33 us).
#pragma once
#include "scored.h"

namespace kvb {

// Partials of item w: (max score, l) pairs of its head-rows, then the
// numerators: scratch[(w * row_heads + rh) * 2], scratch[2 * items * row_heads +
// (w * row_heads + rh) * dim], rh = row * q_heads + head.  They are stored and
// read by agent-scope atomics of 8 bytes, which every XCD sees without a
// write-back of its L2.
struct PartialPlace {
  float* ml;
  float* o;
};
__device__ __forceinline__ PartialPlace partial_place(const ScoredArgs& a, uint32_t item, uint32_t rh) {
  const uint64_t row_heads = uint64_t(a.rows) * a.q_heads, at = item * row_heads + rh;
  return PartialPlace{a.scratch + at * 2u, a.scratch + a.items * row_heads * 2u + at * a.dim};
}
struct Pair {
  float x, y;
};
__device__ __forceinline__ void store_pair(float* p, float x, float y) {
  const uint64_t v = uint64_t(__float_as_uint(x)) | uint64_t(__float_as_uint(y)) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Pair load_pair(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return Pair{__uint_as_float(uint32_t(v)), __uint_as_float(uint32_t(v >> 32))};
}

__device__ __forceinline__ void store_out4(const ScoredArgs& a, uint64_t at, f32x4 o) {
  if (a.out_type == 1u) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = o;
  } else if (a.out_type == 2u) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<f16x4*>(static_cast<_Float16*>(a.out) + at) =
        f16x4{_Float16(o[0]), _Float16(o[1]), _Float16(o[2]), _Float16(o[3])};
  } else {
    typedef __bf16 bf16x4_s __attribute__((ext_vector_type(4)));
    *reinterpret_cast<bf16x4_s*>(static_cast<__bf16*>(a.out) + at) =
        bf16x4_s{__bf16(o[0]), __bf16(o[1]), __bf16(o[2]), __bf16(o[3])};
  }
}

// Running state of a wave: acc[f] columns are head-rows (times F), rows dims.
// The reference `ref` is a whole number of factors of 2, and so is ve, so that
// both go into one exponent: w' = exp2(fma(score, log2 e, ve - ref)) rounds
// once, and l, mid and the products all carry 2^(ve - ref).
template <class C>
struct AttendState {
  f32x4 acc[2 * C::kGroups];
  float mid[C::kBits == 4 ? C::kH : 1];
  float mtop, l;         // maximum of the lane's scores, sum
  float ref, down, vf;   // reference, ve - reference, 2^ve (F = 1: the largest of the row's)
  int ve;
};
constexpr float kNoRef = -0x1p100f;  // below any score's exponent
__device__ __forceinline__ float weight(float score, float down) {
  return __builtin_amdgcn_exp2f(fmaf(score, kLog2e, down));
}
// The factor from 2^(ve - ref) to exp(-top), the rounding of top * log2 e taken
// back: 2^(ref - ve) / e^top as a fraction's exponential and a whole power.
struct ToTop {
  float fraction;
  int power;
};
__device__ __forceinline__ ToTop to_top(float ref, int ve, float top) {
  const float t2 = top * kLog2e, up = __builtin_ceilf(t2);
  return ToTop{__builtin_amdgcn_exp2f((up - t2) - fmaf(top, kLog2e, -t2)), int(fmaxf(ref - up, -1000.f)) - ve};
}

__device__ __forceinline__ float row_max_f16(float x) {
  x = fmaxf(x, row_ror<8>(x));
  x = fmaxf(x, row_ror<4>(x));
  x = fmaxf(x, row_ror<2>(x));
  return fmaxf(x, row_ror<1>(x));
}

// Moves the reference to the head-row's maximum and sets ve by the tile's
// largest weight of the column.  mult(j): the largest step of the lane's token j.
template <class C, typename F>
__device__ __forceinline__ void rescale(AttendState<C>& s, const float (&x)[8], F mult) {
  const float ref = fmaxf(s.ref, __builtin_ceilf(rows_max(s.mtop) * kLog2e));
  const float jump = ref - s.ref;
  float w = 0.f;
  unrolled<0, 8>([&](auto jc) {
    constexpr int j = jc;
    const float p = weight(x[j], -ref), big = mult(jc);
    w = fmaxf(w, p > 0.f ? p * big : 0.f);
  });
  w = rows_max(w);
  int ve = s.ve;
  const int moved = int(fminf(jump, 2000.f));
  if (w > 0.f && w <= FLT_MAX) {
    // Upwards only as far as the reference moved: the numerators must not grow.
    const int room = s.ve + (moved < 200 ? moved : 200);
    ve = -__builtin_amdgcn_frexp_expf(w);
    ve = ve < room ? ve : room;
    ve = ve < -64 ? -64 : (ve > 64 ? 64 : ve);  // l and mid carry 2^ve
  }
  const int dv = ve - s.ve - moved;  // 0 or less, or a score is not finite
#pragma unroll
  for (int f = 0; f < 2 * C::kGroups; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) s.acc[f][i] = ldexpf(s.acc[f][i], dv);
  s.l = ldexpf(s.l, dv);
  if constexpr (C::kBits == 4) {
#pragma unroll
    for (int h = 0; h < C::kH; ++h) s.mid[h] = ldexpf(s.mid[h], dv);
  }
  s.ref = ref;
  s.ve = ve;
  // One column per head-row: a lane holds parameters that all 16 of its row use.
  s.vf = ldexpf(1.f, ve);
  if constexpr (C::kF == 1) s.vf = row_max_f16(s.vf);
  s.down = float(ve) - ref;
}

template <int PD>
struct PDigits {
  f16x8 d[PD];
};
// w less an fp16 (the low or high half of a dword) in one instruction; the
// compiler converts first and subtracts then.
template <int HALF>
__device__ __forceinline__ float less_half(float w, uint32_t halves) {
  float r;
  if constexpr (HALF == 0) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(halves), "v"(w));
  else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(halves), "v"(w));
  return r;
}
template <int PD>
__device__ __forceinline__ PDigits<PD> p_digits(const float (&w)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  uint32_t d[PD][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = w[2 * j], b = w[2 * j + 1];
    d[0][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
    if constexpr (PD == 2)
      d[1][j] = __builtin_bit_cast(
          uint32_t, __builtin_convertvector((f32x2{less_half<0>(a, d[0][j]), less_half<1>(b, d[0][j])}), f16x2));
  }
  PDigits<PD> p;
#pragma unroll
  for (int i = 0; i < PD; ++i) p.d[i] = as_f16x8(d[i][0], d[i][1], d[i][2], d[i][3]);
  return p;
}

// Whether a tile asks for another reference or scale: p < 2^8 and step * 2^ve
// <= 2^7 keep every weight below 2^16.  And the rescale itself.
template <int G, int F>
__device__ __forceinline__ void keep_range(const typename Cache4<G, F>::V& v, const float (&x)[8], AttendState<Cache4<G, F>>& s) {
  using C = Cache4<G, F>;
  // The largest step as the largest word (of an integer: the low half may only
  // add 2^-7; a NaN asks for the rescale too).
  int most = int(v.p.w[0]);
#pragma unroll
  for (int i = 1; i < C::kPWords; ++i) most = int(v.p.w[i]) > most ? int(v.p.w[i]) : most;
  if (!__any(fmaf(s.mtop, kLog2e, -s.ref) > 8.f || !(__int_as_float(most) * s.vf <= 128.f))) return;
  typename C::Params p;
#pragma unroll
  for (int i = 0; i < C::kPWords; ++i) p.step[i] = __uint_as_float(v.p.w[i] & 0xffff0000u);
  rescale(s, x, [&](auto jc) {
    constexpr int j = jc;
    float t = 0.f;
    unrolled<0, C::kH>([&](auto hc) {
      constexpr int h = hc;
      t = fmaxf(t, p.template step_of<j, h>());
    });
    return t;
  });
}
template <int G>
__device__ __forceinline__ void keep_range(const typename Cache8<G>::V& v, const float (&x)[8], AttendState<Cache8<G>>& s) {
  if (!__any(fmaf(s.mtop, kLog2e, -s.ref) > 8.f || !(v.p * s.vf <= 128.f))) return;
  rescale(s, x, [&](auto jc) {
    constexpr int j = jc;
    return bc<j>(v.p);
  });
}

// A tile in which some head-row does not see every token: an infinite or NaN
// parameter times the weight 0 would reach that head-row.  Such parameters
// become 0, and the head-rows that do see the token get a NaN in its block.
template <int G, int F>
__device__ __forceinline__ void hide_odd_params(typename Cache4<G, F>::V& v, const float (&x)[8],
                                                AttendState<Cache4<G, F>>& s, uint32_t kg) {
  using C = Cache4<G, F>;
  constexpr int PW = C::kPWords;
  bool odd[PW], any = false;
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    odd[i] = (v.p.w[i] & 0x7f800000u) == 0x7f800000u || (v.p.w[i] & 0x7f80u) == 0x7f80u;
    any = any || odd[i];
  }
  if (!__any(any)) return;
  const float nan = __builtin_nanf("");
  if constexpr (F == 1) {
    uint32_t seen = 0u;  // bit 2 j: the lane's token j has a weight
#pragma unroll
    for (int j = 0; j < 8; ++j) seen |= weight(x[j], s.down) != 0.f ? 1u << (2 * j) : 0u;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const uint32_t lanes = uint32_t(__ballot(odd[i]) >> (16u * kg));  // bit 2 j + h: token j, block h * PW + i
      s.mid[i] = (lanes & seen) != 0u ? nan : s.mid[i];
      s.mid[PW + i] = ((lanes >> 1) & seen) != 0u ? nan : s.mid[PW + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < PW; ++i)
      s.mid[i % C::kH] = odd[i] && weight(x[i / C::kH], s.down) != 0.f ? nan : s.mid[i % C::kH];
  }
#pragma unroll
  for (int i = 0; i < PW; ++i) v.p.w[i] = odd[i] ? 0u : v.p.w[i];
}
template <int G>
__device__ __forceinline__ void hide_odd_params(typename Cache8<G>::V&, const float (&)[8], AttendState<Cache8<G>>&, uint32_t) {}

// One tile's weights and their products with V.  code_bits: 1024 as two fp16,
// held in a register (an instruction takes one constant, the mask).
template <int PD, int G, int F>
__device__ __forceinline__ void tile_values(const typename Cache4<G, F>::V& v, const float (&x)[8],
                                            AttendState<Cache4<G, F>>& s, uint32_t code_bits) {
  using C = Cache4<G, F>;
  const typename C::Params par = C::template unpack<true>(v.p);
  float p[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) p[j] = weight(x[j], s.down);
  s.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
  unrolled<0, C::kH>([&](auto hc) {
    constexpr int h = hc;
    float w[8];
    if constexpr (F == 1) {
      constexpr int PW = C::kPWords;
      weigh_block<h / PW>(w, s.mid[h], par.step[h % PW], par.other[h % PW], p);
    } else {
      unrolled<0, 8>([&](auto jc) {
        constexpr int j = jc;
        const float step = par.template step_of<j, h>(), at8 = par.template other_of<j, h>();
        w[j] = step * p[j];
        s.mid[h] = fmaf(at8, p[j], s.mid[h]);
      });
    }
    const PDigits<PD> d = p_digits<PD>(w);
    unrolled<0, F>([&](auto fc) {
      constexpr int g = fc * C::kH + h;
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        constexpr uint32_t sel = 0x0c000c00u | uint32_t(g % 4) | uint32_t(4 + g % 4) << 16;
        u[i] = __builtin_amdgcn_perm(v.v[2 * i + 1].w[g / 4], v.v[2 * i].w[g / 4], sel);
      }
      // 1024 + c and 1024 + 16 c as fp16 bits, less 1032 and 1152
      const uint32_t m = code_bits;
      f16x8 even = as_f16x8((u[0] & 0x000f000fu) | m, (u[1] & 0x000f000fu) | m, (u[2] & 0x000f000fu) | m, (u[3] & 0x000f000fu) | m);
      f16x8 odd = as_f16x8((u[0] & 0x00f000f0u) | m, (u[1] & 0x00f000f0u) | m, (u[2] & 0x00f000f0u) | m, (u[3] & 0x00f000f0u) | m);
      even -= (_Float16)1032.f;
      odd -= (_Float16)1152.f;
#pragma unroll
      for (int i = 0; i < PD; ++i) {
        s.acc[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, d.d[i], s.acc[2 * g], 0, 0, 0);
        s.acc[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, d.d[i], s.acc[2 * g + 1], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);  // one block's operands at a time in registers
    });
  });
}
template <int PD, int G>
__device__ __forceinline__ void tile_values(const typename Cache8<G>::V& v, const float (&x)[8], AttendState<Cache8<G>>& s,
                                            uint32_t) {
  float p[8], w[8];
  unrolled<0, 8>([&](auto jc) {
    constexpr int j = jc;
    p[j] = weight(x[j], s.down);
    w[j] = bc<j>(v.p) * p[j];
    w[j] = p[j] == 0.f ? 0.f : w[j];
  });
  s.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
  const PDigits<PD> d = p_digits<PD>(w);
#pragma unroll
  for (int f = 0; f < 2 * G; ++f) {
    const f16x8 c = i8x8_to_f16(v.v[f].w[0], v.v[f].w[1]);
#pragma unroll
    for (int i = 0; i < PD; ++i) s.acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c, d.d[i], s.acc[f], 0, 0, 0);
  }
}

// Four consecutive dims of a lane's head-row in units of 2^(ve - ref): chunk c
// of its 2 H, and the first of its dims.
template <int G, int F>
__device__ __forceinline__ f32x4 chunk_value(const AttendState<Cache4<G, F>>& s, int c, const float (&mid)[G / F], uint32_t r) {
  constexpr int H = G / F;
  const int h = c / 2, half = c % 2;
  f32x4 a = s.acc[2 * h], o = s.acc[2 * h + 1];  // even and odd dims of the lane's block f * H + h
#pragma unroll
  for (int f = 1; f < F; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = r % F == uint32_t(f) ? s.acc[2 * (f * H + h)][i] : a[i];
      o[i] = r % F == uint32_t(f) ? s.acc[2 * (f * H + h) + 1][i] : o[i];
    }
  return f32x4{a[2 * half] + mid[h], fmaf(o[2 * half], 0.0625f, mid[h]), a[2 * half + 1] + mid[h],
               fmaf(o[2 * half + 1], 0.0625f, mid[h])};
}
template <int G>
__device__ __forceinline__ f32x4 chunk_value(const AttendState<Cache8<G>>& s, int c, const float (&)[1], uint32_t) {
  return s.acc[c];
}
template <class C>
__device__ __forceinline__ uint32_t chunk_dim(uint32_t c, uint32_t r, uint32_t kg) {
  return C::kBits == 4 ? 32u * (r % C::kF * C::kH + c / 2u) + 8u * kg + 4u * (c % 2u) : 16u * c + 4u * kg;
}

// The joint result of `own` splits of one block's `count` head-rows, by NT
// threads.  Each wave takes head-rows in turn for the maximum and l (lane =
// split), then the factors of 64 splits at a time lie in LDS, and a thread adds
// four dims of a head-row over every GR-th split, eight loads in flight.
// AGENT: the partials come from work-groups of the same launch.
constexpr uint32_t kMergeSplits = 64;
struct MergeLds {
  float factor[16][kMergeSplits];
  float top[16], sum[16];
  f32x4 part[1];  // NT
};
// Row * q_heads + head of head-row hr of a kv head.
__device__ __forceinline__ uint32_t row_head(const ScoredArgs& a, uint32_t kv, uint32_t hr) {
  return hr / a.group * a.q_heads + kv * a.group + hr % a.group;
}
template <int DIM, bool AGENT>
__device__ __forceinline__ void merge_splits(const ScoredArgs& a, uint32_t b, uint32_t item0, uint32_t kv, uint32_t hr0,
                                             uint32_t count, uint32_t own, MergeLds& lds, uint32_t NT) {
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  constexpr uint32_t Q = DIM / 4, kAtOnce = 8;
  const uint32_t items = count * Q;                     // (head-row, four dims)
  const uint32_t groups = items < NT ? NT / items : 1u;  // of splits
  const uint32_t ml_step = a.rows * a.q_heads * 2u;
  const uint64_t step = uint64_t(a.rows) * a.q_heads * DIM;
  for (uint32_t r = wave; r < count; r += NT / 64u) {
    const float* ml = partial_place(a, item0, row_head(a, kv, hr0 + r)).ml;
    float top = neg_inf(), sum = 0.f;
    for (uint32_t j = lane; j < own; j += 64u) top = fmaxf(top, load_pair(ml + uint64_t(ml_step) * j).x);
    top = wave_max(top);
    for (uint32_t j = lane; j < own; j += 64u) {
      const Pair p = load_pair(ml + uint64_t(ml_step) * j);
      const float f = p.y == 0.f ? 0.f : exp_e(p.x - top);
      sum += p.y == 0.f ? 0.f : p.y * f;
      lds.factor[r][j % kMergeSplits] = f;  // of the last 64 splits in the end
    }
    sum = wave_sum(sum);
    if (lane == 0u) {
      lds.top[r] = top;
      lds.sum[r] = sum;
    }
  }
  for (uint32_t base = 0; base < items; base += NT) {
    const uint32_t item = groups > 1u ? tid % items : base + tid, group = groups > 1u ? tid / items : 0u;
    const bool in = item < items && group < groups;
    const uint32_t r = in ? item / Q : 0u, local = row_head(a, kv, hr0 + r);
    const float* o = partial_place(a, item0, local).o + 4u * (item % Q);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t c0 = 0; c0 < own; c0 += kMergeSplits) {
      if (own > kMergeSplits) {  // the factors of these splits
        __syncthreads();
        for (uint32_t i = tid; i < count * kMergeSplits; i += NT) {
          const uint32_t rr = i / kMergeSplits, j = c0 + i % kMergeSplits;
          if (j < own) {
            const Pair p = load_pair(partial_place(a, item0 + j, row_head(a, kv, hr0 + rr)).ml);
            lds.factor[rr][i % kMergeSplits] = p.y == 0.f ? 0.f : exp_e(p.x - lds.top[rr]);
          }
        }
      }
      __syncthreads();
      const uint32_t n = own - c0 < kMergeSplits ? own - c0 : kMergeSplits;
      for (uint32_t j0 = group; in && j0 < n; j0 += kAtOnce * groups) {
        f32x4 x[kAtOnce];
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) {
          const uint32_t j = j0 + i * groups;
          x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (j >= n) continue;
          const float* p = o + (c0 + j) * step;
          if constexpr (AGENT) {
            const Pair lo = load_pair(p), hi = load_pair(p + 2);
            x[i] = f32x4{lo.x, lo.y, hi.x, hi.y};
          } else {
            x[i] = *reinterpret_cast<const f32x4*>(p);
          }
        }
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) {
          const uint32_t j = j0 + i * groups;
          const float f = j < n ? lds.factor[r][j] : 0.f;
          if (f != 0.f) acc += x[i] * f;  // an empty split's are not written
        }
      }
    }
    if (groups > 1u) {
      lds.part[tid] = acc;
      __syncthreads();
      for (uint32_t g = 1; in && group == 0u && g < groups; ++g) acc += lds.part[g * items + item];
    }
    if (in && group == 0u) {
      const float sum = lds.sum[r];
      const uint64_t rh = uint64_t(b) * a.rows * a.q_heads + local;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] = sum == 0.f ? 0.f : acc[k] / sum;
      store_out4(a, rh * a.dim + 4u * (item % Q), acc);
      if (item % Q == 0u) {
        a.m[rh] = sum == 0.f ? neg_inf() : lds.top[r];
        a.l[rh] = sum;
      }
    }
  }
}

// LDS of a work-group of `waves`: Q's operands while the tiles run, then the
// waves' numerators, up to eight chunks at a time, then the merge.
template <class C>
constexpr int kChunksAtOnce = 2 * C::kH < 8 ? 2 * C::kH : 8;
template <class C, int QD>
constexpr uint32_t attend_lds(uint32_t waves) {
  const uint32_t q = sizeof(QBlock<C, QD>), o = waves * kChunksAtOnce<C> * 64u * 16u, m = sizeof(MergeLds) + waves * 64u * 16u;
  return q > o ? (q > m ? q : m) : (o > m ? o : m);
}

// What the first wave finds out for the work-group: its item and the columns'
// visible tokens.
struct AttendPlan {
  WorkItem it;
  uint32_t found, pre, min_lo, max_hi, all_lo, all_hi;
  uint32_t lo[16], hi[16];
  float slope[16];
  int back[16];
  int64_t qref;
};

// Waves per SIMD that the registers allow without spills.
template <class C, bool ONE>
constexpr int kAttendOccupancy = C::kGroups == 8 || (C::kF > 1 && C::kH > 1) || (C::kBits == 8 && !ONE) ? 2 : 3;

template <class C, int QD, int PD, bool ONE>
__global__ __launch_bounds__((256 * kAttendOccupancy<C, ONE>), (kAttendOccupancy<C, ONE>)) void scored_attend_kernel(const ScoredArgs a) {
  constexpr int F = C::kF, NC = 2 * C::kH, NR = kChunksAtOnce<C>, MW = 4 * kAttendOccupancy<C, ONE>;
  extern __shared__ __align__(16) uint8_t lds_raw[];
  QBlock<C, QD>& lds_q = *reinterpret_cast<QBlock<C, QD>*>(lds_raw);
  f32x4(*const lds_o)[NR][64] = reinterpret_cast<f32x4(*)[NR][64]>(lds_raw);  // [wave]
  __shared__ AttendPlan plan;
  __shared__ float lds_m[MW][16], lds_l[MW][16];
  const uint32_t NW = blockDim.x >> 6;
  const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, kg = lane >> 4;
  const uint32_t wave = uniform(threadIdx.x >> 6);
  const uint32_t kv = blockIdx.x % a.kv_heads, at = blockIdx.x / a.kv_heads;
  const uint32_t block = at % a.blocks, item = at / a.blocks;
  const uint32_t hr = block * 16u + r / F;  // F > 1: one block
  const bool valid = hr < a.head_rows;
  const uint32_t hrc = valid ? hr : a.head_rows - 1u;
  const uint32_t row = hrc / a.group, head = kv * a.group + hrc % a.group;

  // The first wave finds the item; everybody clears Q's operands meanwhile.
  if (wave == 0u) {
    WorkItem w{0u, 0u, 0u, 0u, ScoredSeq{0u, 0u, 0u}};
    const bool found = item_of(a, item, w);
    if (lane == 0u) {
      plan.it = w;
      plan.found = found ? 1u : 0u;
    }
  }
  clear_q(lds_q, threadIdx.x, 64u * NW);
  __syncthreads();
  if (uniform(plan.found) == 0u) return;
  WorkItem it;
  it.seq = uniform(plan.it.seq);
  it.split = uniform(plan.it.split);
  it.count = uniform(plan.it.count);
  it.first = uniform(plan.it.first);
  it.e = ScoredSeq{uniform(plan.it.e.start), uniform(plan.it.e.tokens), uniform(plan.it.e.table_off)};
  const uint32_t b = it.seq, split = it.split;
  const uint32_t local = row * a.q_heads + head;
  const uint64_t rh = uint64_t(b) * a.rows * a.q_heads + local;
  const ScoredSeq e = it.e;

  // Everything the first K request depends on is asked for before any of it is
  // waited for: by the first wave the positions around the rows' limits, by the
  // next four Q, and by all the pages of the tiles that would be theirs if
  // positions count up from 0 to the last row's.
  const auto share = [&](const LiveTiles& t) {  // tiles of a split
    uint32_t per = t.n / it.count + (t.n % it.count != 0u ? 1u : 0u);
    per = per > a.split_tiles ? per : a.split_tiles;
    return t.n <= a.alone_tiles ? a.alone_tiles : per;
  };
  // The wave's i-th tile, from its last one backwards: with a bias by distance
  // the largest scores come first, and the reference moves once instead of with
  // every tile.
  const auto tile_at = [&](const LiveTiles& t, uint32_t per, uint32_t i) {
    const uint32_t first = split * per + wave, end = t.n - split * per > per ? split * per + per : t.n;
    const uint32_t n = first < end ? (end - first - 1u) / NW : 0u, x = first + (i < n ? n - i : 0u) * NW;
    return t.tile(x < t.n ? x : t.n - 1u);
  };
  const int64_t prefix = a.prefix ? a.prefix[b] : 0;
  const uint64_t behind = uint64_t(a.rows) - 1u + a.window;
  const LiveTiles likely = live_tiles(prefix <= 0 ? 0u : (uint64_t(prefix) < e.tokens ? uint32_t(prefix) : e.tokens),
                                      a.window != 0u && behind < e.tokens ? e.tokens - uint32_t(behind) : 0u, e.tokens);
  TilePages pages{0u, 0u};
  if (e.tokens > 0u) {
    const uint32_t guess = share(likely);
    if (split * guess < likely.n) pages = tile_pages(a, e, [&](uint32_t i) { return tile_at(likely, guess, i); }, 0u, lane);
  }
  if (wave == 0u) {
    const int64_t qref = a.q_positions[uint64_t(b) * a.rows], qpos = a.q_positions[uint64_t(b) * a.rows + row];
    const Visible v = visible_tokens(a, e, valid, ask_visible(a, e, qpos, prefix));
    if (kg == 0u) {
      plan.lo[r] = v.lo;
      plan.hi[r] = v.hi;
      plan.slope[r] = a.slopes ? a.slopes[head] : 0.f;
      plan.back[r] = near(int64_t(uint64_t(qpos) - uint64_t(qref)));
    }
    if (lane == 0u) {
      plan.pre = v.pre;
      plan.min_lo = v.min_lo;
      plan.max_hi = v.max_hi;
      plan.all_lo = v.all_lo;
      plan.all_hi = v.all_hi;
      plan.qref = qref;
    }
  }
  const uint32_t stager = NW > 4u ? wave - 1u : wave;  // four waves for Q, not the first where there are more
  if (stager < 4u) {
    const uint32_t tid = stager * 64u + lane, q_hr = block * 16u + tid / 16u;
    stage_q<C, QD>(a, (uint64_t(b) * a.rows + q_hr / a.group) * a.q_stride + uint64_t(kv * a.group + q_hr % a.group) * a.dim,
                   q_hr < a.head_rows, lds_q, tid);
  }
  __syncthreads();
  const Visible vis{plan.lo[r], plan.hi[r], uniform(plan.pre), uniform(plan.min_lo), uniform(plan.max_hi), uniform(plan.all_lo),
                    uniform(plan.all_hi)};
  const int64_t qref = plan.qref;
  const LiveTiles live = live_tiles(vis.pre, vis.min_lo, vis.max_hi);
  const uint32_t per = share(live);
  const uint32_t own = live.n > 0u ? (live.n - 1u) / per + 1u : 1u;
  const bool writer = wave == 0u && valid && kg == 0u && r % F == 0u;  // of m and l
  if (split >= own) {
    if (a.counters == nullptr && writer) store_pair(partial_place(a, item, local).ml, neg_inf(), 0.f);
    return;
  }
  const ScoreForm form = score_form(a, lds_q.factor[r], plan.slope[r], plan.back[r]);

  AttendState<C> s;
#pragma unroll
  for (int f = 0; f < 2 * C::kGroups; ++f) s.acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int h = 0; h < (C::kBits == 4 ? C::kH : 1); ++h) s.mid[h] = 0.f;
  s.mtop = neg_inf();
  s.l = 0.f;
  s.ref = kNoRef;
  s.down = -kNoRef;
  s.vf = 1.f;
  s.ve = 0;

  const uint32_t first = split * per + wave;
  const uint32_t end = live.n - split * per > per ? split * per + per : live.n;
  const uint32_t n = first < end ? (end - first + NW - 1u) / NW : 0u;
  const auto tile_of = [&](uint32_t i) { return tile_at(live, per, i); };
  uint32_t code_bits = 0x64006400u;
  asm("" : "+v"(code_bits));
  if (n > 0u) {
    if (!live.same(likely) || split * per >= likely.n) pages = tile_pages(a, e, tile_of, 0u, lane);
    TilePages ahead_pages = pages;
    TileRows<ONE> rows = tile_rows<ONE>(a, pages, 0u, kv);
    uint32_t t0 = tile_of(0u) * kTileTokens;
    typename C::K k = C::template load_k<ONE>(a, rows, r, kg, e.tokens - t0);
    int ahead = load_ahead<C>(a, e, t0, r, kg, qref);
    for (uint32_t i = 0; i < n; ++i) {
      if (i % 16u == 0u) ahead_pages = tile_pages(a, e, tile_of, i + 16u, lane);  // a window ahead
      typename C::V v = C::template load_v<ONE>(a, rows, r, kg, e.tokens - t0);
      const uint32_t t_next = tile_of(i + 1u < n ? i + 1u : i) * kTileTokens;
      if ((i + 1u) % 16u == 0u) pages = ahead_pages;
      const TileRows<ONE> rows_next = tile_rows<ONE>(a, pages, i + 1u < n ? i + 1u : i, kv);
      const typename C::K k_next = C::template load_k<ONE>(a, rows_next, r, kg, e.tokens - t_next);
      const int ahead_next = load_ahead<C>(a, e, t_next, r, kg, qref);
      asm volatile("" ::: "memory");  // Q's operands stay in LDS: not hoisted out of the loop
      float x[8];
      tile_scores<C, QD>(k, lds_q, lane, x);
      const bool whole = t0 + kTileTokens <= vis.pre || (t0 >= vis.all_lo && t0 + kTileTokens <= vis.all_hi);
      apply_form<8>(a, form, !whole, vis.lo, vis.hi, vis.pre, [&](int j) { return t0 + C::token(kg, j); },
                    [&](int(&d)[8]) { unrolled<0, 8>([&](auto j) { d[j] = bci<j>(ahead); }); }, x);
      s.mtop = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])), s.mtop));
      keep_range(v, x, s);
      if (!whole) hide_odd_params(v, x, s, kg);
      tile_values<PD>(v, x, s, code_bits);
      k = k_next;
      rows = rows_next;
      t0 = t_next;
      ahead = ahead_next;
    }
  }

  // The waves' parts: a common maximum, then each chunk of dims is added by one wave.
  const float l = rows_sum(s.l), mtop = rows_max(s.mtop);
  if (kg == 0u) lds_m[wave][r] = mtop;
  float mid[C::kBits == 4 ? C::kH : 1];
#pragma unroll
  for (int h = 0; h < (C::kBits == 4 ? C::kH : 1); ++h) mid[h] = rows_sum(s.mid[h]);
  __syncthreads();  // also: every wave is done with Q
  float top = lds_m[0][r];
  for (uint32_t w = 1; w < NW; ++w) top = fmaxf(top, lds_m[w][r]);
  const ToTop f = to_top(s.ref, s.ve, top);
  // l = 0: a wave without visible tokens
  if (kg == 0u) lds_l[wave][r] = l == 0.f ? 0.f : ldexpf(l * f.fraction, f.power);
  const bool done = own == 1u;
  const PartialPlace part = done ? PartialPlace{nullptr, nullptr} : partial_place(a, item, local);
#pragma unroll
  for (int round = 0; round < NC / NR; ++round) {
#pragma unroll
    for (int c = 0; c < NR; ++c) {
      f32x4 o = chunk_value(s, round * NR + c, mid, r);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = l == 0.f ? 0.f : ldexpf(o[i] * f.fraction, f.power);
      lds_o[wave][c][lane] = o;
    }
    __syncthreads();
    // A chunk to a wave (its lanes are the tiles' lanes again).
    for (uint32_t c = wave; c < uint32_t(NR); c += NW) {
      f32x4 o = lds_o[0][c][lane];
      float sum = lds_l[0][r];
#pragma unroll 4
      for (uint32_t w = 1; w < NW; ++w) {
        o += lds_o[w][c][lane];
        sum += lds_l[w][r];
      }
      if (!valid) continue;
      const uint32_t d = chunk_dim<C>(round * NR + c, r, kg);
      if (done) {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = sum == 0.f ? 0.f : o[k] / sum;
        store_out4(a, rh * a.dim + d, o);
      } else {
        store_pair(part.o + d, o[0], o[1]);
        store_pair(part.o + d + 2, o[2], o[3]);
      }
    }
    if (round + 1 < NC / NR) __syncthreads();
  }
  float sum = lds_l[0][r];
  for (uint32_t w = 1; w < NW; ++w) sum += lds_l[w][r];
  if (writer) {
    if (done) {
      a.m[rh] = sum == 0.f ? neg_inf() : top;
      a.l[rh] = sum;
      if (a.counters == nullptr) store_pair(partial_place(a, item, local).ml, top, -1.f);  // the merge passes it by
    } else {
      store_pair(part.ml, top, sum);
    }
  }
  if (a.counters == nullptr || done) return;
  // Every wave's partials have reached memory before the work-group's ticket is
  // taken, so whoever draws the last ticket sees them all.
  __shared__ uint32_t last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  uint32_t* counter = a.counters + (uint64_t(b) * a.kv_heads + kv) * a.blocks + block;
  if (threadIdx.x == 0u) last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == own;
  __syncthreads();
  if (last == 0u) return;
  const uint32_t left = a.head_rows - block * 16u;
  merge_splits<32 * C::kGroups, true>(a, b, it.first, kv, block * 16u, left < 16u ? left : 16u, own,
                                      *reinterpret_cast<MergeLds*>(lds_raw), 64u * NW);
  if (threadIdx.x == 0u) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The same as a second launch: a work-group per head-row.
template <int DIM>
__global__ __launch_bounds__(256) void scored_merge_kernel(const ScoredArgs a) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  const uint32_t hr = blockIdx.x % a.head_rows, item = blockIdx.x / a.head_rows, kv = item % a.kv_heads, b = item / a.kv_heads;
  const WorkItem it = items_of(a, b);
  if (partial_place(a, it.first, row_head(a, kv, hr)).ml[1] == -1.f) return;  // one split: written
  merge_splits<DIM, false>(a, b, it.first, kv, hr, 1u, it.count, *reinterpret_cast<MergeLds*>(lds_raw), 256u);
}

template <class C, int QD, int PD>
inline hipError_t launch_attend_kernel(const ScoredArgs& a, hipStream_t stream) {
  const uint32_t groups = a.items * a.blocks * a.kv_heads;
  const bool one = a.page_tokens % kTileTokens == 0u;
  const uint32_t most = 4u * uint32_t(one ? kAttendOccupancy<C, true> : kAttendOccupancy<C, false>);
  const uint32_t waves = a.waves < most ? a.waves : most, bytes = attend_lds<C, QD>(waves);
  // LDS past 64 KiB, 2 KiB of it static, has to be asked for.
  if (bytes > 65536u - 2048u) {
    const hipError_t e = hipFuncSetAttribute(one ? reinterpret_cast<const void*>(scored_attend_kernel<C, QD, PD, true>)
                                                 : reinterpret_cast<const void*>(scored_attend_kernel<C, QD, PD, false>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    if (e != hipSuccess) return e;
  }
  if (one) scored_attend_kernel<C, QD, PD, true><<<groups, 64u * waves, bytes, stream>>>(a);
  else scored_attend_kernel<C, QD, PD, false><<<groups, 64u * waves, bytes, stream>>>(a);
  return hipGetLastError();
}
// Weights of one digit only where the output is bf16 and q has 16 bits.
template <class C>
inline hipError_t launch_attend_cache(const ScoredArgs& a, hipStream_t stream) {
  constexpr int QD = kQDigits<C, false>;
  if (a.q_type == 1u) return launch_attend_kernel<C, 2, 2>(a, stream);
  if (a.out_type == 3u) return launch_attend_kernel<C, QD, 1>(a, stream);
  return launch_attend_kernel<C, QD, 2>(a, stream);
}
// A column per block where the head-rows leave room for that; at dim 256 else
// two blocks per column (16 heads over 4, 4 x 32K: 47 us against 53 with one
// column per head-row).  At dim 128 that takes 216 VGPRs, two waves per SIMD, and
// one column per head-row is faster (64 heads over 8, 4 x 128K: 187 -> 165 us).
template <int G>
inline hipError_t launch_attend_cache4(const ScoredArgs& a, hipStream_t stream) {
  if (a.head_rows <= 16u / G) return launch_attend_cache<Cache4<G, G>>(a, stream);
  if constexpr (G == 8) {
    if (a.head_rows <= 32u / G) return launch_attend_cache<Cache4<G, G / 2>>(a, stream);
  }
  return launch_attend_cache<Cache4<G, 1>>(a, stream);
}

// Loads a unit's code object by one of its kernels.
template <typename K>
inline hipError_t preload_kernel(K* kernel) {
  hipFuncAttributes attr;
  return hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(kernel));
}
hipError_t preload_attend4_d64();
hipError_t preload_attend4_d128();
hipError_t preload_attend4_d256();
hipError_t preload_attend8_d64();
hipError_t preload_attend8_d128();
hipError_t preload_attend8_d256();
hipError_t launch_attend4_d64(const ScoredArgs& a, hipStream_t stream);
hipError_t launch_attend4_d128(const ScoredArgs& a, hipStream_t stream);
hipError_t launch_attend4_d256(const ScoredArgs& a, hipStream_t stream);
hipError_t launch_attend8_d64(const ScoredArgs& a, hipStream_t stream);
hipError_t launch_attend8_d128(const ScoredArgs& a, hipStream_t stream);
hipError_t launch_attend8_d256(const ScoredArgs& a, hipStream_t stream);

}  // namespace kvb
