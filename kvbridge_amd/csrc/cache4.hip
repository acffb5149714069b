// Writer of the 4-bit cache and reader of either format (kvb_append_kv_i4,
// kvb_read_kv; formats in include/kvbridge_c.h).
//
// A row of DIM = 32 G dims is handled by four lanes: lane kg takes dims 8 kg ..
// 8 kg + 7 of every block, which are the 4 G consecutive bytes 4 kg G .. of the
// packed row, so sources, packed rows and values all move in pieces of 4 to 32
// bytes, and a block's least and largest value are two DPP steps over the four
// lanes.  Arithmetic is IEEE fp32 step by step, so the stored bits are those of
// any correctly rounded evaluation of the same formula.
// Measured at 16,384 tokens of 8 kv heads, dim 128: writing fp16 rows 26-31 us
// (88 MB, 2.8-3.4 TB/s; the 672 vector instructions of a wave take 20 of them;
// with a division per element 37), reading them back as fp32 26 us (155 MB, 5.9
// TB/s); 64 tokens 4.4 and 2.9 us, launch and one chain of loads.
#include <cfloat>

#include "device_common.h"
#include "scored_args.h"

namespace kvb {
namespace {

typedef uint32_t u32x2_c __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_c __attribute__((ext_vector_type(4)));

// Lane i ^ M of each group of four (DPP quad_perm).
template <int M>
__device__ __forceinline__ float quad_xor(float x) {
  constexpr int kPerm = (0 ^ M) | (1 ^ M) << 2 | (2 ^ M) << 4 | (3 ^ M) << 6;
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kPerm, 0xF, 0xF, false));
}

// bf16 bits of a finite x, round to nearest even (may overflow to infinity).
__device__ __forceinline__ uint32_t bf16_bits(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ float from_bf16(uint32_t b) { return __uint_as_float(b << 16); }

// Eight codes clamp(rint(y / step), 0, 15), y = x - least, the quotient correctly
// rounded, four bits each.  Mostly without the division: with the hardware
// reciprocal (1 ulp) y * per is within 1.5 * 2^-23 of that quotient relatively,
// 2^-18 absolutely up to code 15 and a half, so where it lies more than 2^-14
// from a half the nearest integer is the same.  The rest (exact halves, one in
// 700 of 16-bit sources, and any product that is not finite) divides.  Adding 1.5 *
// 2^23 rounds to an integer in the low bits of the sum (quotients stay below
// 2^20), so the codes are put together as the sums' bits, the constants' sum
// taken off.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float least, float step) {
  constexpr float kRound = 12582912.f;  // bits 0x4b400000
  const float per = __builtin_amdgcn_rcpf(step);
  uint32_t codes = 0u, constants = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = x[i] - least;
    float r = fmaf(y, per, kRound);
    if (!(fabsf(fmaf(y, per, -(r - kRound))) <= 0.5f - 0x1p-14f)) r = __builtin_rintf(y / step) + kRound;
    codes += __float_as_uint(__builtin_amdgcn_fmed3f(r, kRound, kRound + 15.f)) << (4 * i);
    constants += 0x4b400000u << (4 * i);
  }
  return codes - constants;
}

// The lane's 4 G bytes: byte i * G + g is byte i of block g's codes.
template <int G>
__device__ __forceinline__ void interleave(const uint32_t (&codes)[G], uint32_t (&packed)[G]) {
  if constexpr (G == 2) {
    packed[0] = __builtin_amdgcn_perm(codes[1], codes[0], 0x05010400u);
    packed[1] = __builtin_amdgcn_perm(codes[1], codes[0], 0x07030602u);
  } else {
#pragma unroll
    for (int h = 0; h < G / 4; ++h) {
      const uint32_t* c = codes + 4 * h;
      const uint32_t lo01 = __builtin_amdgcn_perm(c[1], c[0], 0x05010400u), hi01 = __builtin_amdgcn_perm(c[1], c[0], 0x07030602u);
      const uint32_t lo23 = __builtin_amdgcn_perm(c[3], c[2], 0x05010400u), hi23 = __builtin_amdgcn_perm(c[3], c[2], 0x07030602u);
      packed[h] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
      packed[G / 4 + h] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
      packed[2 * (G / 4) + h] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
      packed[3 * (G / 4) + h] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
    }
  }
}

// Eight elements from p: 16-byte loads where the host has checked that every
// row's pieces are aligned to them.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (VEC && sizeof(T) == 4) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else if constexpr (VEC) {
    const u32x4_c v = *reinterpret_cast<const u32x4_c*>(p);
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = float(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = float(p[i]);
  }
}

template <class T, int G, bool VEC>
__global__ __launch_bounds__(256) void append4_kernel(const Append4Args a) {
  const uint32_t kg = threadIdx.x & 3u;
  const uint64_t item = uint64_t(blockIdx.x) * 64u + threadIdx.x / 4u;  // (token, kv head, K or V)
  const uint64_t pairs = uint64_t(a.tokens) * a.kv_heads;
  const bool is_v = blockIdx.y != 0u;
  if (item >= pairs) return;
  const uint32_t token = uint32_t(item / a.kv_heads), kv = uint32_t(item - uint64_t(token) * a.kv_heads);
  const uint32_t slot_id = a.slots[token];
  const uint32_t page = slot_id / a.page_tokens, slot = slot_id - page * a.page_tokens;
  if (page >= a.pages) return;
  const T* src = static_cast<const T*>(is_v ? a.v_new : a.k_new) + uint64_t(token) * (is_v ? a.v_stride : a.k_stride) +
                 uint64_t(kv) * (32u * G) + kg * 8u;
  float x[G][8];
#pragma unroll
  for (int g = 0; g < G; ++g) load8<T, VEC>(src + 32 * g, x[g]);
  uint32_t codes[G], packed[G], word[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float lo = x[g][0], hi = x[g][0], odd = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo = fminf(lo, x[g][i]);
      hi = fmaxf(hi, x[g][i]);
      odd = fmaf(x[g][i], 0.f, odd);  // NaN once an element is not finite
    }
    if (odd != 0.f) hi = lo = __builtin_huge_valf();  // carried by hi to the other lanes
    lo = fminf(lo, quad_xor<1>(lo));
    hi = fmaxf(hi, quad_xor<1>(hi));
    lo = fminf(lo, quad_xor<2>(lo));
    hi = fmaxf(hi, quad_xor<2>(hi));
    uint32_t least_b = bf16_bits(lo);
    const float least = from_bf16(least_b);
    uint32_t step_b = bf16_bits(fmaxf(hi - least, 0.f) / 15.f);
    const float step = from_bf16(step_b);
    const bool fine = hi <= FLT_MAX && fabsf(least) <= FLT_MAX && step <= FLT_MAX;
    codes[g] = 0u;
    if (fine && step > 0.f) codes[g] = codes_of(x[g], least, step);
    if (!fine) least_b = step_b = 0x7fc0u;
    word[g] = step_b << 16 | least_b;
  }
  interleave<G>(codes, packed);
  const uint64_t row = (uint64_t(page) * a.kv_heads + kv) * a.page_tokens + slot;
  uint8_t* dst = (is_v ? a.v : a.k) + row * (16u * G) + kg * (4u * G);
  if constexpr (G == 2) {
    *reinterpret_cast<u32x2_c*>(dst) = u32x2_c{packed[0], packed[1]};
  } else {
#pragma unroll
    for (int i = 0; i < G / 4; ++i)
      reinterpret_cast<u32x4_c*>(dst)[i] = u32x4_c{packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]};
  }
  uint32_t* words = (is_v ? a.v_scales : a.k_scales) + row * G;
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (uint32_t(g) % 4u == kg) words[g] = word[g];
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = T(x[i]);
    *reinterpret_cast<t8*>(p) = v;
  }
}

template <class T, int G>
__global__ __launch_bounds__(256) void read4_kernel(const ReadArgs a) {
  const uint32_t kg = threadIdx.x & 3u;
  const uint64_t item = uint64_t(blockIdx.x) * 64u + threadIdx.x / 4u;
  if (item >= uint64_t(a.tokens) * a.kv_heads) return;
  const bool is_v = blockIdx.y != 0u;
  const uint32_t token = uint32_t(item / a.kv_heads), kv = uint32_t(item - uint64_t(token) * a.kv_heads);
  const uint32_t slot_id = a.slots[token];
  const uint32_t page = slot_id / a.page_tokens, slot = slot_id - page * a.page_tokens;
  T* dst = static_cast<T*>(is_v ? a.v_out : a.k_out) + item * (32u * G) + kg * 8u;
  uint32_t packed[G], word[G];
  if (page < a.pages) {
    const uint64_t row = (uint64_t(page) * a.kv_heads + kv) * a.page_tokens + slot;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(is_v ? a.v : a.k) + row * (16u * G) + kg * (4u * G));
    const uint32_t* words = static_cast<const uint32_t*>(is_v ? a.v_scales : a.k_scales) + row * G;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      packed[i] = src[i];
      word[i] = words[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < G; ++i) packed[i] = word[i] = 0u;
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float step = __uint_as_float(word[g] & 0xffff0000u), least = __uint_as_float(word[g] << 16);
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = i * G + g;
      const uint32_t byte = packed[at / 4] >> (8 * (at % 4));
      // code * step is exact in fp32 (4 by 8 bits), so the sum is the only rounding
      x[2 * i] = fmaf(float(byte & 15u), step, least);
      x[2 * i + 1] = fmaf(float((byte >> 4) & 15u), step, least);
    }
    store8(dst + 32 * g, x);
  }
}

// int8: a work-group takes 64 tokens of one kv head, lane = token for V (its
// bytes of a dim lie beside the neighbours'), lanes along the dims for K.
template <class T, int G>
__global__ __launch_bounds__(256) void read8_kernel(const ReadArgs a) {
  constexpr uint32_t D = 32u * G, W = D + 8u;  // LDS row: 16-byte pieces, rows two banks apart
  __shared__ __align__(16) uint8_t tile[64 * W];
  __shared__ uint32_t pages[64], slots[64];
  const uint32_t kv = blockIdx.y, t0 = blockIdx.x * 64u;
  const bool is_v = blockIdx.z != 0u;
  const uint32_t n = a.tokens - t0 < 64u ? a.tokens - t0 : 64u;
  if (threadIdx.x < 64u) {
    const uint32_t id = threadIdx.x < n ? a.slots[t0 + threadIdx.x] : 0xffffffffu;
    const uint32_t page = id / a.page_tokens;
    pages[threadIdx.x] = threadIdx.x < n ? page : 0xffffffffu;
    slots[threadIdx.x] = id - page * a.page_tokens;
  }
  __syncthreads();
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  if (is_v) {
    const bool in = pages[lane] < a.pages;
    const uint8_t* src = static_cast<const uint8_t*>(a.v) + (uint64_t(in ? pages[lane] : 0u) * a.kv_heads + kv) * D * a.page_tokens + (in ? slots[lane] : 0u);
    for (uint32_t d = wave; d < D; d += 4u)
      if (in) tile[lane * W + d] = src[uint64_t(d) * a.page_tokens];
    __syncthreads();
  }
  for (uint32_t i = threadIdx.x; i < n * (D / 8u); i += 256u) {
    const uint32_t t = i / (D / 8u), d = i % (D / 8u) * 8u;
    float x[8];
    if (pages[t] < a.pages) {
      const uint64_t row = (uint64_t(pages[t]) * a.kv_heads + kv) * a.page_tokens + slots[t];
      const float scale = static_cast<const float*>(is_v ? a.v_scales : a.k_scales)[row];
      const u32x2_c c = is_v ? *reinterpret_cast<const u32x2_c*>(tile + t * W + d)
                             : *reinterpret_cast<const u32x2_c*>(static_cast<const uint8_t*>(a.k) + row * D + d);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = float(int8_t(c[j / 4] >> (8 * (j % 4)))) * scale;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
    }
    store8(static_cast<T*>(is_v ? a.v_out : a.k_out) + (uint64_t(t0 + t) * a.kv_heads + kv) * D + d, x);
  }
}

template <class T, int G>
hipError_t append_dim(const Append4Args& a, bool vec, dim3 grid, hipStream_t stream) {
  if (vec) append4_kernel<T, G, true><<<grid, 256, 0, stream>>>(a);
  else append4_kernel<T, G, false><<<grid, 256, 0, stream>>>(a);
  return hipGetLastError();
}
template <class T>
hipError_t append_type(const Append4Args& a, hipStream_t stream) {
  const uint64_t el = sizeof(T);
  const auto al16 = [](uint64_t x) { return x % 16u == 0u; };
  const bool vec = al16(reinterpret_cast<uintptr_t>(a.k_new)) && al16(reinterpret_cast<uintptr_t>(a.v_new)) &&
                   al16(a.k_stride * el) && al16(a.v_stride * el);
  const dim3 grid(uint32_t((uint64_t(a.tokens) * a.kv_heads + 63u) / 64u), 2u);
  if (a.dim == 64u) return append_dim<T, 2>(a, vec, grid, stream);
  if (a.dim == 128u) return append_dim<T, 4>(a, vec, grid, stream);
  return append_dim<T, 8>(a, vec, grid, stream);
}

template <class T, int G>
hipError_t read_dim(const ReadArgs& a, hipStream_t stream) {
  if (a.kv_bits == 4u)
    read4_kernel<T, G><<<dim3(uint32_t((uint64_t(a.tokens) * a.kv_heads + 63u) / 64u), 2u), 256, 0, stream>>>(a);
  else
    read8_kernel<T, G><<<dim3(a.tokens / 64u + (a.tokens % 64u != 0u ? 1u : 0u), a.kv_heads, 2u), 256, 0, stream>>>(a);
  return hipGetLastError();
}
template <class T>
hipError_t read_type(const ReadArgs& a, hipStream_t stream) {
  if (a.dim == 64u) return read_dim<T, 2>(a, stream);
  if (a.dim == 128u) return read_dim<T, 4>(a, stream);
  return read_dim<T, 8>(a, stream);
}

}  // namespace

hipError_t launch_append4(const Append4Args& a, hipStream_t stream) {
  if (a.src_type == 1u) return append_type<float>(a, stream);
  if (a.src_type == 2u) return append_type<_Float16>(a, stream);
  return append_type<__bf16>(a, stream);
}

hipError_t launch_read(const ReadArgs& a, hipStream_t stream) {
  if (a.out_type == 1u) return read_type<float>(a, stream);
  if (a.out_type == 2u) return read_type<_Float16>(a, stream);
  return read_type<__bf16>(a, stream);
}

hipError_t preload_cache4() {
  hipFuncAttributes attr;
  return hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&append4_kernel<float, 2, true>));
}

}  // namespace kvb
