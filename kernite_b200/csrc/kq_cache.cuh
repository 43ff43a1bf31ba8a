// kq_cache.cuh -- the paged cache's format (include/kq.h, kq_cache) as the kernels see it: record
// geometry, the unit permutation, the scale bytes, and activations in and out of f32.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "kq.h"

namespace kq {

// Geometry of a cache, passed to kernels by value.
struct CacheView {
  uint8_t* k;
  uint8_t* v;
  uint64_t record;     // bytes of one head's part of a page
  uint32_t kind;       // KQ_CACHE_*
  uint32_t n_kv, dim, pitch;
  uint32_t page_log2;  // log2(page_size)
  uint32_t n_pages;
  uint32_t row;        // bytes of one position's codes
  uint32_t scales;     // scale bytes of one position (0: f16)

  __host__ __device__ uint32_t page() const { return 1u << page_log2; }
  // Byte offset of head h's record in page p of k or v.
  __host__ __device__ uint64_t at(uint32_t p, uint32_t h) const { return (uint64_t(p) * n_kv + h) * record; }
};

// What the 16-byte unit index of position p is XORed with, in rows of `row` bytes.
__host__ __device__ __forceinline__ uint32_t cache_swizzle(uint32_t p, uint32_t row) {
  return row >= 128 ? (p & 7u) : row == 64 ? ((p >> 1) & 3u) << 1 : ((p >> 2) & 1u) << 2;
}

// The same for many positions of one row size: (p >> a & m) << b.
struct Swizzle {
  uint32_t a, m, b;  // b: of bytes
  __device__ explicit Swizzle(uint32_t row)
      : a(row >= 128 ? 0 : row == 64 ? 1 : 2), m(row >= 128 ? 7 : row == 64 ? 3 : 1), b(4 + a) {}
  __device__ uint32_t bytes(uint32_t p) const { return (p >> a & m) << b; }
};

// Offset in a record's codes of byte `byte` of position p's row.
__host__ __device__ __forceinline__ uint32_t cache_offset(uint32_t p, uint32_t byte, uint32_t row) {
  return (p * row + byte) ^ (cache_swizzle(p, row) << 4);
}

// The largest code and the largest scale byte. A kernel turns a code u (stored with its offset) into
// its value by one fused multiply-add, (1024 + u) * scale - (1024 + offset) * scale, exact as long as
// the subtrahend is an f16: 1152 * 56 and 72 * 896 are the largest such.
__host__ __device__ constexpr float cache_top(uint32_t kind) { return kind == KQ_CACHE_Q8 ? 127.f : 7.f; }
__host__ __device__ constexpr uint32_t cache_last_scale(uint32_t kind) {
  return kind == KQ_CACHE_Q8 ? 0xA6u : 0xC6u;  // 56 and 896
}
constexpr uint32_t kScaleNan = 0xFFu;

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(byte << 7)));
}

// The scale byte of a block whose largest magnitude has the bits `most` (f32): the smallest value of
// 4 significant bits not below most / top (the correctly rounded quotient). Magnitudes compare as their
// bits do, NaN above infinity.
__device__ __forceinline__ uint32_t scale_byte(uint32_t most, uint32_t kind) {
  if (most >= 0x7f800000u) return kScaleNan;
  const float top = cache_top(kind);
  // the product with 1 / top is off by two units at most: only near a value of 4 bits, where that would
  // choose another one, and below f16's normal range is the quotient itself needed
  float want = __uint_as_float(most) * (kind == KQ_CACHE_Q8 ? 1.f / 127.f : 1.f / 7.f);
  if (want < 0x1p-13f || ((__float_as_uint(want) + 3u) & 0xFFFFFu) <= 6u) want = __fdiv_rn(__uint_as_float(most), top);
  // normal f16 range: round the fraction up to 3 bits and rebias the exponent (127 - 15); below
  // it the values are multiples of 2^-17
  const uint32_t b = want >= 0x1p-14f ? ((__float_as_uint(want) + 0xFFFFFu) >> 20) - (112u << 3)
                                      : static_cast<uint32_t>(ceilf(want * 0x1p17f));
  return min(b, cache_last_scale(kind));
}

// ---------------------------------------------------------------- activations

template <typename T>
__device__ __forceinline__ float act_to_f32(T x);
template <>
__device__ __forceinline__ float act_to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float act_to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float act_to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T act_from_f32(float x);
template <>
__device__ __forceinline__ float act_from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half act_from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 act_from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements at p, one wide access (p aligned to it) when N * sizeof(T) is 8 or 16, else
// one by one.
template <typename T, int N>
__device__ __forceinline__ void load_act(const T* p, float (&v)[N]) {
  if constexpr (N * sizeof(T) == 16) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = act_to_f32<T>(e[i]);
  } else if constexpr (N * sizeof(T) == 8) {
    const uint2 raw = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = act_to_f32<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = act_to_f32<T>(p[i]);
  }
}

// W words at p (16-byte aligned; W 4 or 8), and words as the values they hold.
template <int W>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
    w[i] = v.x;
    w[i + 1] = v.y;
    w[i + 2] = v.z;
    w[i + 3] = v.w;
  }
}
template <typename T, int N, int W>
__device__ __forceinline__ void words_to_f32(const uint32_t (&w)[W], float (&v)[N]) {
  static_assert(N * sizeof(T) == W * 4);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __half>) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    } else {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// A word of v[0] (and, 16-bit types, v[1]).
template <typename T>
__device__ __forceinline__ uint32_t act_word(const float* v);
template <>
__device__ __forceinline__ uint32_t act_word<float>(const float* v) { return __float_as_uint(v[0]); }
template <>
__device__ __forceinline__ uint32_t act_word<__half>(const float* v) {
  const __half2 h = __floats2half2_rn(v[0], v[1]);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t act_word<__nv_bfloat16>(const float* v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int N>
__device__ __forceinline__ void store_act(T* p, const float (&v)[N]) {
  constexpr int W = 4 / sizeof(T);  // elements a word
  if constexpr (N * sizeof(T) == 16) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(act_word<T>(v), act_word<T>(v + W), act_word<T>(v + 2 * W), act_word<T>(v + 3 * W));
  } else if constexpr (N * sizeof(T) == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(act_word<T>(v), act_word<T>(v + W));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = act_from_f32<T>(v[i]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_wide(T* p, const float (&v)[N]) {
  if constexpr (N * sizeof(T) <= 16) {
    store_act<T, N>(p, v);
  } else {
    float lo[N / 2], hi[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      lo[i] = v[i];
      hi[i] = v[N / 2 + i];
    }
    store_act<T, N / 2>(p, lo);
    store_act<T, N / 2>(p + N / 2, hi);
  }
}

}  // namespace kq
