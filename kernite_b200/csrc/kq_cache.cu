// kq_cache.cu -- rotary positions, and the quantised paged cache: written (heads rotated on the way),
// read back, and its rows moved. The format is kq_cache.cuh's.
//
// All four move bytes once; for a few tokens one launch is what they take.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>
#include <type_traits>

#include "kq_cache.cuh"
#include "kq_device.cuh"
#include "kq_internal.h"
#include "kq_launch.h"

namespace kq {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kMaxMoves = 64;

// One kernel rotates heads into an array (queries, kq_rope_apply) and into the cache (keys), and
// copies heads into the cache (values). A CTA takes one token and a share of its rows (heads); a warp
// takes the rows of `together` heads at once, VE consecutive elements a lane.
struct RopeArgs {
  float gain;
  uint32_t layout;
  const void* q;   // rows [0, nq): to q_out
  const void* k;   // rows [nq, nq + n_kv): rotated, to the cache
  const void* v;   // rows [nq + n_kv, nq + 2 n_kv): to the cache
  void* q_out;
  const int* positions;
  const long long* slots;
  uint64_t q_token, q_head, k_token, v_token, out_token, out_head;
  uint32_t nq, dim;
  uint32_t rot_half;  // rotated pairs a head (0: none)
  uint32_t together;  // heads a warp takes at once
  uint32_t tokens, per_block;  // tokens; of those, a CTA's (rope_rows_kernel)
  CacheView cache;
  unsigned* err;
};

// The pairs' turns per position, times 2^64. Kernels take the smaller table where it will do: 1 KB of
// parameters costs the host 2 us a launch more than 100 bytes do.
template <uint32_t PAIRS>
struct Turns {
  uint64_t at[PAIRS];
};

// (x_a, x_b) of a pair whose (gain cos, gain sin) is w.
__device__ __forceinline__ float turned_a(float a, float b, float2 w) { return fmaf(a, w.x, -b * w.y); }
__device__ __forceinline__ float turned_b(float a, float b, float2 w) { return fmaf(a, w.y, b * w.x); }

// VE neighbouring elements e.. of a row, pairs (2i, 2i + 1), rotated; elements past the rotated part
// (rot_half pairs) as they are. VE == 1 reads the pair's other element too.
template <typename T, int VE>
__device__ __forceinline__ void rotate_pairs(const T* row, uint32_t e, uint32_t rot_half, const float2* cs,
                                             float (&y)[VE]) {
  load_act<T, VE>(row + e, y);
  if constexpr (VE == 1) {
    if (e < 2 * rot_half) {
      const float other = act_to_f32<T>(row[e ^ 1u]);
      y[0] = (e & 1u) ? turned_b(other, y[0], cs[e >> 1]) : turned_a(y[0], other, cs[e >> 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VE; i += 2) {
      if (e + i < 2 * rot_half) {
        const float2 w = cs[(e + i) >> 1];
        const float x0 = y[i], x1 = y[i + 1];
        y[i] = turned_a(x0, x1, w);
        y[i + 1] = turned_b(x0, x1, w);
      }
    }
  }
}

// The same for pairs (i, i + rot_half); the partners come from memory too (the same row, so from L1).
// rot_half is a multiple of VE.
template <typename T, int VE>
__device__ __forceinline__ void rotate_halves(const T* row, uint32_t e, uint32_t rot_half, const float2* cs,
                                              float (&y)[VE]) {
  load_act<T, VE>(row + e, y);
  if (e >= 2 * rot_half) return;
  const bool first = e < rot_half;
  float o[VE];
  load_act<T, VE>(row + (first ? e + rot_half : e - rot_half), o);
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const float2 w = cs[(first ? e : e - rot_half) + i];
    y[i] = first ? turned_a(y[i], o[i], w) : turned_b(o[i], y[i], w);
  }
}

// 1 / x to a unit or two of the last place.
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// VE values of elements e.. of a head's row into the cache: their codes to `to`, their block's scale to
// `scale_to`; the 32 / VE lanes of a block of 32 elements call this together (mask: the lanes that do).
//
// A code is the correctly rounded quotient's nearest integer, so that which of two a value near a tie gets
// does not depend on how it was divided. The sum q + 1.5 2^23, q the product with the rounded reciprocal (off
// by 2^-15 at most), has that integer in its low bits; what it left of q says whether q was so near a tie
// that the quotient itself is needed. Rounding and conversion instructions would take the special
// function unit, four lanes a cycle.
template <int VE>
__device__ __forceinline__ void keep(uint32_t kind, uint8_t* to, uint8_t* scale_to, uint32_t e, const float (&x)[VE],
                                     uint32_t mask) {
  if (kind == KQ_CACHE_F16) {
    __half h[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) h[i] = __float2half_rn(x[i]);
    if constexpr (VE == 8) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(h);
    else if constexpr (VE == 4) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(h);
    else *reinterpret_cast<__half*>(to) = h[0];
    return;
  }
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < VE; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 16 / VE; o; o >>= 1) most = max(most, __shfl_xor_sync(mask, most, o));
  const uint32_t byte = scale_byte(most, kind);
  const float scale = scale_value(byte);
  float inverse = reciprocal(scale);
  float y[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) y[i] = x[i];
  if (byte == 0 || byte >= cache_last_scale(kind)) {
    // nothing to hold (zeros, or a block that reads back as NaN), or magnitudes that may saturate
    const float lim = byte == cache_last_scale(kind) ? cache_top(kind) * scale : 0.f;
    if (lim == 0.f) inverse = 0.f;
#pragma unroll
    for (int i = 0; i < VE; ++i) y[i] = lim == 0.f ? 0.f : fminf(fmaxf(y[i], -lim), lim);
  }
  const float magic = 12582912.f + (kind == KQ_CACHE_Q8 ? 128.f : 8.f);  // 1.5 2^23, and the code's offset
  float sum[VE], near = 0.f;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    sum[i] = fmaf(y[i], inverse, magic);
    near = fmaxf(near, fabsf(fmaf(y[i], inverse, magic - sum[i])));
  }
  if (near > 0.5f - 0x1p-12f) {
#pragma unroll
    for (int i = 0; i < VE; ++i) sum[i] = magic + rintf(__fdiv_rn(y[i], scale));
  }
  uint32_t u[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) u[i] = __float_as_uint(sum[i]);
  if (e % 32 == 0) *scale_to = static_cast<uint8_t>(byte);
  if (kind == KQ_CACHE_Q8) {
    const auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    };
    if constexpr (VE == 8)
      *reinterpret_cast<uint2*>(to) = make_uint2(four(u[0], u[1], u[2], u[3]), four(u[4], u[5], u[6], u[7]));
    else if constexpr (VE == 4) *reinterpret_cast<uint32_t*>(to) = four(u[0], u[1], u[2], u[3]);
    else *to = static_cast<uint8_t>(u[0]);
    return;
  }
  // eight elements a word, element 2i at nibble i and 2i + 1 at nibble i + 4
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const uint32_t j = (e + i) & 7u;
    word |= (u[i] & 15u) << (4 * ((j >> 1) + 4 * (j & 1)));
  }
#pragma unroll
  for (int o = 4 / VE; o; o >>= 1) word |= __shfl_xor_sync(mask, word, o);
  if (e % 8 == 0) *reinterpret_cast<uint32_t*>(to) = word;
}

// (gain cos, gain sin) of pair i at a position. Whole turns do not matter, so position * turns is taken
// modulo 1 as a 64-bit fraction, exactly but for the table's rounding (position 2^31: 2^-33 turns). Quarters of
// a turn are taken off it, and what is left, an eighth at most, goes to f32 and sincospi: it is then off by 2^-28
// turns, where a half turn in f32 would be by 2^-26, more than the roundings of the cosine and of the rotation
// (relative error of f32 heads 5.6e-8 in the mean square, so 3.9e-8).
__device__ __forceinline__ float2 angle(int position, uint64_t turns, float gain) {
  const uint64_t at = static_cast<uint64_t>(static_cast<int64_t>(position)) * turns;
  const uint32_t quarter = static_cast<uint32_t>((at + (1ull << 61)) >> 62);  // the nearest, modulo 4 with `at`
  const int64_t rest = static_cast<int64_t>(at - (static_cast<uint64_t>(quarter) << 62));
  float s, c;
  sincospif(static_cast<float>(static_cast<int>((rest + (1ll << 31)) >> 32)) * 0x1p-31f, &s, &c);
  const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
  return make_float2(gain * (quarter == 1 || quarter == 2 ? -x : x), gain * (quarter >= 2 ? -y : y));
}

// Token t's slot, -1 where it is not kept (or out of the cache, which is recorded).
__device__ __forceinline__ long long take_slot(const RopeArgs& a, uint32_t t) {
  if (!a.slots) return -1;
  const long long slot = a.slots[t];
  if (slot < 0) return -1;
  if (static_cast<uint64_t>(slot) >> a.cache.page_log2 < a.cache.n_pages) return slot;
  if (threadIdx.x % 32 == 0) report_error(a.err, kErrCacheRange);
  return -1;
}

constexpr int kLane = 8;  // elements a lane of rope_rows_kernel has of a row

// Heads of 64, 128 or 256 elements, every row on 16 bytes. A lane holds E consecutive elements of a row, dim /
// E lanes a row, so that its place in a head, and with it its angles, are the same for every row it takes: they
// stay in registers. A pair's other element is in the lane (pairs) or rot_half / E lanes away (halves). Bound
// by memory in principle (4001 tokens of 40 16-bit heads: 12.7 us of copying, 22 taken; 6144 tokens of 32 + 32
// + 32 f32 heads written to 8 bits: 70 us of copying, 96 taken) and by instructions and latencies in fact: the
// quantisation of a block, the exchange of halves. A CTA takes per_block tokens, as many warps each; with one,
// the grid's y shares out its rows.
template <typename T, uint32_t PAIRS>
__global__ void __launch_bounds__(kThreads, 4)
    rope_rows_kernel(const __grid_constant__ RopeArgs a, const __grid_constant__ Turns<PAIRS> turns_of) {
  constexpr int E = kLane, WORDS = E * sizeof(T) / 4;
  // Rows whose loads are in flight: 16 words, at four CTAs a SM (4001 tokens of 40 16-bit heads 21 us, 6144 of
  // 96 f32 rows written and read back 125). Half the words 22 and 133; three CTAs 24 and 134, five, which
  // spill, 28 and 145.
  constexpr uint32_t AHEAD = 16 / WORDS;
  extern __shared__ float2 angles[];  // [per_block][rot_half]
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t t0 = blockIdx.x * a.per_block;
  for (uint32_t i = threadIdx.x; i < a.per_block * a.rot_half; i += kThreads) {
    const uint32_t k = i / a.rot_half;
    if (t0 + k < a.tokens) angles[i] = angle(a.positions[t0 + k], turns_of.at[i - k * a.rot_half], a.gain);
  }
  __syncthreads();
  const uint32_t each = kWarps / a.per_block;  // warps a token
  const uint32_t warp = threadIdx.x / 32 % each, lane = threadIdx.x % 32;
  const uint32_t t = t0 + threadIdx.x / 32 / each;
  if (t >= a.tokens) return;
  const float2* cs = angles + (t - t0) * a.rot_half;
  const long long slot = take_slot(a, t);
  const uint32_t rows = a.nq + (slot >= 0 ? 2 * a.cache.n_kv : 0);
  const uint32_t page = static_cast<uint32_t>(slot >= 0 ? slot >> a.cache.page_log2 : 0);
  const uint32_t p = static_cast<uint32_t>(slot) & (a.cache.page() - 1);
  const uint32_t per_row = a.dim / E, e = lane % per_row * E, sub = lane / per_row;
  const uint32_t at_once = 32 / per_row;  // rows a warp takes at once
  const bool halves = a.layout == KQ_ROPE_HALVES;
  // y = x * by + other * with, where the lane's elements turn (all of them or none)
  const bool lane_turns = e < 2 * a.rot_half;
  float by[E], with[E];
  uint32_t partner = lane;
  if (lane_turns) {
    const bool first = e < a.rot_half;
    const float2* w = cs + (halves ? (first ? e : e - a.rot_half) : e / 2);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float2 v = w[halves ? i : i / 2];
      by[i] = v.x;
      with[i] = (halves ? first : (i & 1) == 0) ? -v.y : v.y;
    }
    if (halves) partner = first ? lane + a.rot_half / E : lane - a.rot_half / E;
  }
  // where a row r is: queries first, then the keys, then the values, addressed by r throughout
  const uint32_t keys_end = a.nq + a.cache.n_kv;
  const T* q = static_cast<const T*>(a.q) + t * a.q_token + e;
  const T* k_in = static_cast<const T*>(a.k) + t * a.k_token + e;
  const T* v_in = static_cast<const T*>(a.v) + t * a.v_token + e;
  T* q_out = static_cast<T*>(a.q_out) + t * a.out_token + e;
  const uint32_t byte_at = a.cache.kind == KQ_CACHE_F16  ? 2 * e
                           : a.cache.kind == KQ_CACHE_Q8 ? e
                                                         : e / 8 * 4;  // of its word
  const uint64_t page_at = a.cache.at(page, 0);
  const uint32_t code_at = cache_offset(p, byte_at, a.cache.row);
  const uint32_t scale_at = a.cache.page() * a.cache.row + p * a.cache.scales + e / 32;
  const uint32_t step = gridDim.y * each * at_once;
  for (uint32_t r0 = (blockIdx.y * each + warp) * at_once; r0 < rows; r0 += AHEAD * step) {
    uint32_t raw[AHEAD][WORDS];
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k) {
      const uint32_t row = r0 + k * step + sub;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) raw[k][i] = 0;
      if (row >= rows) continue;
      const T* from = row < a.nq       ? q + row * a.q_head
                      : row < keys_end ? k_in + uint64_t(row - a.nq) * a.dim
                                       : v_in + uint64_t(row - keys_end) * a.dim;
      load_words(from, raw[k]);
    }
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; ++k) {
      const uint32_t row0 = r0 + k * step, row = row0 + sub;
      if (row0 >= rows) break;  // the warp's first row: all its lanes leave
      const bool in = row < rows, turns = row < keys_end;
      float x[E], y[E];
      words_to_f32<T>(raw[k], x);
      if (row0 >= keys_end) {  // all values
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = x[i];
      } else {
        if (halves) {
          uint32_t other[WORDS];
#pragma unroll
          for (int i = 0; i < WORDS; ++i) other[i] = __shfl_sync(0xffffffffu, raw[k][i], partner);
          words_to_f32<T>(other, y);
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) y[i] = x[i ^ 1];
        }
        const bool turned = turns && lane_turns;
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = turned ? fmaf(x[i], by[i], y[i] * with[i]) : x[i];
      }
      const uint32_t mask = __ballot_sync(0xffffffffu, in && row >= a.nq);
      if (!in) continue;
      if (row < a.nq) {
        store_wide<T, E>(q_out + row * a.out_head, y);
      } else {
        uint8_t* record = (turns ? a.cache.k : a.cache.v) + page_at +
                          uint64_t(row - (turns ? a.nq : keys_end)) * a.cache.record;
        keep<E>(a.cache.kind, record + code_at, record + scale_at, e, y, mask);
      }
    }
  }
}

// Any other head, stride or alignment: a warp takes the rows of `together` heads at once, VE consecutive
// elements a lane. Grid (tokens, shares of the rows). One row's loads are in flight a warp, and lanes stay
// idle where a row is no multiple of a warp's elements: 4001 tokens of 5120 elements, heads of 80, 96, 160 or
// 192, take 38 to 64 us in bf16 (13 of copying) and 46 to 54 in f32 (25); 6144 tokens of 32 + 32 + 32 f32 heads
// of 96 written to 8 bits 161 us (55).
template <typename T, int VE, uint32_t PAIRS>
__global__ void __launch_bounds__(kThreads)
    rope_kernel(const __grid_constant__ RopeArgs a, const __grid_constant__ Turns<PAIRS> turns_of) {
  __shared__ float2 cs[PAIRS];
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t t = blockIdx.x;
  for (uint32_t i = threadIdx.x; i < a.rot_half; i += kThreads) cs[i] = angle(a.positions[t], turns_of.at[i], a.gain);
  const long long slot = take_slot(a, t);
  __syncthreads();
  const uint32_t rows = a.nq + (slot >= 0 ? 2 * a.cache.n_kv : 0);
  const uint32_t page = static_cast<uint32_t>(slot >= 0 ? slot >> a.cache.page_log2 : 0);
  const uint32_t p = static_cast<uint32_t>(slot) & (a.cache.page() - 1);
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t step = gridDim.y * kWarps * a.together;
  const bool halves = a.layout == KQ_ROPE_HALVES;
  for (uint32_t r0 = (blockIdx.y * kWarps + warp) * a.together; r0 < rows; r0 += step) {
    if (r0 < a.nq) {
      // queries: a lane takes VE elements, for halves with their partners, so that nothing it reads
      // is written by another pass of the row (q_out may be q)
      const uint32_t width = halves ? a.dim - a.rot_half : a.dim;
      for (uint32_t at = lane * VE; at < a.together * width + lane * VE; at += 32 * VE) {
        const uint32_t row = r0 + at / width;
        uint32_t e = at % width;
        const bool in = at < a.together * width;
        const T* x = static_cast<const T*>(a.q) + t * a.q_token + row * a.q_head;
        T* y = static_cast<T*>(a.q_out) + t * a.out_token + row * a.out_head;
        if (halves) {
          if (!in) continue;
          if (e < a.rot_half) {
            float u[VE], v[VE];
            load_act<T, VE>(x + e, u);
            load_act<T, VE>(x + e + a.rot_half, v);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
              const float2 w = cs[e + i];
              const float u0 = u[i];
              u[i] = turned_a(u0, v[i], w);
              v[i] = turned_b(u0, v[i], w);
            }
            store_act<T, VE>(y + e, u);
            store_act<T, VE>(y + e + a.rot_half, v);
          } else {
            float u[VE];
            e += a.rot_half;
            load_act<T, VE>(x + e, u);
            store_act<T, VE>(y + e, u);
          }
        } else {
          float u[VE];
          if (in) rotate_pairs<T, VE>(x, e, a.rot_half, cs, u);
          __syncwarp();  // both elements of a pair are read before either is written
          if (in) store_act<T, VE>(y + e, u);
        }
      }
      continue;
    }
    const uint32_t width = a.cache.pitch;
    for (uint32_t c0 = 0; c0 < a.together * width; c0 += 32 * VE) {
      const uint32_t at = c0 + lane * VE;
      const uint32_t row = r0 + at / width - a.nq, e = at % width;
      const bool in = at < a.together * width && row < 2 * a.cache.n_kv;
      const uint32_t mask = __ballot_sync(0xffffffffu, in);
      if (!in) continue;
      const bool key = row < a.cache.n_kv;
      const uint32_t h = key ? row : row - a.cache.n_kv;
      const T* x = key ? static_cast<const T*>(a.k) + t * a.k_token + h * a.dim
                       : static_cast<const T*>(a.v) + t * a.v_token + h * a.dim;
      float y[VE];
      if (e >= a.dim) {
#pragma unroll
        for (int i = 0; i < VE; ++i) y[i] = 0.f;
      } else if (!key) {
        load_act<T, VE>(x + e, y);
      } else if (halves) {
        rotate_halves<T, VE>(x, e, a.rot_half, cs, y);
      } else {
        rotate_pairs<T, VE>(x, e, a.rot_half, cs, y);
      }
      __syncwarp(mask);
      uint8_t* record = (key ? a.cache.k : a.cache.v) + a.cache.at(page, h);
      const uint32_t byte_at = a.cache.kind == KQ_CACHE_F16  ? 2 * e
                               : a.cache.kind == KQ_CACHE_Q8 ? e
                                                             : e / 8 * 4;  // of its word
      keep<VE>(a.cache.kind, record + cache_offset(p, byte_at, a.cache.row),
               record + a.cache.page() * a.cache.row + p * a.cache.scales + e / 32, e, y, mask);
    }
  }
}

template <uint32_t PAIRS>
int launch_rope(void (*kernel)(RopeArgs, Turns<PAIRS>), RopeArgs& a, const kq_rope* rope, uint32_t rows, int sm_count,
                cudaStream_t s, const char* call, bool by_rows) {
  Turns<PAIRS> turns;
  if (rope) std::memcpy(turns.at, rope->turns, sizeof(turns.at[0]) * a.rot_half);
  // Below some hundred tokens one CTA a token leaves most SMs idle: a token's rows are then shared by more
  // CTAs, each taking the angles again. With many tokens a CTA takes four, so that the angles' latency is
  // paid once for them (4001 tokens of 40 16-bit heads: 29 -> 21 us; 6144 of 96 rows 131 -> 125).
  const uint32_t groups = (rows + kWarps * a.together - 1) / (kWarps * a.together);
  a.per_block = by_rows && a.tokens >= 16u * sm_count ? 4 : 1;
  const uint32_t shares = std::max<uint32_t>(1, std::min<uint32_t>(groups, 4u * sm_count / a.tokens));
  const uint32_t shared = by_rows ? a.per_block * a.rot_half * sizeof(float2) : 0;
  const cudaError_t e = launch_pdl(kernel, dim3((a.tokens + a.per_block - 1) / a.per_block, shares), kThreads, shared,
                                   s, a, turns);
  return e == cudaSuccess ? KQ_OK : cuda_fail(e, "cudaLaunchKernelExC", call);
}

// The wide forms want every row they read or write on 16 bytes and, for halves, partners a whole lane
// apart (rope_rows_kernel also, for pairs, whole lanes that turn); anything else is served one element a
// lane.
template <typename T, uint32_t PAIRS>
int dispatch_rope(RopeArgs& a, const kq_rope* rope, bool aligned, uint32_t rows, int sm_count, cudaStream_t s,
                  const char* call) {
  constexpr int VE = 16 / sizeof(T);
  const bool pairs = a.layout == KQ_ROPE_PAIRS;
  const bool wide = aligned && a.dim % VE == 0;
  if (wide && (pairs ? 2 * a.rot_half : a.rot_half) % kLane == 0 && (a.dim == 64 || a.dim == 128 || a.dim == 256)) {
    a.together = 32 * kLane / a.dim;
    return launch_rope(rope_rows_kernel<T, PAIRS>, a, rope, rows, sm_count, s, call, true);
  }
  if (wide && (pairs || a.rot_half % VE == 0)) {
    // narrow heads: a warp takes several at once, where the queries come out even
    const uint32_t width = a.slots ? a.cache.pitch : a.dim;
    const uint32_t n = std::max<uint32_t>(1, 32 * VE / width);
    a.together = a.nq % n == 0 ? n : 1;
    return launch_rope(rope_kernel<T, VE, PAIRS>, a, rope, rows, sm_count, s, call, false);
  }
  a.together = 1;
  return launch_rope(rope_kernel<T, 1, PAIRS>, a, rope, rows, sm_count, s, call, false);
}

uint32_t type_size(uint32_t type) {
  return type == KQ_TYPE_F32 ? 4 : type == KQ_TYPE_F16 || type == KQ_TYPE_BF16 ? 2 : 0;
}

template <typename T>
int run_rope_of(RopeArgs& a, const kq_rope* rope, bool aligned, uint32_t rows, int sm_count, cudaStream_t s,
                const char* call) {
  return a.rot_half <= 64 ? dispatch_rope<T, 64>(a, rope, aligned, rows, sm_count, s, call)
                          : dispatch_rope<T, 128>(a, rope, aligned, rows, sm_count, s, call);
}

int run_rope(RopeArgs& a, const kq_rope* rope, uint32_t type, bool aligned, uint32_t tokens, uint32_t rows,
             int sm_count, cudaStream_t s, const char* call) {
  a.tokens = tokens;
  if (rope) {
    a.gain = rope->gain;
    a.layout = rope->layout;
    a.rot_half = rope->rot_dim / 2;
  }
  if (type == KQ_TYPE_F32) return run_rope_of<float>(a, rope, aligned, rows, sm_count, s, call);
  if (type == KQ_TYPE_F16) return run_rope_of<__half>(a, rope, aligned, rows, sm_count, s, call);
  return run_rope_of<__nv_bfloat16>(a, rope, aligned, rows, sm_count, s, call);
}

bool rope_ok(const kq_rope* r) {
  return r->rot_dim >= 2 && r->rot_dim <= 256 && r->rot_dim % 2 == 0 && r->layout <= KQ_ROPE_HALVES;
}

bool on16(uint64_t bytes) { return bytes % 16 == 0; }

// ---------------------------------------------------------------- reading back

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// E elements (16 bytes of output) a thread, of ROWS rows at once so that their loads are in flight together;
// a CTA has `subs` rows side by side where a row is less than its threads. Grid: (row groups, parts of a
// row, K then V). What differs by rows alone is worked out once a thread, and codes become f32 by their
// place in the low bits of 2^23 (conversions take the special function unit): the kernel was bound by its
// instructions (65536 rows of 1024, 8 bits to f16: 75 -> 71 us, 89 % of the copy rate).
template <typename T, int KIND, int ROWS>
__global__ void __launch_bounds__(kThreads)
    cache_read_kernel(CacheView c, T* k_out, T* v_out, const long long* slots, uint64_t token_stride, uint32_t count,
                      uint32_t units, uint32_t subs, uint32_t over_units, uint32_t per_head, uint32_t over_head,
                      bool wide, unsigned* err) {
  constexpr int E = 16 / sizeof(T);
  constexpr int B = KIND == KQ_CACHE_F16 ? 2 * E : KIND == KQ_CACHE_Q8 ? E : 4;  // bytes of codes (Q4: a word)
  pdl_wait();
  pdl_launch_dependents();
  const bool value = blockIdx.z;
  const uint32_t thread = blockIdx.y * kThreads + threadIdx.x;
  const uint32_t sub = subs > 1 ? __umulhi(thread, over_units) : 0, i = thread - sub * units;
  const uint32_t h = over_head ? __umulhi(i, over_head) : i, e = (i - h * per_head) * E;
  if (sub >= subs || h >= c.n_kv) return;
  const uint32_t r0 = blockIdx.x * (ROWS * subs) + sub;
  const uint8_t* base = (value ? c.v : c.k) + h * c.record;
  const uint64_t page_bytes = c.n_kv * c.record;
  const uint32_t byte = KIND == KQ_CACHE_F16 ? 2 * e : KIND == KQ_CACHE_Q8 ? e : e / 8 * 4;
  const uint32_t scales = c.page() * c.row + e / 32;
  const Swizzle swizzle(c.row);
  T* to = (value ? v_out : k_out) + r0 * token_stride + h * c.dim + e;
  const uint64_t step = subs * token_stride, slots_end = uint64_t(c.n_pages) << c.page_log2;
  long long slot[ROWS];
  // codes of a row that is not there: zeros, with the kind's offset
  constexpr uint32_t kNone = KIND == KQ_CACHE_F16 ? 0u : KIND == KQ_CACHE_Q8 ? 0x80808080u : 0x88888888u;
  uint32_t raw[ROWS][B / 4], scale[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) slot[k] = r0 + k * subs < count ? slots[r0 + k * subs] : -1;
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
#pragma unroll
    for (int w = 0; w < B / 4; ++w) raw[k][w] = kNone;
    scale[k] = 0;
    if (slot[k] < 0) continue;
    if (static_cast<uint64_t>(slot[k]) >= slots_end) {
      report_error(err, kErrCacheRange);
      slot[k] = -2;  // this row is left as it is
      continue;
    }
    const uint8_t* rec = base + static_cast<uint32_t>(slot[k] >> c.page_log2) * page_bytes;
    const uint32_t p = static_cast<uint32_t>(slot[k]) & (c.page() - 1);
    const uint8_t* from = rec + ((p * c.row + byte) ^ swizzle.bytes(p));
    if constexpr (B == 16) {
      const uint4 w = *reinterpret_cast<const uint4*>(from);
      raw[k][0] = w.x;
      raw[k][1] = w.y;
      raw[k][2] = w.z;
      raw[k][3] = w.w;
    } else if constexpr (B == 8) {
      const uint2 w = *reinterpret_cast<const uint2*>(from);
      raw[k][0] = w.x;
      raw[k][1] = w.y;
    } else {
      raw[k][0] = *reinterpret_cast<const uint32_t*>(from);
    }
    if constexpr (KIND != KQ_CACHE_F16) scale[k] = rec[scales + p * c.scales];
  }
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    if (r0 + k * subs >= count || slot[k] == -2) continue;
    T* at = to + k * step;
    const uint32_t s16 = slot[k] < 0 ? 0u : scale[k] << 7;  // the scale as f16
    if constexpr (KIND != KQ_CACHE_F16 && std::is_same_v<T, __half>) {
      // 1024 + code, less 1024 + offset, times the scale: each exact
      const __half2 by = as_half2(s16 | s16 << 16);
      uint32_t w[E / 2];
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const uint32_t x = KIND == KQ_CACHE_Q8 ? __byte_perm(raw[k][j / 2], 0x64646464u, j % 2 ? 0x4342 : 0x4140)
                                               : ((raw[k][0] >> (4 * j)) & 0x000f000fu) | 0x64006400u;
        const __half2 y = __hmul2(__hsub2(as_half2(x), __float2half2_rn(KIND == KQ_CACHE_Q8 ? 1152.f : 1032.f)), by);
        w[j] = *reinterpret_cast<const uint32_t*>(&y);
      }
      if (wide) {
        *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          at[j] = __ushort_as_half(static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2))));
      }
      continue;
    }
    float y[E];
    const float s = h2f(s16);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if constexpr (KIND == KQ_CACHE_F16) {
        y[j] = h2f(raw[k][j / 2] >> (16 * (j % 2)) & 0xffffu);
      } else if constexpr (KIND == KQ_CACHE_Q8) {
        y[j] = (__uint_as_float(__byte_perm(raw[k][j / 4], 0x4b000000u, 0x7650 + j % 4)) - 8388736.f) * s;
      } else {
        // elements 2 i at nibble i, 2 i + 1 at i + 4; the word's second four are 8 bits up
        const uint32_t x = E == 4 ? raw[k][0] >> (2 * (e & 4u)) : raw[k][0];
        y[j] = (__uint_as_float((x >> (4 * (j / 2 + 4 * (j % 2))) & 15u) | 0x4b000000u) - 8388616.f) * s;
      }
    }
    if (wide) {
      store_act<T, E>(at, y);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) at[j] = act_from_f32<T>(y[j]);
    }
  }
}

// ---------------------------------------------------------------- moving rows

// A CTA takes one head of one group, keys or values: every source row (codes and scales) into shared
// memory, then out, so a group's rows may slide over one another. The permutation of units depends
// on the position, so rows move as unpermuted 16-byte units. One launch is what a step's few rows take: 32
// groups of 5 rows of 8 heads of 128, 8 bits, 3.7 us; 64 groups of 64 10.3 us (17 MB read and written), two
// latencies and a barrier a CTA.
__global__ void __launch_bounds__(kThreads) cache_move_kernel(CacheView c, const long long* src,
                                                              const long long* dst, const int* starts,
                                                              uint32_t moves, unsigned* err) {
  extern __shared__ uint4 rows[];
  __shared__ uint8_t scales[kMaxMoves][8];
  uint8_t* base = blockIdx.z ? c.v : c.k;
  const uint32_t h = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  const int a = starts[blockIdx.x], b = starts[blockIdx.x + 1];
  if (a < 0 || b < a || static_cast<uint32_t>(b) > moves || b - a > static_cast<int>(kMaxMoves)) {
    if (threadIdx.x == 0) report_error(err, kErrCacheRange);
    return;
  }
  const uint32_t n = b - a, units = c.row / 16;
  const uint64_t capacity = uint64_t(c.n_pages) << c.page_log2;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads)
    if ((src[a + i] >= 0 && static_cast<uint64_t>(src[a + i]) >= capacity) ||
        (dst[a + i] >= 0 && static_cast<uint64_t>(dst[a + i]) >= capacity))
      report_error(err, kErrCacheRange);
  for (int write = 0; write < 2; ++write) {
    for (uint32_t i = threadIdx.x; i < n * (units + 1); i += kThreads) {
      const uint32_t m = i / (units + 1), u = i % (units + 1);
      const long long from = src[a + m], to = dst[a + m];
      if (from < 0 || to < 0 || static_cast<uint64_t>(from) >= capacity || static_cast<uint64_t>(to) >= capacity)
        continue;
      const long long slot = write ? to : from;
      const uint32_t p = static_cast<uint32_t>(slot) & (c.page() - 1);
      uint8_t* rec = base + c.at(static_cast<uint32_t>(slot >> c.page_log2), h);
      if (u < units) {
        uint4* at = reinterpret_cast<uint4*>(rec + cache_offset(p, 16 * u, c.row));
        if (write) *at = rows[m * units + u];
        else rows[m * units + u] = *at;
      } else {
        uint8_t* at = rec + c.page() * c.row + p * c.scales;
        for (uint32_t j = 0; j < c.scales; ++j) {
          if (write) at[j] = scales[m][j];
          else scales[m][j] = at[j];
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace

int cache_view(const kq_cache* c, CacheView* out) {
  if (c->type > KQ_CACHE_Q4 || c->n_kv == 0 || c->head_dim == 0 || c->head_dim % 32 || c->head_dim > 256 ||
      c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) || c->n_pages == 0 ||
      c->n_pages > 0x7fffffffu || c->n_kv > 0xffffu)
    return KQ_E_INVALID;
  CacheView v = {};
  v.k = reinterpret_cast<uint8_t*>(c->k);
  v.v = reinterpret_cast<uint8_t*>(c->v);
  v.kind = c->type;
  v.n_kv = c->n_kv;
  v.dim = c->head_dim;
  v.pitch = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  while ((1u << v.page_log2) < c->page_size) ++v.page_log2;
  v.n_pages = c->n_pages;
  v.row = c->type == KQ_CACHE_F16 ? 2 * v.pitch : c->type == KQ_CACHE_Q8 ? v.pitch : v.pitch / 2;
  v.scales = c->type == KQ_CACHE_F16 ? 0 : v.pitch / 32;
  v.record = uint64_t(c->page_size) * (v.row + v.scales);
  *out = v;
  return KQ_OK;
}

uint64_t cache_bytes(const kq_cache& c) {
  CacheView v;
  return cache_view(&c, &v) == KQ_OK ? v.at(v.n_pages, 0) : 0;
}

int check_cache(const kq_cache* c, const char* call, CacheView* out) {
  if (!c) return fail(KQ_E_INVALID, call, "null cache");
  if (cache_view(c, out) != KQ_OK)
    return fail(KQ_E_INVALID, call, "the cache wants a type F16, Q8 or Q4, n_kv 1..65535, head_dim a multiple "
                                    "of 32 up to 256, page_size 16, 32, 64, 128 or 256 and pages");
  if (!c->k || !c->v || !on16(c->k) || !on16(c->v))
    return fail(KQ_E_INVALID, call, "the cache's k and v must be 16-byte aligned and not null");
  return KQ_OK;
}

int cache_prepare(kq_ctx* ctx) {
  const cudaError_t e = cudaFuncSetAttribute(cache_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(kMaxMoves * 512));
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute", "cache move kernel");
  return KQ_OK;
}

int rope_init(const kq_rope_params* p, kq_rope* out) {
  const char* call = "kq_rope_init";
  if (!p || !out) return fail(KQ_E_INVALID, call, "null argument");
  if (p->rot_dim < 2 || p->rot_dim > 256 || p->rot_dim % 2 || p->layout > KQ_ROPE_HALVES)
    return fail(KQ_E_INVALID, call, "rot_dim must be even, 2..256, and the layout a KQ_ROPE_* one");
  if (!(p->base > 1.0) || !(p->freq_scale > 0.0) || !(p->ext_factor >= 0.0) || !(p->attn_factor > 0.0) ||
      !std::isfinite(p->base) || !std::isfinite(p->freq_scale) || !std::isfinite(p->ext_factor) ||
      !std::isfinite(p->attn_factor))
    return fail(KQ_E_INVALID, call, "base must be above 1, freq_scale and attn_factor above 0, ext_factor >= 0");
  if (p->ext_factor > 0.0 && (p->orig_ctx == 0 || !(p->beta_fast > 0.0) || !(p->beta_slow > 0.0) ||
                              !std::isfinite(p->beta_fast) || !std::isfinite(p->beta_slow)))
    return fail(KQ_E_INVALID, call, "ext_factor needs orig_ctx, beta_fast and beta_slow");
  // The turns in 64-bit significands (long double of x86-64, more elsewhere): a position multiplies their error.
  using Long = long double;
  constexpr Long kTwoPi = 6.283185307179586476925286766559L;
  const double rot = p->rot_dim;
  double low = 0, high = 0;
  if (p->ext_factor > 0.0) {
    // the pair that turns beta times in orig_ctx positions
    const auto pair = [&](double beta) {
      return rot * std::log(p->orig_ctx / (beta * static_cast<double>(kTwoPi))) / (2 * std::log(p->base));
    };
    low = std::max(0.0, std::floor(pair(p->beta_fast)));
    high = std::min(rot - 1, std::ceil(pair(p->beta_slow)));
  }
  kq_rope r = {};
  r.rot_dim = p->rot_dim;
  r.layout = p->layout;
  r.gain = static_cast<float>(p->attn_factor *
                              (p->ext_factor > 0.0 ? 1.0 + 0.1 * std::log(1.0 / p->freq_scale) : 1.0));
  for (uint32_t i = 0; i < p->rot_dim / 2; ++i) {
    Long f = std::pow(static_cast<Long>(p->base), static_cast<Long>(-2.0 * i) / p->rot_dim);
    if (p->freq_factors) {
      if (!(p->freq_factors[i] > 0.f) || !std::isfinite(p->freq_factors[i]))
        return fail(KQ_E_INVALID, call, "freq_factors must be above 0");
      f /= p->freq_factors[i];
    }
    Long slow = p->freq_scale;
    if (p->ext_factor > 0.0) {
      const Long ramp = std::min<Long>(1, std::max<Long>(0, (i - low) / std::max<Long>(0.001, high - low)));
      const Long mix = (1 - ramp) * p->ext_factor;
      slow = p->freq_scale * (1 - mix) + mix;
    }
    // modulo 1, to the nearest 2^-64 (2^64 itself is 0)
    const Long turns = f * slow / kTwoPi, part = turns - std::floor(turns);
    const Long scaled = std::floor(std::ldexp(part, 64) + 0.5L);
    r.turns[i] = scaled >= 0x1p64L ? 0 : static_cast<uint64_t>(scaled);
  }
  *out = r;
  return KQ_OK;
}

int rope_apply(kq_ctx* ctx, const kq_rope_desc& d, cudaStream_t s) {
  const char* call = "kq_rope_apply";
  const uint32_t size = type_size(d.type);
  if (!size) return fail(KQ_E_INVALID, call, "type must be F32, F16 or BF16");
  if (!d.rope || !rope_ok(d.rope)) return fail(KQ_E_INVALID, call, "rope must come from kq_rope_init");
  if (d.tokens == 0 || d.heads == 0) return KQ_OK;
  if (!d.x || !d.y || !d.positions) return fail(KQ_E_INVALID, call, "null pointer");
  if (d.head_dim == 0 || d.head_dim > 1024 || d.head_dim < d.rope->rot_dim)
    return fail(KQ_E_INVALID, call, "head_dim must be rot_dim..1024");
  if (d.tokens > 0x7fffffffu || d.heads > 0xffffffu)
    return fail(KQ_E_INVALID, call, "too many tokens or heads");
  if (d.x % size || d.y % size || d.positions % 4)
    return fail(KQ_E_INVALID, call, "x and y must be aligned to their elements, positions to 4 bytes");
  RopeArgs a = {};
  a.q = reinterpret_cast<const void*>(d.x);
  a.q_out = reinterpret_cast<void*>(d.y);
  a.positions = reinterpret_cast<const int*>(d.positions);
  a.q_head = d.x_head ? d.x_head : d.head_dim;
  a.q_token = d.x_token ? d.x_token : uint64_t(d.heads) * d.head_dim;
  a.out_head = d.y_head ? d.y_head : d.head_dim;
  a.out_token = d.y_token ? d.y_token : uint64_t(d.heads) * d.head_dim;
  if (d.y == d.x && ((d.tokens > 1 && a.out_token != a.q_token) || (d.heads > 1 && a.out_head != a.q_head)))
    return fail(KQ_E_INVALID, call, "y may be x with the same strides only");
  a.nq = d.heads;
  a.dim = d.head_dim;
  a.err = ctx->err;
  const bool aligned = on16(d.x) && on16(d.y) && on16(a.q_head * size) && on16(a.q_token * size) &&
                       on16(a.out_head * size) && on16(a.out_token * size);
  return run_rope(a, d.rope, d.type, aligned, d.tokens, d.heads, ctx->sm_count, s, call);
}

int cache_write(kq_ctx* ctx, const kq_cache_write_desc& d, cudaStream_t s) {
  const char* call = "kq_cache_write";
  RopeArgs a = {};
  int rc = check_cache(d.cache, call, &a.cache);
  if (rc) return rc;
  const uint32_t size = type_size(d.type);
  if (!size) return fail(KQ_E_INVALID, call, "type must be F32, F16 or BF16");
  if (d.rope && (!rope_ok(d.rope) || d.rope->rot_dim > d.cache->head_dim))
    return fail(KQ_E_INVALID, call, "rope must come from kq_rope_init with rot_dim up to head_dim");
  if (d.tokens == 0) return KQ_OK;
  if (!d.k || !d.v || !d.slots || (d.rope && !d.positions) || (d.q && !d.q_out))
    return fail(KQ_E_INVALID, call, "null pointer");
  if (d.q && d.n_heads == 0) return fail(KQ_E_INVALID, call, "queries without heads");
  if (d.tokens > 0x7fffffffu || d.n_heads > 0xffffffu)
    return fail(KQ_E_INVALID, call, "too many tokens or heads");
  if (d.q % size || d.k % size || d.v % size || d.q_out % size || d.positions % 4 || d.slots % 8)
    return fail(KQ_E_INVALID, call, "q, k, v and q_out must be aligned to their elements, positions to 4 bytes, "
                                    "slots to 8");
  a.q = reinterpret_cast<const void*>(d.q);
  a.k = reinterpret_cast<const void*>(d.k);
  a.v = reinterpret_cast<const void*>(d.v);
  a.q_out = reinterpret_cast<void*>(d.q_out);
  a.positions = reinterpret_cast<const int*>(d.positions);
  a.slots = reinterpret_cast<const long long*>(d.slots);
  const uint64_t dim = d.cache->head_dim;
  const uint64_t packed = (uint64_t(d.n_heads) + 2ull * d.cache->n_kv) * dim;
  a.q_head = a.out_head = dim;
  a.q_token = d.q_token ? d.q_token : packed;
  a.k_token = d.k_token ? d.k_token : packed;
  a.v_token = d.v_token ? d.v_token : packed;
  // in place by default where q_out is q: rows of another stride would be written over tokens not yet read
  const bool in_place = d.q && d.q_out == d.q;
  a.out_token = d.q_out_token ? d.q_out_token : in_place ? a.q_token : uint64_t(d.n_heads) * dim;
  if (in_place && d.tokens > 1 && a.out_token != a.q_token)
    return fail(KQ_E_INVALID, call, "q_out may be q with q's own token stride only");
  a.nq = d.q ? d.n_heads : 0;
  a.dim = d.cache->head_dim;
  a.err = ctx->err;
  const bool aligned = on16(d.q) && on16(d.k) && on16(d.v) && on16(d.q_out) && on16(a.q_token * size) &&
                       on16(a.k_token * size) && on16(a.v_token * size) && on16(a.out_token * size);
  return run_rope(a, d.rope, d.type, aligned, d.tokens, a.nq + 2 * d.cache->n_kv, ctx->sm_count, s, call);
}

int cache_read(kq_ctx* ctx, const kq_cache_read_desc& d, cudaStream_t s) {
  const char* call = "kq_cache_read";
  CacheView c;
  int rc = check_cache(d.cache, call, &c);
  if (rc) return rc;
  const uint32_t size = type_size(d.type);
  if (!size) return fail(KQ_E_INVALID, call, "type must be F32, F16 or BF16");
  if (d.count == 0 || (!d.k_out && !d.v_out)) return KQ_OK;
  if (!d.slots) return fail(KQ_E_INVALID, call, "null slots");
  if (d.count > 0x7fffffffu) return fail(KQ_E_INVALID, call, "too many rows");
  const uint64_t dense = uint64_t(c.n_kv) * c.dim;
  const uint64_t stride = d.token_stride ? d.token_stride : dense;
  if (stride < dense) return fail(KQ_E_INVALID, call, "token_stride must be at least n_kv * head_dim");
  if (d.k_out % size || d.v_out % size || d.slots % 8)
    return fail(KQ_E_INVALID, call, "k_out and v_out must be aligned to their elements, slots to 8 bytes");
  const bool wide = on16(d.k_out) && on16(d.v_out) && on16(stride * size);
  const auto slots = reinterpret_cast<const long long*>(d.slots);
  // a grid row for each output that is wanted
  const auto go = [&](auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    CacheView view = c;
    T* k = reinterpret_cast<T*>(d.k_out);
    T* v = reinterpret_cast<T*>(d.v_out);
    uint32_t arrays = 2;
    if (!k) {  // values alone, as the grid's first row
      k = v;
      view.k = view.v;
      arrays = 1;
    } else if (!v) {
      arrays = 1;
    }
    constexpr uint32_t E = 16 / sizeof(T);
    const uint32_t per_head = c.dim / E, over_head = static_cast<uint32_t>(((1ull << 32) + per_head - 1) / per_head);
    const uint32_t units = c.n_kv * per_head, parts = (units + kThreads - 1) / kThreads;
    const uint32_t subs = std::max<uint32_t>(1, kThreads / units);
    const uint32_t over_units = static_cast<uint32_t>(((1ull << 32) + units - 1) / units);
    // four rows a thread hide the loads' latency (65536 rows of 1024: 109 -> 71 us, 1001 rows 4.6 -> 4.3);
    // one where that would leave SMs idle
    const bool many = uint64_t(d.count) / subs * parts * arrays >= 32u * ctx->sm_count;
    const auto run = [&](auto kind) {
      constexpr int K = decltype(kind)::value;
      const uint32_t rows = subs * (many ? 4 : 1);
      return launch_pdl(many ? cache_read_kernel<T, K, 4> : cache_read_kernel<T, K, 1>,
                        dim3((d.count + rows - 1) / rows, parts, arrays), kThreads, 0, s, view, k, v, slots, stride,
                        d.count, units, subs, over_units, per_head, over_head, wide, ctx->err);
    };
    return c.kind == KQ_CACHE_F16  ? run(std::integral_constant<int, KQ_CACHE_F16>())
           : c.kind == KQ_CACHE_Q8 ? run(std::integral_constant<int, KQ_CACHE_Q8>())
                                   : run(std::integral_constant<int, KQ_CACHE_Q4>());
  };
  const cudaError_t e = d.type == KQ_TYPE_F32   ? go(static_cast<float*>(nullptr))
                        : d.type == KQ_TYPE_F16 ? go(static_cast<__half*>(nullptr))
                                                : go(static_cast<__nv_bfloat16*>(nullptr));
  return e == cudaSuccess ? KQ_OK : cuda_fail(e, "cudaLaunchKernelExC", call);
}

int cache_move(kq_ctx* ctx, const kq_cache_move_desc& d, cudaStream_t s) {
  const char* call = "kq_cache_move";
  CacheView c;
  int rc = check_cache(d.cache, call, &c);
  if (rc) return rc;
  if (d.groups == 0 || d.moves == 0) return KQ_OK;
  if (!d.src || !d.dst || !d.starts) return fail(KQ_E_INVALID, call, "null pointer");
  if (d.src % 8 || d.dst % 8 || d.starts % 4)
    return fail(KQ_E_INVALID, call, "src and dst must be 8-byte aligned, starts 4-byte aligned");
  if (d.groups > 0x7fffffffu || d.moves > 0x7fffffffu) return fail(KQ_E_INVALID, call, "too many moves");
  const cudaError_t e = launch_pdl(cache_move_kernel, dim3(d.groups, c.n_kv, 2), kThreads,
                                   std::min(d.moves, kMaxMoves) * c.row, s, c, reinterpret_cast<const long long*>(d.src),
                                   reinterpret_cast<const long long*>(d.dst), reinterpret_cast<const int*>(d.starts),
                                   d.moves, ctx->err);
  return e == cudaSuccess ? KQ_OK : cuda_fail(e, "cudaLaunchKernelExC", call);
}

}  // namespace kq
