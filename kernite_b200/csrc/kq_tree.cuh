// kq_tree.cuh -- attention of drafted tokens over the paged cache: how the work is cut, and the
// warp-MMA kernel. The caches' three kinds are compiled in a file each (kq_tree_f16.cu, kq_tree_q8.cu,
// kq_tree_q4.cu); kq_tree.cu dispatches and joins split items.
//
// The work. An item is (sequence, key/value head, tile of rows): a row is a drafted token with one of
// the head's group of query heads, r = token * group + head, so that a position's key and value serve
// all of them. An item's positions come in tiles of TW (64 or 128). The tiles of all items, in order, are cut
// into equal ranges, one a CTA, whatever the sequences' lengths: a CTA does the end of one item, some
// whole ones and the start of another. Whole ones are written out; parts leave (max, sum, unnormalised
// output) in the workspace, two slots a CTA at most, and the join kernel finds by the same arithmetic
// which CTAs hold an item's parts. So a long context is split over the whole GPU, and a ragged batch leaves
// no CTA idle.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "kq_cache.cuh"
#include "kq_device.cuh"
#include "kq_launch.h"

namespace kq {
namespace tree {

constexpr uint32_t kTile = 128;      // positions a tile of the warp-MMA kernel
constexpr uint32_t kMaxDrafts = 64;  // bits of a mask word

struct TreeArgs {
  CacheView c;
  const void* q;
  void* out;
  uint64_t q_token, out_token;
  const int* starts;
  const int* prefix;
  const int* pages;
  const unsigned long long* mask;
  float* part;
  uint4* splits;  // two a CTA: Split
  float scale_log2;
  uint32_t n_seq, n_heads, group, tokens, max_drafts, max_pages;
  uint32_t per_group;  // ceil(2^32 / group); 0 for a group of one
  uint32_t type;
  unsigned* err;
};

// Row r's drafted token and query head in the group (r < 2^16, so the product is exact).
__device__ __forceinline__ uint32_t token_of(const TreeArgs& a, uint32_t r) {
  return a.per_group ? __umulhi(r, a.per_group) : r;
}
__device__ __forceinline__ uint32_t head_of(const TreeArgs& a, uint32_t r, uint32_t token) { return r - token * a.group; }

// A sequence as the kernels take it: no drafts when there are none, or when its numbers do not fit
// (recorded in the error word).
struct Seq {
  uint32_t first, drafts, prefix;
  __device__ uint32_t length() const { return prefix + drafts; }
};

__device__ __forceinline__ Seq load_seq(const TreeArgs& a, uint32_t s) {
  const int b = a.starts[s], e = a.starts[s + 1], p = a.prefix[s];
  Seq q = {static_cast<uint32_t>(b), static_cast<uint32_t>(e - b), static_cast<uint32_t>(p)};
  const bool ok = b >= 0 && e >= b && static_cast<uint32_t>(e) <= a.tokens && q.drafts <= a.max_drafts &&
                  p >= 0 && uint64_t(q.prefix) + q.drafts <= uint64_t(a.max_pages) << a.c.page_log2;
  if (!ok) {
    report_error(a.err, kErrCacheRange);
    q.drafts = 0;
  }
  return q;
}

template <uint32_t ROWS>
__device__ __forceinline__ uint32_t row_tiles(const TreeArgs& a, const Seq& s) {
  return (s.drafts * a.group + ROWS - 1) / ROWS;
}

template <uint32_t TW>
__device__ __forceinline__ uint32_t position_tiles(const Seq& s) {
  return (s.length() + TW - 1) / TW;
}

template <uint32_t ROWS, uint32_t TW>
__device__ __forceinline__ uint64_t seq_work(const TreeArgs& a, const Seq& s) {
  return s.drafts ? uint64_t(position_tiles<TW>(s)) * a.c.n_kv * row_tiles<ROWS>(a, s) : 0;
}

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// All sequences' tiles; the first 32 sequences stay in the warp's lanes. Made by whole warps.
template <uint32_t ROWS, uint32_t TW>
struct Work {
  Seq seq;         // of sequence `lane`
  uint64_t tiles;  // its tiles
  uint64_t total;

  __device__ explicit Work(const TreeArgs& a) {
    const uint32_t lane = threadIdx.x % 32;
    seq = Seq{0, 0, 0};
    if (lane < a.n_seq) seq = load_seq(a, lane);
    tiles = seq_work<ROWS, TW>(a, seq);
    uint64_t w = tiles;
    for (uint32_t s = 32 + lane; s < a.n_seq; s += 32) w += seq_work<ROWS, TW>(a, load_seq(a, s));
    total = warp_sum(w);
  }
};

// Where a CTA is: an item and the next of its tiles.
struct Place {
  Seq seq;
  uint32_t s, head, rows;  // sequence, key/value head, row tile
  uint32_t tile;
};

// The place of tile `at` of the whole work. Called by whole warps, at < total.
template <uint32_t ROWS, uint32_t TW>
__device__ __forceinline__ Place locate(const TreeArgs& a, const Work<ROWS, TW>& work, uint64_t at) {
  const uint32_t lane = threadIdx.x % 32;
  Place p = {};
  Seq seq = work.seq;
  uint64_t w = work.tiles;
  for (uint32_t s0 = 0; s0 < a.n_seq; s0 += 32) {
    if (s0) {
      seq = Seq{0, 0, 0};
      if (s0 + lane < a.n_seq) seq = load_seq(a, s0 + lane);
      w = seq_work<ROWS, TW>(a, seq);
    }
    uint64_t upto = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, upto > at);
    if (past) {
      const int who = __ffs(past) - 1;
      p.s = s0 + who;
      const uint32_t rest = static_cast<uint32_t>(at - __shfl_sync(0xffffffffu, upto - w, who));
      p.seq.first = __shfl_sync(0xffffffffu, seq.first, who);
      p.seq.drafts = __shfl_sync(0xffffffffu, seq.drafts, who);
      p.seq.prefix = __shfl_sync(0xffffffffu, seq.prefix, who);
      const uint32_t pt = position_tiles<TW>(p.seq), rt = row_tiles<ROWS>(a, p.seq);
      const uint32_t item = rest / pt;
      p.tile = rest - item * pt;
      p.head = item / rt;
      p.rows = item - p.head * rt;
      return p;
    }
    at -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return p;
}

// The item after p's, at its first tile.
template <uint32_t ROWS>
__device__ __forceinline__ void next_item(const TreeArgs& a, Place& p) {
  p.tile = 0;
  if (++p.rows < row_tiles<ROWS>(a, p.seq)) return;
  p.rows = 0;
  if (++p.head < a.c.n_kv) return;
  p.head = 0;
  do {
    if (++p.s >= a.n_seq) return;
    p.seq = load_seq(a, p.s);
  } while (p.seq.drafts == 0);
}

// CTA c of n <= total takes tiles [range_start(c), range_start(c + 1)) of `total`, at least one (n < 2^16,
// so that where total has 32 bits, all of this has: 64-bit divisions are calls of some 100 cycles).
__device__ __forceinline__ uint64_t range_start(uint64_t total, uint32_t c, uint32_t n) {
  if (total >> 32 == 0) {
    const uint32_t whole = static_cast<uint32_t>(total) / n;
    return uint64_t(whole) * c + (static_cast<uint32_t>(total) - whole * n) * c / n;
  }
  return total / n * c + total % n * c / n;
}

// Which CTA has tile `at` < total: the largest c with floor(total c / n) <= at.
__device__ __forceinline__ uint32_t range_owner(uint64_t total, uint64_t at, uint32_t n) {
  return static_cast<uint32_t>(((at + 1) * n - 1) / total);
}

// Floats of one slot of partial results: rows x pitch outputs, then rows maxima and rows sums.
__host__ __device__ constexpr uint64_t part_floats(uint32_t rows, uint32_t pitch) {
  return uint64_t(rows) * (pitch + 2);
}

// What a CTA tells the join kernel of an item that it began and others went on with: the last of those,
// the item. (CTA 0 is never the last, so 0 says that there is none.)
struct Split {
  uint32_t last, rows, head, drafts, first;
  __device__ static Split load(const TreeArgs& a, uint32_t cta) {
    const uint4 x = a.splits[2 * cta], y = a.splits[2 * cta + 1];
    return {x.x, x.y, x.z, x.w, y.x};
  }
  __device__ void store(const TreeArgs& a, uint32_t cta) const {
    a.splits[2 * cta] = make_uint4(last, rows, head, drafts);
    a.splits[2 * cta + 1] = make_uint4(first, 0, 0, 0);
  }
};

// By one thread of each CTA, once: after its last item p (end: one past its tiles, of n, of which it did the
// item's first ones or not), or for a CTA without work.
__device__ __forceinline__ void leave_split(const TreeArgs& a, const Place& p, bool began, bool whole, uint64_t total,
                                            uint64_t end, uint32_t done, uint32_t tiles, uint32_t n) {
  Split s = {0, 0, 0, 0, 0};
  if (began && !whole) s = {range_owner(total, end - done + tiles - 1, n), p.rows, p.head, p.seq.drafts, p.seq.first};
  s.store(a, blockIdx.x);
}

// Whether row token t (of the sequence) sees position pos.
__device__ __forceinline__ bool sees(unsigned long long bits, uint32_t pos, const Seq& s) {
  return pos < s.prefix || (pos < s.length() && (bits >> (pos - s.prefix) & 1ull));
}

__device__ __forceinline__ unsigned long long mask_bits(const TreeArgs& a, const Seq& s, uint32_t t) {
  // without a mask the drafts up to t; bits of drafts that are not there do not count
  return (a.mask ? a.mask[s.first + t] : (2ull << t) - 1ull) & ~0ull >> (kMaxDrafts - s.drafts);
}

// Bit i: whether position base + c + i is seen, base + c = the prefix's end + from (i < 32).
__device__ __forceinline__ uint32_t seen_word(unsigned long long bits, int from) {
  if (from <= -32) return ~0u;
  if (from >= static_cast<int>(kMaxDrafts)) return 0u;
  return from < 0 ? static_cast<uint32_t>(bits << -from) | ((1u << -from) - 1u) : static_cast<uint32_t>(bits >> from);
}

__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// Elements at(0), at(1), .. of q from element `row` on, N (4 or 8) each; zeros from element `dim` on and
// where there is no row. All loads are issued before any is looked at, so that they are one latency: a
// choice of type at each would wait for each (4 sequences of 64 drafts: 138 -> 132 us).
template <uint32_t COUNT, uint32_t N, class At>
__device__ __forceinline__ void load_row(const TreeArgs& a, uint64_t row, bool have, const At& at,
                                         float (&x)[COUNT][N]) {
  const uint32_t dim = have ? a.c.dim : 0;
  if (a.type == KQ_TYPE_F32) {
    const float* q = static_cast<const float*>(a.q) + row;
#pragma unroll
    for (uint32_t j = 0; j < COUNT; ++j)
#pragma unroll
      for (uint32_t k = 0; k < N; k += 4) {
        const float4 v = at(j) < dim ? *reinterpret_cast<const float4*>(q + at(j) + k) : make_float4(0, 0, 0, 0);
        x[j][k] = v.x;
        x[j][k + 1] = v.y;
        x[j][k + 2] = v.z;
        x[j][k + 3] = v.w;
      }
    return;
  }
  uint32_t w[COUNT][N / 2];
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + row;
#pragma unroll
  for (uint32_t j = 0; j < COUNT; ++j) {
    if constexpr (N == 8) {
      const uint4 v = at(j) < dim ? *reinterpret_cast<const uint4*>(q + at(j)) : make_uint4(0, 0, 0, 0);
      w[j][0] = v.x;
      w[j][1] = v.y;
      w[j][2] = v.z;
      w[j][3] = v.w;
    } else {
      const uint2 v = at(j) < dim ? *reinterpret_cast<const uint2*>(q + at(j)) : make_uint2(0, 0);
      w[j][0] = v.x;
      w[j][1] = v.y;
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < COUNT; ++j)
#pragma unroll
    for (uint32_t k = 0; k < N; k += 2) {
      float2 v;
      if (a.type == KQ_TYPE_F16) v = __half22float2(as_h2(w[j][k / 2]));
      else v = make_float2(__uint_as_float(w[j][k / 2] << 16), __uint_as_float(w[j][k / 2] & 0xffff0000u));
      x[j][k] = v.x;
      x[j][k + 1] = v.y;
    }
}

__device__ __forceinline__ void store_one(void* p, uint64_t i, float v, uint32_t type) {
  if (type == KQ_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == KQ_TYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------- the warp-MMA kernel
//
// For few rows (8 an item). mma.sync.m16n8k16 (f16 in, f32 accumulated), operands from registers: the
// positions are M of S^T = K Q^T, the head's elements M of O^T += V^T P^T, and the rows N = 8 of both, so
// no part of an MMA is spent on rows that are not there; P^T comes from S^T by movmatrix. Seven warps take
// 32 positions each in turn and keep separate maxima, sums and outputs, joined at an item's end; the
// eighth copies tiles of 128 positions into a ring, ahead over items' ends. For f32 activations Q and P are
// sums of two f16 (about 22 bits): two MMAs into one sum.
//
// Codes become f16 in registers, exactly. The order of a contraction is free, so a thread's piece of a
// key row is 16 consecutive bytes, and the element M index of V^T is chosen the same way. Index n of 8
// positions is position pi(n) = 4 (n mod 2) + n / 2: with the cache's unit permutation the reads of a warp
// then meet no bank twice.
//
// What bounds it. Read once, 8-bit keys and values come at the memory's rate: 32 sequences of 64 / 8 heads of
// 128, one f32 token each, take 63 us at 4096 positions and 106 us at 8192, so the second half at 6.5 TB/s; the
// first 20 us are launches, the lengths' and pages' latencies, the items' ends and the join. 16-bit ones take
// 90 us at 4096 (85 at the copy rate). In 4 bits there are half the bytes and an eighth more instructions: one token
// over 131001 positions takes 64 us, 2.2 TB/s, and 57600 instructions a scheduler, 56 % of its issue slots (of
// the integer pipe 50 %, of the tensor pipe 27 %). No pipe is full: the rest is latency, with 3.5 warps a
// scheduler. Parts of 16 positions a warp, one chain of latencies, took 69 us.
// Why seven readers and one copier: a warp that copies in its turn makes its tile late (77 us against 68).
// Why one pass: a maximum that only ever grows costs a rescaling of O when it does, which kSlack makes rare.

constexpr uint32_t kReaders = 7;
constexpr uint32_t kThreads = (kReaders + 1) * 32;
constexpr uint32_t kSubs = 2;                     // times 16 positions a warp takes at once: two chains of
constexpr uint32_t kPart = 16 * kSubs;            // latencies side by side
constexpr uint32_t kParts = kTile / kPart;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same without a sum so far.
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// The transpose of an 8 x 8 matrix of 16-bit elements, two of a row a thread.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// 2^x, to 2^-22 of it; results below f32's normal range are zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Codes as f16 pairs: a code under the exponent of 1024 is 1024 + u (8 bits) or 1024 + 16 u (a nibble
// at bits 4..7), and one fused multiply-add gives (u - offset) * scale, exactly (kq_cache.cuh).
constexpr uint32_t kMagic = 0x64646464u;

// A block's scale for decode2: the factor and the subtrahend, twice each.
struct Scale2 {
  __half2 by, minus;
};

template <uint32_t KIND>
__device__ __forceinline__ Scale2 scale2(uint32_t low_byte, uint32_t high_byte) {
  const __half2 s = as_h2(low_byte << 7 | high_byte << 23);
  if constexpr (KIND == KQ_CACHE_Q4)
    return {__hmul2(s, __float2half2_rn(0.0625f)), __hmul2(s, __float2half2_rn(-72.f))};
  else
    return {s, __hmul2(s, __float2half2_rn(-1152.f))};
}

__device__ __forceinline__ uint32_t decode2(uint32_t magic, const Scale2& s) {
  return h2(__hfma2(as_h2(magic), s.by, s.minus));
}

// Nibble e (0..3) of both halves of v moved to bits 4..7.
__device__ __forceinline__ constexpr uint32_t nibble_up(uint32_t v, uint32_t e) {
  return e == 0 ? v << 4 : v >> (4 * e - 4);
}

// The nibbles at bits 4..7 of both halves of v.
__device__ __forceinline__ uint32_t nibbles(uint32_t v) { return (v & 0x00f000f0u) | (kMagic & 0xff00ff00u); }

// hi + lo of a pair of f32: f16(x), f16(x - f16(x)).
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = h2(h);
  lo = h2(__floats2half2_rn(x - f.x, y - f.y));
}

// How a row of q becomes an f16 operand: times `up`; and the logits (in log2 units) of the product: times
// `unit`. The power of two in `up` brings the row's largest magnitude (most) to [2^7, 2^8) (or, split, near
// it), so that f16's range fits any q; it is 1 for a row of zeros or with infinities. 16-bit rows stay exact
// but for elements below 2^-21 of the row's largest, which are rounded at 2^-32 of it; split ones take the
// softmax's scale along, so that `unit` is a power of two and a product's largest logit is the maximum exactly,
// however large. unit is never zero: masked logits are -inf times it.
struct RowScale {
  float up, unit;
};

template <bool SPLIT>
__device__ __forceinline__ RowScale row_scale(float most, float scale_log2) {
  const int ex = static_cast<int>(__float_as_uint(most) >> 23) - 127;
  const int sh = most > 0.f && ex < 128 ? min(max(7 - ex, -120), 120) : 0;
  const float up = __int_as_float((127 + sh) << 23), down = __int_as_float((127 - sh) << 23);
  if constexpr (SPLIT) {
    // scale_log2 = fraction x power of two, the fraction in [1, 2)
    const uint32_t bits = __float_as_uint(scale_log2);
    const float part = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
    const float power = __uint_as_float(bits & 0x7f800000u);
    return {up * part, fmaxf(down * power, 0x1p-149f)};
  }
  return {up, fmaxf(down * scale_log2, 0x1p-149f)};
}

// How a head of pitch D lies in rows of codes, per kind: bytes of a row, EK elements of a thread's piece of
// a key row, EV of its piece of a value row.
template <uint32_t KIND, uint32_t D>
struct Shape {
  static constexpr uint32_t kBits = KIND == KQ_CACHE_F16 ? 16 : KIND == KQ_CACHE_Q8 ? 8 : 4;
  static constexpr uint32_t kRow = D * kBits / 8;
  static constexpr uint32_t kScales = KIND == KQ_CACHE_F16 ? 0 : D / 32;
  static constexpr uint32_t kMost = 128 / kBits;  // elements of 16 bytes
  static constexpr uint32_t EK = kMost < D / 4 ? kMost : D / 4;
  static constexpr uint32_t EV = kMost < D / 8 ? kMost : D / 8;
  static constexpr uint32_t kSteps = D / 16;      // MMAs along a head
  static constexpr bool kPermuted = EV * kBits == 128;  // value pieces of 16 bytes go in the order pi
  static constexpr uint32_t kSlot = kTile * (kRow + kScales);
};

__device__ __forceinline__ uint32_t pi8(uint32_t n) { return ((n & 1u) << 2) | (n >> 1); }

// First of the four elements of step ks in thread t's key pieces.
template <class S>
__device__ __forceinline__ constexpr uint32_t key_element(uint32_t ks, uint32_t t) {
  return S::EK * (t + 4 * (ks / (S::EK / 4))) + 4 * (ks % (S::EK / 4));
}

// The element that M index g (h = 0) or g + 8 (h = 1) of O^T's tile j stands for.
template <class S>
__device__ __forceinline__ uint32_t value_element(uint32_t j, uint32_t g, uint32_t h) {
  return S::EV * (8 * (j / (S::EV / 2)) + (S::kPermuted ? pi8(g) : g)) + 2 * (j % (S::EV / 2)) + h;
}

// `B` bytes of shared memory as words.
template <uint32_t B>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[B / 4]) {
  if constexpr (B == 16) {
    const uint4 v = lds_v4(addr);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  } else if constexpr (B == 8) {
    const uint2 v = lds_v2(addr);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    w[0] = lds_u32(addr);
  }
}

__device__ __forceinline__ uint32_t lds_u8(uint32_t addr) {
  uint16_t v;
  asm volatile("{.reg .u8 b; ld.shared.u8 %0, [%1];}" : "=h"(v) : "r"(addr));
  return v;
}

// The numbers of a tile's pages, as the table has them.
template <uint32_t TW>
struct PageIds {
  uint32_t id[TW / 16];

  __device__ __forceinline__ void load(const TreeArgs& a, const Place& p) {
    const uint32_t base = p.tile * TW, length = p.seq.length();
    const int* row = a.pages + uint64_t(p.s) * a.max_pages + (base >> a.c.page_log2);
    const uint32_t n = (min(TW, length - base) + a.c.page() - 1) >> a.c.page_log2;
    id[0] = static_cast<uint32_t>(row[0]);
#pragma unroll
    for (uint32_t i = 1; i < TW / 16; ++i) id[i] = i < n ? static_cast<uint32_t>(row[i]) : 0u;
  }
};

// One thread's copies of a tile: whole records where a page is at most a tile, else its rows and its
// scales. A page that is not there is recorded, and page 0 copied.
template <class S, uint32_t TW>
__device__ __forceinline__ void copy_tile(const TreeArgs& a, const Place& p, const PageIds<TW>& ids,
                                          const uint8_t* src, uint32_t dst, uint32_t bar) {
  constexpr uint32_t row = S::kRow + S::kScales;
  const uint32_t base = p.tile * TW, left = p.seq.length() - base;
  const auto record = [&](uint32_t id) {
    if (id >= a.c.n_pages) {
      report_error(a.err, kErrCacheRange);
      id = 0;
    }
    return src + a.c.at(id, p.head);
  };
  if (a.c.page() > TW) {
    const uint8_t* rec = record(ids.id[0]);
    const uint32_t at = base & (a.c.page() - 1);
    mbar_arrive_expect_tx(bar, TW * row);
    bulk_g2s(dst, rec + at * S::kRow, TW * S::kRow, bar);
    if constexpr (S::kScales != 0)
      bulk_g2s(dst + TW * S::kRow, rec + a.c.page() * S::kRow + at * S::kScales, TW * S::kScales, bar);
    return;
  }
  const uint32_t n = (min(TW, left) + a.c.page() - 1) >> a.c.page_log2, bytes = row << a.c.page_log2;
  mbar_arrive_expect_tx(bar, n * bytes);
#pragma unroll
  for (uint32_t i = 0; i < TW / 16; ++i)
    if (i < n) bulk_g2s(dst + i * bytes, record(ids.id[i]), bytes, bar);
}

// Positions of a tile in shared memory: where a position's row starts (its swizzle apart) and its
// scale bytes.
template <class S>
struct TileView {
  uint32_t base, seg_log2;
  __device__ uint32_t seg_base(uint32_t p) const {
    return base + ((p >> seg_log2) << seg_log2) * (S::kRow + S::kScales);
  }
  __device__ uint32_t code(uint32_t p, uint32_t byte) const {
    return seg_base(p) + cache_offset(p & ((1u << seg_log2) - 1), byte, S::kRow);
  }
  __device__ uint32_t scale(uint32_t p) const {
    return seg_base(p) + (S::kRow << seg_log2) + (p & ((1u << seg_log2) - 1)) * S::kScales;
  }
};

// A warp's copies of a tile of kTile positions, lane i's of segment i (a page, or a tile's part of one):
// its record, or where a page is longer than a tile its rows and its scales. id: the segment's page. A
// page that is not there is recorded, and page 0 copied.
template <class S>
__device__ __forceinline__ void copy_segments(const TreeArgs& a, const Place& p, uint32_t id, const uint8_t* src,
                                              uint32_t dst, uint32_t bar) {
  constexpr uint32_t row = S::kRow + S::kScales;
  const uint32_t lane = threadIdx.x % 32, base = p.tile * kTile;
  const uint32_t seg_log2 = min(a.c.page_log2, 7u), bytes = row << seg_log2;
  const uint32_t n = (min(kTile, p.seq.length() - base) + (1u << seg_log2) - 1) >> seg_log2;
  if (id >= a.c.n_pages) {
    report_error(a.err, kErrCacheRange);
    id = 0;
  }
  const uint8_t* rec = src + a.c.at(id, p.head);
  if (lane == 0) mbar_arrive_expect_tx(bar, n * bytes);
  __syncwarp();
  if (lane < n) {
    if (a.c.page_log2 <= 7) {
      bulk_g2s(dst + lane * bytes, rec, bytes, bar);
    } else {  // a page of two tiles
      const uint32_t at = base & (a.c.page() - 1);
      bulk_g2s(dst, rec + at * S::kRow, kTile * S::kRow, bar);
      if constexpr (S::kScales != 0)
        bulk_g2s(dst + kTile * S::kRow, rec + a.c.page() * S::kRow + at * S::kScales, kTile * S::kScales, bar);
    }
  }
}

// f16 pairs whose exponent is all ones (infinity, NaN) become zero.
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t v) {
  if ((v & 0x7c00u) == 0x7c00u) v &= 0xffff0000u;
  if ((v & 0x7c000000u) == 0x7c000000u) v &= 0x0000ffffu;
  return v;
}

// Shared memory of the warp-MMA kernel: the ring of key and value tiles, the join of the warps (four at a
// time), Q where registers are short. Two CTAs a SM where five slots fit twice, so that one's waits and
// joins are the other's time.
template <uint32_t KIND, uint32_t D>
struct Narrow {
  using S = Shape<KIND, D>;
  static constexpr uint32_t kJoinRow = D + 16;
  static constexpr uint32_t kJoin = 4 * 8 * kJoinRow * 4 + 4 * 8 * 2 * 4;
  static constexpr bool kQShared = D >= 128;
  static constexpr uint32_t kQ = kQShared ? S::kSteps * 32 * 16 : 0;
  static constexpr uint32_t kFixed = kJoin + kQ + 256;
  static constexpr uint32_t kCtas = kFixed + 5 * S::kSlot <= 113 * 1024 ? 2 : 1;
  static constexpr uint32_t kFit = ((kCtas == 2 ? 113 : 226) * 1024 - kFixed) / S::kSlot;
  static constexpr uint32_t kSlots = kFit > 12 ? 12 : kFit;  // keys and values in turn
  static constexpr uint32_t kBytes = kFixed + kSlots * S::kSlot;
  static_assert(kSlots >= 2, "a tile");
};

// Where a lane's pieces lie in 16 positions. Of its two key positions pi(g), pi(g) + 8 and four value
// positions t, t + 4, t + 8, t + 12 the ones 8 apart differ by 8 rows (their units are permuted alike); a
// key row's pieces are 4 units apart, the second in the other half of a line of 128 bytes.
template <class S>
struct Lane {
  uint32_t key[2], value[2], key_scale, value_scale;

  __device__ Lane(uint32_t g, uint32_t t) {
    const uint32_t pg = S::kPermuted ? pi8(g) : g;
    constexpr uint32_t BK = S::EK * S::kBits / 8, BV = S::EV * S::kBits / 8;
    key[0] = cache_offset(pi8(g), BK * t, S::kRow);
    key[1] = key[0] ^ 64u;
    value[0] = cache_offset(t, BV * pg, S::kRow);
    value[1] = cache_offset(t + 4, BV * pg, S::kRow);
    key_scale = pi8(g) * S::kScales + S::EK * t / 32;
    value_scale = t * S::kScales + S::EV * pg / 32;
  }
};

// Where 16 positions (from p0 on, in a tile) lie: the first one's row and scales. A segment (a page, or a
// tile's part of one) is its rows and then its scales; 16 rows are whole lines of 128 bytes, so the
// permutation is that of the positions in them.
template <class S>
struct PartView {
  uint32_t code, scale;

  __device__ PartView(uint32_t slot, uint32_t p0, uint32_t seg_log2) {
    const uint32_t in = p0 & ((1u << seg_log2) - 1);
    const uint32_t seg = slot + (p0 - in) * (S::kRow + S::kScales);
    code = seg + in * S::kRow;
    scale = seg + (S::kRow << seg_log2) + in * S::kScales;
  }
};

// S^T of the warp's positions, 16 at a time: c = sum of K Q^T over the head, q the rows' operand B (hi, lo).
template <uint32_t KIND, uint32_t D, bool SPLIT, class Q>
__device__ __forceinline__ void key_product(const PartView<Shape<KIND, D>> (&part)[kSubs],
                                            const Lane<Shape<KIND, D>>& at, const Q& q, float (&c)[kSubs][4]) {
  using S = Shape<KIND, D>;
  constexpr uint32_t B = S::EK * S::kBits / 8;
  float acc[kSubs][2][4];  // two sums each: an MMA's result is some 20 cycles away
#pragma unroll
  for (uint32_t s = 0; s < kSubs; ++s)
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) acc[s][i][k] = 0.f;
#pragma unroll
  for (uint32_t j = 0; j < D / 4 / S::EK; ++j) {
    uint32_t w[kSubs][2][B / 4];
    Scale2 scale[kSubs][2];
#pragma unroll
    for (uint32_t s = 0; s < kSubs; ++s)
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        lds_words<B>(part[s].code + at.key[j & 1] + h * 8 * S::kRow + (j >> 1) * 128, w[s][h]);
        if constexpr (S::kScales != 0) {
          const uint32_t b = lds_u8(part[s].scale + at.key_scale + h * 8 * S::kScales + j * (S::EK * 4 / 32));
          scale[s][h] = scale2<KIND>(b, b);
        }
      }
#pragma unroll
    for (uint32_t k = 0; k < S::EK / 4; ++k) {
      const uint32_t ks = j * (S::EK / 4) + k;
      uint32_t b[4];
      q(ks, b);
#pragma unroll
      for (uint32_t s = 0; s < kSubs; ++s) {
        uint32_t f[2][2];  // positions pi(g) and pi(g) + 8, the step's first and last two elements
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          if constexpr (KIND == KQ_CACHE_F16) {
            f[h][0] = w[s][h][2 * k];
            f[h][1] = w[s][h][2 * k + 1];
          } else if constexpr (KIND == KQ_CACHE_Q8) {
            f[h][0] = decode2(prmt(w[s][h][k], kMagic, 0x4140), scale[s][h]);
            f[h][1] = decode2(prmt(w[s][h][k], kMagic, 0x4342), scale[s][h]);
          } else {
            f[h][0] = decode2(nibbles(nibble_up(w[s][h][k / 2], 2 * (k % 2))), scale[s][h]);
            f[h][1] = decode2(nibbles(nibble_up(w[s][h][k / 2], 2 * (k % 2) + 1)), scale[s][h]);
          }
        }
        mma16816(acc[s][SPLIT ? 0 : ks & 1], f[0][0], f[1][0], f[0][1], f[1][1], b[0], b[1]);
        if constexpr (SPLIT) mma16816(acc[s][1], f[0][0], f[1][0], f[0][1], f[1][1], b[2], b[3]);
      }
    }
  }
#pragma unroll
  for (uint32_t s = 0; s < kSubs; ++s)
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) c[s][k] = acc[s][0][k] + acc[s][1][k];
}

__device__ __forceinline__ void add_to(float (&o)[4], const float (&c)[4]) {
#pragma unroll
  for (uint32_t i = 0; i < 4; i += 2) {
    const float2 s = add2(make_float2(o[i], o[i + 1]), make_float2(c[i], c[i + 1]));
    o[i] = s.x;
    o[i + 1] = s.y;
  }
}

// O^T += V^T P^T of 16 of the warp's positions, b the weights as operand B (hi, and lo). EDGE: the tile
// reaches past the prefix, so rows past the end (left: positions the tile has) and values that are not
// finite count as zero here (P is zero where a position is masked, and zero times those would not be);
// the caller adds the latter where they are seen. APART (f32 activations): the sum so far is added by an f32
// addition; the tensor core's cuts off what it cannot hold, which over a long context is a loss that grows
// with the additions. Half of them apart bring the result nearer than f32 torch (131001 positions: relative
// error 1.3e-6 -> 7e-7, torch 8e-7) and cost nothing; all of them 3e-7, but registers spill (32 sequences
// 74 -> 80 us).
template <uint32_t KIND, uint32_t D, bool SPLIT, bool EDGE, bool APART>
__device__ __forceinline__ void value_product(const PartView<Shape<KIND, D>>& part,
                                              const Lane<Shape<KIND, D>>& at, uint32_t first,
                                              uint32_t left, const uint32_t (&b)[4], float (&o)[D / 16][4]) {
  using S = Shape<KIND, D>;
  constexpr uint32_t B = S::EV * S::kBits / 8;
#pragma unroll
  for (uint32_t jj = 0; jj < D / 8 / S::EV; ++jj) {
    uint32_t w[4][B / 4];
    uint32_t byte[4] = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {  // position first + 4 i
      lds_words<B>(part.code + at.value[i & 1] + (i >> 1) * 8 * S::kRow + jj * 128, w[i]);
      const bool there = !EDGE || first + 4 * i < left;
      if constexpr (KIND == KQ_CACHE_F16) {
        if constexpr (EDGE) {
#pragma unroll
          for (uint32_t k = 0; k < B / 4; ++k) w[i][k] = there ? finite_or_zero(w[i][k]) : 0u;
        }
      } else {
        byte[i] = lds_u8(part.scale + at.value_scale + i * 4 * S::kScales + jj * (S::EV * 8 / 32));
        if constexpr (EDGE) byte[i] = there && byte[i] < 0xf8u ? byte[i] : 0u;
      }
    }
    Scale2 s[2];
    if constexpr (S::kScales != 0) {
      s[0] = scale2<KIND>(byte[0], byte[1]);
      s[1] = scale2<KIND>(byte[2], byte[3]);
    }
    const auto product = [&](uint32_t j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
      if constexpr (SPLIT && APART) {
        float c[4];
        mma16816_first(c, a0, a1, a2, a3, b[2], b[3]);
        mma16816(c, a0, a1, a2, a3, b[0], b[1]);
        add_to(o[j], c);
      } else {
        mma16816(o[j], a0, a1, a2, a3, b[0], b[1]);
        if constexpr (SPLIT) mma16816(o[j], a0, a1, a2, a3, b[2], b[3]);
      }
    };
#pragma unroll
    for (uint32_t k = 0; k < B / 4; ++k) {
      // pairs (position first, + 4) and (+ 8, + 12) of each element of word k
      const uint32_t j0 = jj * (S::EV / 2);
      if constexpr (KIND == KQ_CACHE_F16) {
        product(j0 + k, prmt(w[0][k], w[1][k], 0x5410), prmt(w[0][k], w[1][k], 0x7632),
                prmt(w[2][k], w[3][k], 0x5410), prmt(w[2][k], w[3][k], 0x7632));
      } else if constexpr (KIND == KQ_CACHE_Q8) {
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
          const uint32_t x = prmt(w[0][k], w[1][k], half ? 0x7362 : 0x5140);
          const uint32_t y = prmt(w[2][k], w[3][k], half ? 0x7362 : 0x5140);
          product(j0 + 2 * k + half, decode2(prmt(x, kMagic, 0x4140), s[0]), decode2(prmt(x, kMagic, 0x4342), s[0]),
                  decode2(prmt(y, kMagic, 0x4140), s[1]), decode2(prmt(y, kMagic, 0x4342), s[1]));
        }
      } else {
        // elements 2 e at nibbles e of the low halves, 2 e + 1 of the high ones
        const uint32_t x0 = prmt(w[0][k], w[1][k], 0x5410), x1 = prmt(w[0][k], w[1][k], 0x7632);
        const uint32_t y0 = prmt(w[2][k], w[3][k], 0x5410), y1 = prmt(w[2][k], w[3][k], 0x7632);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          product(j0 + 4 * k + e, decode2(nibbles(nibble_up(x0, e)), s[0]), decode2(nibbles(nibble_up(x1, e)), s[0]),
                  decode2(nibbles(nibble_up(y0, e)), s[1]), decode2(nibbles(nibble_up(y1, e)), s[1]));
      }
    }
  }
}

// Of the warp's positions p0 .. p0 + 31 below `left`, those with a value that is not finite, as bits.
template <uint32_t KIND, uint32_t D>
__device__ __noinline__ uint32_t special_positions(TileView<Shape<KIND, D>> tile, uint32_t p0, uint32_t left) {
  using S = Shape<KIND, D>;
  const uint32_t lane = threadIdx.x % 32;
  uint32_t found = 0;
  for (uint32_t p = p0; p < p0 + kPart && p < left; ++p) {
    bool odd = false;
    if constexpr (KIND == KQ_CACHE_F16) {
      for (uint32_t u = lane; u < S::kRow / 16; u += 32) {
        const uint4 v = lds_v4(tile.code(p, 16 * u));
        odd |= finite_or_zero(v.x) != v.x || finite_or_zero(v.y) != v.y || finite_or_zero(v.z) != v.z ||
               finite_or_zero(v.w) != v.w;
      }
    } else {
      if (lane < S::kScales) odd = lds_u8(tile.scale(p) + lane) >= 0xf8u;
    }
    if (__any_sync(0xffffffffu, odd)) found |= 1u << (p - p0);
  }
  return found;
}

// What value_product<EDGE> left out of element e of position p: its value where that is not finite.
template <uint32_t KIND, uint32_t D>
__device__ __forceinline__ float special_value(const TileView<Shape<KIND, D>>& tile, uint32_t p, uint32_t e) {
  if constexpr (KIND == KQ_CACHE_F16) {
    const uint32_t v = lds_u16(tile.code(p, 2 * e));
    return (v & 0x7c00u) == 0x7c00u ? h2f(v) : 0.f;
  } else {
    return lds_u8(tile.scale(p) + e / 32) >= 0xf8u ? __int_as_float(0x7fc00000) : 0.f;
  }
}

// Weights are kept times 2^kLift of the reference they were taken to, and outputs are rescaled to a new
// reference only when a logit is more than 2^kSlack above it, which after an item's first tile hardly
// happens: the largest weight is below 2^15, in f16's range, and what f16 loses of a small one (2^-25) is
// 2^-27 of the reference's own weight at most. 16-bit activations leave it at that one f16, 2^-11 of a weight
// at most: a second one would double the products of P V for less than their type's own rounding (4 sequences of
// 64 bf16 drafts: relative error 1.670e-3, of f32 weights 1.657e-3).
constexpr float kLift = 2.f;
constexpr float kSlack = 13.f;

template <uint32_t KIND, uint32_t D, bool SPLIT>
__global__ void __launch_bounds__(kThreads, Narrow<KIND, D>::kCtas) tree_kernel(const __grid_constant__ TreeArgs a) {
  using S = Shape<KIND, D>;
  using M = Narrow<KIND, D>;
  constexpr uint32_t ROWS = 8, NS = M::kSlots;
  extern __shared__ __align__(128) uint8_t smem[];
  float* join = reinterpret_cast<float*>(smem + NS * S::kSlot);  // 4 warps x 8 rows
  float* join_m = join + 4 * 8 * M::kJoinRow;                    // [warp of 4][row], then sums
  float* join_l = join_m + 4 * 8;
  uint4* q_smem = reinterpret_cast<uint4*>(join_l + 4 * 8);
  const uint32_t ring = smem_u32(smem), bars = ring + NS * S::kSlot + M::kJoin + M::kQ;  // full, empty of each slot
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < NS; ++i) {
      mbar_init(bars + 16 * i, 1);
      mbar_init(bars + 16 * i + 8, kReaders);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const Work<ROWS, kTile> work(a);
  const uint64_t total = work.total;
  const uint32_t ctas = static_cast<uint32_t>(min(uint64_t(gridDim.x), total));
  if (blockIdx.x >= ctas) {
    if (threadIdx.x == 0) Split{0, 0, 0, 0, 0}.store(a, blockIdx.x);
    return;
  }
  const uint64_t at = range_start(total, blockIdx.x, ctas);
  const uint32_t count = static_cast<uint32_t>(range_start(total, blockIdx.x + 1, ctas) - at);  // this CTA's tiles
  Place p = locate(a, work, at);
  const uint32_t seg_log2 = min(a.c.page_log2, 7u);
  bool live = true;  // no wait has given up

  if (warp == kReaders) {
    // ---- copies: uses 2 i and 2 i + 1 of the ring for tile i's keys and values, lane k segment k
    const auto page_of = [&]() {
      const uint32_t pos = p.tile * kTile + (lane << seg_log2);
      return lane < kTile >> seg_log2 && pos < p.seq.length()
                 ? static_cast<uint32_t>(a.pages[uint64_t(p.s) * a.max_pages + (pos >> a.c.page_log2)])
                 : 0u;
    };
    uint32_t page = page_of(), sent = 0;  // uses copied
    for (uint32_t i = 0; i < count; ++i) {
      const Place now = p;
      const uint32_t now_page = page;
      if (i + 1 < count) {  // the next tile's pages come in while this one waits for its slots
        if (++p.tile == position_tiles<kTile>(p.seq)) next_item<ROWS>(a, p);
        page = page_of();
      }
#pragma unroll
      for (uint32_t kv = 0; kv < 2; ++kv) {
        const uint32_t use = 2 * i + kv, slot = use % NS, bar = bars + 16 * slot;
        if (use >= NS && live && !mbar_wait(bar + 8, (use / NS - 1) & 1)) {
          report_error(a.err, kErrWaitEmpty);
          live = false;
        }
        live = __all_sync(0xffffffffu, live);
        if (!live) continue;
        copy_segments<S>(a, now, now_page, kv ? a.c.v : a.c.k, ring + slot * S::kSlot, bar);
        sent = use + 1;
      }
    }
    // no copy is in flight when the CTA ends, whatever gave up
    for (uint32_t use = sent > NS ? sent - NS : 0; use < sent; ++use)
      if (!mbar_wait(bars + 16 * (use % NS), (use / NS) & 1)) report_error(a.err, kErrWaitFull);
    return;
  }

  const uint32_t g = lane >> 2, t = lane & 3u;
  const Lane<S> place(g, t);
  uint32_t done = 0;  // tiles of this CTA read
  while (done < count) {
    // ---- the item's rows as operand B (row n = g), scaled (row_scale), and what rows 2 t, 2 t + 1 need
    const uint32_t rows = p.seq.drafts * a.group;
    uint32_t qb[M::kQShared ? 1 : S::kSteps][4];
    float2 unit2;  // logits in log2 units a unit of the scaled product, of rows 2 t and 2 t + 1
    {
      const uint32_t r = p.rows * ROWS + g;
      const bool have = r < rows;
      const uint32_t tok = token_of(a, r);
      const uint64_t row = have ? (p.seq.first + tok) * a.q_token +
                                      uint64_t(p.head * a.group + head_of(a, r, tok)) * a.c.dim
                                : 0;
      float x[S::kSteps][4];
      load_row(a, row, have, [&](uint32_t ks) { return key_element<S>(ks, t); }, x);
      float most = 0.f;
#pragma unroll
      for (uint32_t ks = 0; ks < S::kSteps; ++ks)
        most = fmaxf(most, fmaxf(fmaxf(fabsf(x[ks][0]), fabsf(x[ks][1])), fmaxf(fabsf(x[ks][2]), fabsf(x[ks][3]))));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const RowScale scale = row_scale<SPLIT>(most, a.scale_log2);
      const float up = scale.up, unit = scale.unit;
      unit2.x = __shfl_sync(0xffffffffu, unit, 8 * t);
      unit2.y = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
#pragma unroll
      for (uint32_t ks = 0; ks < S::kSteps; ++ks) {
        const float(&y)[4] = x[ks];
        uint32_t hi0, lo0, hi1, lo1;
        split2(y[0] * up, y[1] * up, hi0, lo0);
        split2(y[2] * up, y[3] * up, hi1, lo1);
        if constexpr (M::kQShared) {
          // every warp writes the same words, and reads its own
          q_smem[ks * 32 + lane] = make_uint4(hi0, hi1, lo0, lo1);
        } else {
          qb[ks][0] = hi0;
          qb[ks][1] = hi1;
          qb[ks][2] = lo0;
          qb[ks][3] = lo1;
        }
      }
      if constexpr (M::kQShared) __syncwarp();
    }
    const auto q_at = [&](uint32_t ks, uint32_t (&b)[4]) {
      if constexpr (M::kQShared) {
        const uint4 w = q_smem[ks * 32 + lane];
        b[0] = w.x;
        b[1] = w.y;
        b[2] = w.z;
        b[3] = w.w;
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) b[i] = qb[ks][i];
      }
    };

    float o[D / 16][4];
#pragma unroll
    for (uint32_t j = 0; j < D / 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    float m[2] = {-INFINITY, -INFINITY};  // rows 2 t, 2 t + 1, the same in all g
    float2 l = make_float2(0.f, 0.f), minus = make_float2(0.f, 0.f);  // sums (this thread's), -(m - kLift)
    float limit = -INFINITY;  // weights' exponents above this want a new reference

    const uint32_t tiles = position_tiles<kTile>(p.seq), first_tile = p.tile;
    const uint32_t here = min(tiles - first_tile, count - done);  // of the item's tiles, this CTA's
    // The parts go round the warps; a warp also passes the tiles it has no part of, so that it sees every
    // phase of every slot in turn (a parity it had skipped would be taken for the one before).
    uint32_t turn = warp;  // (warp - parts so far) mod kReaders: the warp's part of the tile, if below kParts
    for (uint32_t n = 0; n < here; ++n, turn = turn >= kParts ? turn - kParts : turn + kReaders - kParts) {
      const uint32_t it = 2 * (done + n), p0 = turn * kPart;
      const uint32_t base = (first_tile + n) * kTile, left = p.seq.length() - base;  // positions left
      const bool edge = base + kTile > p.seq.prefix;
      const bool reads = turn < kParts && p0 < left;
      const uint32_t k_slot = it % NS, v_slot = (it + 1) % NS;
      if (live && !mbar_wait(bars + 16 * k_slot, (it / NS) & 1)) {
        report_error(a.err, kErrWaitFull);
        live = false;
      }
      __syncwarp();
      uint32_t pb[kSubs][4];
      const auto row_bits = [&](unsigned long long (&bits)[2]) {  // of rows 2 t, 2 t + 1
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          const uint32_t r = p.rows * ROWS + 2 * t + i;
          bits[i] = r < rows ? mask_bits(a, p.seq, token_of(a, r)) : 0ull;
        }
      };
      if (reads) {
        const uint32_t from = ring + k_slot * S::kSlot;
        const PartView<S> keys[kSubs] = {{from, p0, seg_log2}, {from, p0 + 16, seg_log2}};
        float c[kSubs][4];
        key_product<KIND, D, SPLIT>(keys, place, q_at, c);
        // rows 2 t, 2 t + 1 at position pi(g), then at pi(g) + 8: logits in log2 units, to the reference
        float2 z[kSubs][2];
        float most = -INFINITY;
#pragma unroll
        for (uint32_t s = 0; s < kSubs; ++s) {
          z[s][0] = fma2(make_float2(c[s][0], c[s][1]), unit2, minus);
          z[s][1] = fma2(make_float2(c[s][2], c[s][3]), unit2, minus);
        }
        if (edge) {
          unsigned long long bits[2];
          row_bits(bits);
#pragma unroll
          for (uint32_t s = 0; s < kSubs; ++s)
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
              const uint32_t pos = base + p0 + 16 * s + pi8(g) + 8 * h;
              if (!sees(bits[0], pos, p.seq)) z[s][h].x = -INFINITY;
              if (!sees(bits[1], pos, p.seq)) z[s][h].y = -INFINITY;
            }
        }
#pragma unroll
        for (uint32_t s = 0; s < kSubs; ++s)
          most = max3(max3(most, z[s][0].x, z[s][0].y), z[s][1].x, z[s][1].y);
        if (__any_sync(0xffffffffu, most > limit)) {
          // A new reference for the rows that want one (all rows have one after this, but those that see
          // nothing yet, whose weights are zero whatever it is). It is of the logits themselves, each one
          // rounded: the largest is then exactly the reference, however large it is.
          float f[2];
#pragma unroll
          for (uint32_t i = 0; i < 2; ++i) {
            float x[kSubs][2];
            float top = -INFINITY, now = -INFINITY;  // to the old reference, and itself
#pragma unroll
            for (uint32_t s = 0; s < kSubs; ++s)
#pragma unroll
              for (uint32_t h = 0; h < 2; ++h) {
                const float old = i ? z[s][h].y : z[s][h].x;
                x[s][h] = old == -INFINITY ? -INFINITY : __fmul_rn(c[s][2 * h + i], i ? unit2.y : unit2.x);
                top = fmaxf(top, old);
                now = fmaxf(now, x[s][h]);
              }
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
              now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, s));
            }
            const bool fresh = m[i] == -INFINITY;
            if (!fresh && !(top > kSlack + kLift)) now = m[i];
            const float next = now == -INFINITY ? 0.f : kLift - now;
            f[i] = fresh ? 0.f : exp2f(m[i] - now);
            m[i] = now;
            (i ? minus.y : minus.x) = next;
#pragma unroll
            for (uint32_t s = 0; s < kSubs; ++s)
#pragma unroll
              for (uint32_t h = 0; h < 2; ++h) (i ? z[s][h].y : z[s][h].x) = x[s][h] + next;
          }
          l.x *= f[0];
          l.y *= f[1];
#pragma unroll
          for (uint32_t j = 0; j < D / 16; ++j)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) o[j][i] *= f[i & 1];
          limit = __any_sync(0xffffffffu, m[0] == -INFINITY || m[1] == -INFINITY) ? -INFINITY : kSlack + kLift;
        }
#pragma unroll
        for (uint32_t s = 0; s < kSubs; ++s) {
          const float2 w0 = make_float2(exp2_fast(z[s][0].x), exp2_fast(z[s][0].y));
          const float2 w1 = make_float2(exp2_fast(z[s][1].x), exp2_fast(z[s][1].y));
          l = add2(l, add2(w0, w1));
          if constexpr (SPLIT) {
            uint32_t hi0, lo0, hi1, lo1;
            split2(w0.x, w0.y, hi0, lo0);
            split2(w1.x, w1.y, hi1, lo1);
            pb[s][0] = transpose8(hi0);
            pb[s][1] = transpose8(hi1);
            pb[s][2] = transpose8(lo0);
            pb[s][3] = transpose8(lo1);
          } else {
            pb[s][0] = transpose8(h2(__floats2half2_rn(w0.x, w0.y)));
            pb[s][1] = transpose8(h2(__floats2half2_rn(w1.x, w1.y)));
            pb[s][2] = pb[s][3] = 0;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + 16 * k_slot + 8);
      if (live && !mbar_wait(bars + 16 * v_slot, ((it + 1) / NS) & 1)) {
        report_error(a.err, kErrWaitFull);
        live = false;
      }
      __syncwarp();
      if (reads) {
        const uint32_t slot = ring + v_slot * S::kSlot;
        if (edge) {
#pragma unroll
          for (uint32_t s = 0; s < kSubs; ++s)
            value_product<KIND, D, SPLIT, true, false>(PartView<S>(slot, p0 + 16 * s, seg_log2), place, p0 + 16 * s + t,
                                                       left, pb[s], o);
          const TileView<S> values = {slot, seg_log2};
          // infinities and NaN reach the rows that see their position
          for (uint32_t odd = special_positions<KIND, D>(values, p0, left); odd; odd &= odd - 1) {
            const uint32_t pos = p0 + __ffs(odd) - 1;
            unsigned long long bits[2];
            row_bits(bits);
            const bool see0 = sees(bits[0], base + pos, p.seq), see1 = sees(bits[1], base + pos, p.seq);
#pragma unroll
            for (uint32_t j = 0; j < D / 16; ++j)
#pragma unroll
              for (uint32_t h = 0; h < 2; ++h) {
                const float v = special_value<KIND, D>(values, pos, value_element<S>(j, g, h));
                if (see0) o[j][2 * h] += v;
                if (see1) o[j][2 * h + 1] += v;
              }
          }
        } else {
          value_product<KIND, D, SPLIT, false, false>(PartView<S>(slot, p0, seg_log2), place, p0 + t, left, pb[0], o);
          value_product<KIND, D, SPLIT, false, true>(PartView<S>(slot, p0 + 16, seg_log2), place, p0 + 16 + t, left,
                                                     pb[1], o);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + 16 * v_slot + 8);
    }
    done += here;
    const bool whole = here == tiles;
    float* part = a.part + (uint64_t(blockIdx.x) * 2 + (first_tile ? 0 : 1)) * part_floats(ROWS, D);

    // ---- the warps' maxima, sums and outputs joined: warps 4-6 give theirs to 0-2, register for
    // register; 0-3 lay rows out, and warps sum rows
    constexpr uint32_t RAW = D / 16 * 4 + 4;  // floats a lane gives
    static_assert(RAW * 32 <= 8 * M::kJoinRow, "a warp's registers fit its rows");
    float* mine = join + (warp & 3) * 8 * M::kJoinRow;
    if (warp >= 4) {
#pragma unroll
      for (uint32_t j = 0; j < D / 16; ++j)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) mine[(j * 4 + i) * 32 + lane] = o[j][i];
      mine[(RAW - 4) * 32 + lane] = m[0];
      mine[(RAW - 3) * 32 + lane] = m[1];
      mine[(RAW - 2) * 32 + lane] = l.x;
      mine[(RAW - 1) * 32 + lane] = l.y;
    }
    named_barrier(1, kReaders * 32);
    if (warp < 4) {
      if (warp < kReaders - 4) {
        float f[2], h[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          const float other = mine[(RAW - 4 + i) * 32 + lane], now = fmaxf(m[i], other);
          f[i] = m[i] == now ? 1.f : exp2f(m[i] - now);
          h[i] = other == now ? 1.f : exp2f(other - now);
          m[i] = now;
        }
        l.x = fmaf(h[0], mine[(RAW - 2) * 32 + lane], f[0] * l.x);
        l.y = fmaf(h[1], mine[(RAW - 1) * 32 + lane], f[1] * l.y);
#pragma unroll
        for (uint32_t j = 0; j < D / 16; ++j)
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            o[j][i] = fmaf(h[i & 1], mine[(j * 4 + i) * 32 + lane], f[i & 1] * o[j][i]);
      }
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) {
        l.x += __shfl_xor_sync(0xffffffffu, l.x, s);
        l.y += __shfl_xor_sync(0xffffffffu, l.y, s);
      }
      __syncwarp();
#pragma unroll
      for (uint32_t j = 0; j < D / 16; ++j)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          mine[(2 * t + (i & 1)) * M::kJoinRow + value_element<S>(j, g, i >> 1)] = o[j][i];
      if (g == 0) {
        join_m[warp * 8 + 2 * t] = m[0];
        join_m[warp * 8 + 2 * t + 1] = m[1];
        join_l[warp * 8 + 2 * t] = l.x;
        join_l[warp * 8 + 2 * t + 1] = l.y;
      }
    }
    named_barrier(1, kReaders * 32);
    for (uint32_t row = warp; row < 8; row += kReaders) {
      const uint32_t rr = p.rows * ROWS + row;
      if (rr >= rows) break;
      float mx = -INFINITY;
#pragma unroll
      for (uint32_t w = 0; w < 4; ++w) mx = fmaxf(mx, join_m[w * 8 + row]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      float f[4], den = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < 4; ++w) {
        f[w] = exp2f(join_m[w * 8 + row] - ref);
        den = fmaf(f[w], join_l[w * 8 + row], den);
      }
      const float inv = whole ? (den == 0.f ? 0.f : 1.f / den) : 1.f;
      const uint32_t tok = token_of(a, rr);
      const uint64_t to = (p.seq.first + tok) * a.out_token +
                          uint64_t(p.head * a.group + head_of(a, rr, tok)) * a.c.dim;
#pragma unroll
      for (uint32_t e = lane; e < D; e += 32) {
        float v = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) v = fmaf(f[w], join[(w * 8 + row) * M::kJoinRow + e], v);
        if (!whole) part[row * D + e] = v;
        else if (e < a.c.dim) store_one(a.out, to + e, v * inv, a.type);
      }
      if (!whole && lane == 0) {
        part[ROWS * D + row] = mx;
        part[ROWS * (D + 1) + row] = den;
      }
    }
    if (done == count && threadIdx.x == 0)
      leave_split(a, p, first_tile == 0, whole, total, at + count, here, tiles, ctas);
    if (done < count) {
      next_item<ROWS>(a, p);
      named_barrier(1, kReaders * 32);  // read, before the next item's are written
    }
  }
}

// ---------------------------------------------------------------- the join of split items

// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over the parts of each item that more than one CTA
// did, in an order that the lengths alone decide, with a running maximum M. Grid: (the CTAs that may have
// left parts, shares of the rows): an item is joined by the blocks of the CTA that began it (each began at
// most one that others went on with), which say so in the workspace. CB parts at a time, so that their
// loads share L2's latency, and a warp a row; where items have many parts (SHARED) a block a row, its
// warps the parts in turn, for then there are few rows: 8 items of 37 parts each 66.7 -> 64.0 us with
// their attention, but 256 of 2 or 3 74.0 -> 78.1.
//
// Finding the parts again from the lengths, as the main kernel does, cost each block some 2 us (4 sequences
// of 64 drafts 132 us against 125), and they cannot do it early: they do not fit an SM beside the main
// kernel's CTAs. Joining in the main kernel, by the
// CTA that leaves an item's last part, was slower (one token over 131001 positions 94 us against 92, 25
// drafts 56 against 49): that CTA joins alone, after the fences.
template <uint32_t ROWS, uint32_t D, bool SHARED>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ TreeArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t c0 = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Split split = Split::load(a, c0);
  const uint32_t row = SHARED ? blockIdx.y : blockIdx.y * 8 + warp, rr = split.rows * ROWS + row;
  if (split.last == 0 || rr >= split.drafts * a.group) return;
  constexpr uint64_t stride = part_floats(ROWS, D);
  constexpr uint32_t V = D / 32, CB = 8, STEP = SHARED ? 8 : 1;
  float top = -INFINITY, den = 0.f, v[V] = {};
#pragma unroll 1
  for (uint32_t c = c0 + (SHARED ? warp : 0); c <= split.last; c += CB * STEP) {
    float m[CB], l[CB], x[CB][V];
#pragma unroll
    for (uint32_t j = 0; j < CB; ++j) {
      const bool there = c + j * STEP <= split.last;
      // slot 1 of the CTA that began the item, slot 0 of those that went on
      const float* part = a.part + (uint64_t(c + j * STEP) * 2 + (c + j * STEP == c0 ? 1 : 0)) * stride;
      m[j] = there ? part[ROWS * D + row] : -INFINITY;
      l[j] = there ? part[ROWS * (D + 1) + row] : 0.f;
#pragma unroll
      for (uint32_t i = 0; i < V; i += 2) {
        const float2 y = there ? *reinterpret_cast<const float2*>(part + row * D + lane * V + i) : make_float2(0.f, 0.f);
        x[j][i] = y.x;
        x[j][i + 1] = y.y;
      }
    }
    float mx = top;
#pragma unroll
    for (uint32_t j = 0; j < CB; ++j) mx = fmaxf(mx, m[j]);
    const float ref = mx == -INFINITY ? 0.f : mx, keep = exp2f(top - ref);
    top = mx;
    den *= keep;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) v[i] *= keep;
#pragma unroll
    for (uint32_t j = 0; j < CB; ++j) {
      const float f = exp2f(m[j] - ref);
      den = fmaf(f, l[j], den);
#pragma unroll
      for (uint32_t i = 0; i < V; ++i) v[i] = fmaf(f, x[j][i], v[i]);
    }
  }
  const uint32_t tok = token_of(a, rr);
  const uint64_t to = (split.first + tok) * a.out_token + uint64_t(split.head * a.group + head_of(a, rr, tok)) * a.c.dim;
  if constexpr (!SHARED) {
    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i)
      if (lane * V + i < a.c.dim) store_one(a.out, to + lane * V + i, v[i] * inv, a.type);
  } else {
    __shared__ float tops[8], dens[8], outs[8][D];
    if (lane == 0) {
      tops[warp] = top;
      dens[warp] = den;
    }
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) outs[warp][lane * V + i] = v[i];
    __syncthreads();
    const uint32_t e = threadIdx.x;
    if (e >= a.c.dim) return;
    float mx = -INFINITY;
#pragma unroll
    for (uint32_t w = 0; w < 8; ++w) mx = fmaxf(mx, tops[w]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float y = 0.f, all = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < 8; ++w) {
      const float f = exp2f(tops[w] - ref);
      all = fmaf(f, dens[w], all);
      y = fmaf(f, outs[w][e], y);
    }
    store_one(a.out, to + e, all == 0.f ? 0.f : y / all, a.type);
  }
}

// CTAs of the warp-MMA kernel a SM holds.
inline uint32_t narrow_ctas(uint32_t kind, uint32_t pitch) {
  const auto of = [&](auto kind_tag) {
    constexpr uint32_t K = decltype(kind_tag)::value;
    return pitch == 64 ? Narrow<K, 64>::kCtas : pitch == 128 ? Narrow<K, 128>::kCtas : Narrow<K, 256>::kCtas;
  };
  return kind == KQ_CACHE_F16  ? of(std::integral_constant<uint32_t, KQ_CACHE_F16>())
         : kind == KQ_CACHE_Q8 ? of(std::integral_constant<uint32_t, KQ_CACHE_Q8>())
                               : of(std::integral_constant<uint32_t, KQ_CACHE_Q4>());
}

// Prepares, and launches, the kernels of one kind of cache.
template <uint32_t KIND>
cudaError_t prepare_kind();
template <uint32_t KIND>
cudaError_t launch_kind(const TreeArgs& a, bool split, bool wide, uint32_t ctas, cudaStream_t s);

template <uint32_t KIND, uint32_t D, bool SPLIT>
cudaError_t prepare_one() {
  return cudaFuncSetAttribute(tree_kernel<KIND, D, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Narrow<KIND, D>::kBytes);
}

template <uint32_t KIND, uint32_t D, bool SPLIT>
cudaError_t launch_one(const TreeArgs& a, uint32_t ctas, cudaStream_t s) {
  return launch_pdl(tree_kernel<KIND, D, SPLIT>, dim3(ctas), kThreads, Narrow<KIND, D>::kBytes, s, a);
}

}  // namespace tree
}  // namespace kq
