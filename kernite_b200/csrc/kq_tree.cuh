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
// which CTAs hold an item's parts. So a long context is split over the whole GPU, and a ragged batch
// leaves no CTA idle.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kq_cache.cuh"
#include "kq_device.cuh"

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
  float scale_log2;
  uint32_t n_seq, n_heads, group, tokens, max_drafts, max_pages;
  uint32_t type;
  unsigned* err;
};

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

// The tiles of sequences [0, n). Called by whole warps.
template <uint32_t ROWS, uint32_t TW>
__device__ __forceinline__ uint64_t work_before(const TreeArgs& a, uint32_t n) {
  uint64_t w = 0;
  for (uint32_t s = threadIdx.x % 32; s < n; s += 32) w += seq_work<ROWS, TW>(a, load_seq(a, s));
  return warp_sum(w);
}

// Where a CTA is: an item and the next of its tiles.
struct Place {
  Seq seq;
  uint32_t s, head, rows;  // sequence, key/value head, row tile
  uint32_t tile;
};

// The place of tile `at` of the whole work. Called by whole warps, at < total.
template <uint32_t ROWS, uint32_t TW>
__device__ __forceinline__ Place locate(const TreeArgs& a, uint64_t at) {
  const uint32_t lane = threadIdx.x % 32;
  Place p = {};
  for (uint32_t s0 = 0; s0 < a.n_seq; s0 += 32) {
    const uint64_t w = s0 + lane < a.n_seq ? seq_work<ROWS, TW>(a, load_seq(a, s0 + lane)) : 0;
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
      const uint64_t rest = at - __shfl_sync(0xffffffffu, upto - w, who);
      p.seq = load_seq(a, p.s);
      const uint32_t pt = position_tiles<TW>(p.seq), rt = row_tiles<ROWS>(a, p.seq);
      p.tile = static_cast<uint32_t>(rest % pt);
      const uint64_t item = rest / pt;
      p.rows = static_cast<uint32_t>(item % rt);
      p.head = static_cast<uint32_t>(item / rt);
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

// CTA c of n <= total takes tiles [range_start(c), range_start(c + 1)) of `total`, at least one.
__device__ __forceinline__ uint64_t range_start(uint64_t total, uint32_t c, uint32_t n) {
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

__device__ __forceinline__ float load_one(const void* p, uint64_t i, uint32_t type) {
  return type == KQ_TYPE_F32 ? static_cast<const float*>(p)[i]
         : type == KQ_TYPE_F16 ? __half2float(static_cast<const __half*>(p)[i])
                               : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_one(void* p, uint64_t i, float v, uint32_t type) {
  if (type == KQ_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == KQ_TYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------- the warp-MMA kernel
//
// mma.sync.m16n8k16 (f16 in, f32 accumulated), all from registers: S = Q K^T with the rows as M, then
// O += P V with the accumulators of S as the next A operand. A warp takes 16 of a tile's positions and
// all of an item's rows; the eight warps keep separate maxima, sums and outputs and join them at an
// item's end. For f32 activations the 16 rows of the MMA are 8 rows twice: the f16 rounding of the
// operand and the f16 rounding of what that left, so one MMA gives about 22 bits, and sums of the two
// halves lie in one thread.
//
// Codes become f16 in registers (exactly: c * scale has at most 11 bits). The order of a contraction
// is free, so a thread's B fragment of K is four consecutive elements of a row it reads 16 bytes at a
// time, and the columns of V's fragments are consecutive elements too; position n of an n-tile is
// pi(n) = 4 (n mod 2) + n / 2, so that with the cache's unit permutation the reads of a warp meet no
// bank twice.

constexpr uint32_t kWarps = 8;                    // consumers
constexpr uint32_t kThreads = kWarps * 32 + 32;   // and the producer's warp

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// 2^x, to 2^-22 of it; results below f32's normal range are zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// How a head of pitch D lies in rows of codes, per kind: BYTES of a row, EK elements of a thread's
// piece of a key row, EV of its piece of a value row.
template <uint32_t KIND, uint32_t D>
struct Shape {
  static constexpr uint32_t kBits = KIND == KQ_CACHE_F16 ? 16 : KIND == KQ_CACHE_Q8 ? 8 : 4;
  static constexpr uint32_t kRow = D * kBits / 8;
  static constexpr uint32_t kScales = KIND == KQ_CACHE_F16 ? 0 : D / 32;
  static constexpr uint32_t kMost = 128 / kBits;  // elements of 16 bytes
  static constexpr uint32_t EK = kMost < D / 4 ? kMost : D / 4;
  static constexpr uint32_t EV = kMost < D / 8 ? kMost : D / 8;
  static constexpr uint32_t kSteps = D / 16;      // MMAs along a head
  static constexpr uint32_t kCols = D / 8;        // n-tiles of the output
  static constexpr bool kPermuted = EV * kBits == 128;  // value pieces of 16 bytes go in the order pi
  static constexpr uint32_t kSlot = kTile * (kRow + kScales);
};

__device__ __forceinline__ uint32_t pi8(uint32_t n) { return ((n & 1u) << 2) | (n >> 1); }

// First element of step ks of thread t's key pieces.
template <class S>
__device__ __forceinline__ constexpr uint32_t key_element(uint32_t ks, uint32_t t) {
  return S::EK * (t + 4 * (ks / (S::EK / 4))) + 4 * (ks % (S::EK / 4));
}

// Element of column n (0..7) of output n-tile j.
template <class S>
__device__ __forceinline__ constexpr uint32_t value_element(uint32_t j, uint32_t n) {
  return S::EV * (8 * (j / S::EV) + (S::kPermuted ? ((n & 1u) << 2 | n >> 1) : n)) + j % S::EV;
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

// Shared memory of the warp-MMA kernel: the ring of key and value tiles, the join of the warps.
template <uint32_t KIND, uint32_t D>
struct Smem {
  using S = Shape<KIND, D>;
  static constexpr uint32_t kJoinRow = D + 4;
  static constexpr uint32_t kJoin = kWarps * 8 * kJoinRow * 4 + 2 * kWarps * 16 * 4;
  static constexpr uint32_t kQ = D == 256 ? S::kSteps * 32 * 16 : 0;  // operand A where registers are short
  static constexpr uint32_t kBars = 16 * 16;
  static constexpr uint32_t kFixed = kJoin + kQ + kBars;
  static constexpr uint32_t kFit = (224 * 1024 - kFixed) / S::kSlot;
  static constexpr uint32_t kSlots = kFit > 12 ? 12 : kFit / 2 * 2;  // keys and values in turn
  static constexpr uint32_t kBytes = kFixed + kSlots * S::kSlot + 128;
  static_assert(kSlots >= 2, "a key tile and a value tile must fit");
};

// The producer's copies of one tile of keys (or values): whole records where a page is at most a tile,
// else its rows and its scales. Pages' numbers sit in the warp's lanes, 32 consecutive ones at a time.
struct PageWindow {
  uint32_t s, base;
  uint32_t id;
};

template <class S, uint32_t TW>
__device__ __forceinline__ void produce_tile(const TreeArgs& a, const Place& p, const uint8_t* src, uint32_t dst,
                                             uint32_t bar, PageWindow& w) {
  const uint32_t lane = threadIdx.x % 32;
  const uint32_t seg_log2 = min(a.c.page_log2, TW == 128 ? 7u : 6u), seg = 1u << seg_log2;
  const uint32_t base = p.tile * TW;
  const uint32_t n = (min(TW, p.seq.length() - base) + seg - 1) >> seg_log2;
  const uint32_t first = base >> a.c.page_log2;
  const uint32_t pages = ((n << seg_log2) + (1u << a.c.page_log2) - 1) >> a.c.page_log2;
  if (w.s != p.s || first < w.base || first + pages > w.base + 32) {
    w.s = p.s;
    w.base = first;
    const uint32_t used = (p.seq.length() + a.c.page() - 1) >> a.c.page_log2;
    w.id = 0;
    if (first + lane < used) {
      w.id = static_cast<uint32_t>(a.pages[uint64_t(p.s) * a.max_pages + first + lane]);
      if (w.id >= a.c.n_pages) {
        report_error(a.err, kErrCacheRange);
        w.id = 0;
      }
    }
  }
  constexpr uint32_t row = S::kRow + S::kScales;
  if (lane == 0) mbar_arrive_expect_tx(bar, n * seg * row);
  __syncwarp();
  const uint32_t mine = __shfl_sync(0xffffffffu, w.id, ((base + lane * seg) >> a.c.page_log2) - w.base);
  if (lane < n) {
    const uint8_t* rec = src + a.c.at(mine, p.head);
    if (a.c.page_log2 == seg_log2) {
      bulk_g2s(dst + lane * seg * row, rec, seg * row, bar);
    } else {
      const uint32_t at = base & (a.c.page() - 1);
      bulk_g2s(dst, rec + at * S::kRow, seg * S::kRow, bar);
      if constexpr (S::kScales != 0)
        bulk_g2s(dst + seg * S::kRow, rec + a.c.page() * S::kRow + at * S::kScales, seg * S::kScales, bar);
    }
  }
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

// The K operand of n-tile j (positions 16 warp + 8 j + pi(n)): b0, b1 of every step.
template <uint32_t KIND, uint32_t D>
__device__ __forceinline__ void key_fragments(const TileView<Shape<KIND, D>>& tile, uint32_t p, uint32_t t,
                                              uint32_t (&b)[D / 16][2]) {
  using S = Shape<KIND, D>;
  constexpr uint32_t B = S::EK * S::kBits / 8;
#pragma unroll
  for (uint32_t j = 0; j < D / 4 / S::EK; ++j) {
    uint32_t w[B / 4];
    lds_words<B>(tile.code(p, B * (t + 4 * j)), w);
    if constexpr (KIND == KQ_CACHE_F16) {
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        b[2 * j + k][0] = w[2 * k];
        b[2 * j + k][1] = w[2 * k + 1];
      }
    } else {
      const uint32_t byte = lds_u8(tile.scale(p) + S::EK * (t + 4 * j) / 32);
      const Scale2 s2 = scale2<KIND>(byte, byte);
#pragma unroll
      for (uint32_t k = 0; k < S::EK / 4; ++k) {
        uint32_t lo, hi;
        if constexpr (KIND == KQ_CACHE_Q8) {
          lo = decode2(prmt(w[k], kMagic, 0x4140), s2);
          hi = decode2(prmt(w[k], kMagic, 0x4342), s2);
        } else {
          lo = decode2(nibbles(nibble_up(w[k / 2], 2 * (k % 2))), s2);
          hi = decode2(nibbles(nibble_up(w[k / 2], 2 * (k % 2) + 1)), s2);
        }
        b[j * (S::EK / 4) + k][0] = lo;
        b[j * (S::EK / 4) + k][1] = hi;
      }
    }
  }
}

// f16 pairs whose exponent is all ones (infinity, NaN) become zero.
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t v) {
  if ((v & 0x7c00u) == 0x7c00u) v &= 0xffff0000u;
  if ((v & 0x7c000000u) == 0x7c000000u) v &= 0x0000ffffu;
  return v;
}

// O += P V for the warp's 16 positions. a: P as operand A. EDGE: the tile reaches past the prefix, so
// rows past the end and values that are not finite count as zero here (P is zero where a position is
// masked, and zero times those would not be); add_special adds the latter where they are seen.
template <uint32_t KIND, uint32_t D, bool EDGE>
__device__ __forceinline__ void value_product(const TileView<Shape<KIND, D>>& tile, uint32_t p0, uint32_t g,
                                              uint32_t t, uint32_t left, const uint32_t (&a)[4],
                                              float (&o)[D / 8][4]) {
  using S = Shape<KIND, D>;
  constexpr uint32_t B = S::EV * S::kBits / 8;
  const uint32_t pg = S::kPermuted ? pi8(g) : g;
  const uint32_t p[4] = {p0 + t, p0 + 4 + t, p0 + 8 + t, p0 + 12 + t};
#pragma unroll
  for (uint32_t jj = 0; jj < D / 8 / S::EV; ++jj) {
    uint32_t w[4][B / 4];
    uint32_t byte[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lds_words<B>(tile.code(p[i], B * (pg + 8 * jj)), w[i]);
      if constexpr (KIND == KQ_CACHE_F16) {
        if constexpr (EDGE) {
#pragma unroll
          for (uint32_t k = 0; k < B / 4; ++k) w[i][k] = p[i] < left ? finite_or_zero(w[i][k]) : 0u;
        }
      } else {
        byte[i] = lds_u8(tile.scale(p[i]) + S::EV * (pg + 8 * jj) / 32);
        if constexpr (EDGE) byte[i] = p[i] < left && byte[i] < 0xf8u ? byte[i] : 0u;
      }
    }
    const Scale2 s2[2] = {scale2<KIND>(byte[0], byte[1]), scale2<KIND>(byte[2], byte[3])};
#pragma unroll
    for (uint32_t k = 0; k < B / 4; ++k) {
      // operand pairs (position p[0], p[1]) and (p[2], p[3]) of each element of word k
      if constexpr (KIND == KQ_CACHE_F16) {
        mma16816(o[jj * S::EV + 2 * k], a, prmt(w[0][k], w[1][k], 0x5410), prmt(w[2][k], w[3][k], 0x5410));
        mma16816(o[jj * S::EV + 2 * k + 1], a, prmt(w[0][k], w[1][k], 0x7632), prmt(w[2][k], w[3][k], 0x7632));
      } else if constexpr (KIND == KQ_CACHE_Q8) {
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
          const uint32_t x = prmt(w[0][k], w[1][k], half ? 0x7362 : 0x5140);
          const uint32_t y = prmt(w[2][k], w[3][k], half ? 0x7362 : 0x5140);
          mma16816(o[jj * S::EV + 4 * k + 2 * half], a, decode2(prmt(x, kMagic, 0x4140), s2[0]),
                   decode2(prmt(y, kMagic, 0x4140), s2[1]));
          mma16816(o[jj * S::EV + 4 * k + 2 * half + 1], a, decode2(prmt(x, kMagic, 0x4342), s2[0]),
                   decode2(prmt(y, kMagic, 0x4342), s2[1]));
        }
      } else {
#pragma unroll
        for (uint32_t odd = 0; odd < 2; ++odd) {
          const uint32_t x = prmt(w[0][k], w[1][k], odd ? 0x7632 : 0x5410);
          const uint32_t y = prmt(w[2][k], w[3][k], odd ? 0x7632 : 0x5410);
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e)
            mma16816(o[jj * S::EV + 8 * k + 2 * e + odd], a, decode2(nibbles(nibble_up(x, e)), s2[0]),
                     decode2(nibbles(nibble_up(y, e)), s2[1]));
        }
      }
    }
  }
}

// The values value_product<EDGE> left out, of the warp's positions below `left`: infinities and NaN
// reach the rows that see their position (bits: the mask words of rows g and g + 8; in split form
// both are row g's and the sums of the two halves are what counts).
template <uint32_t KIND, uint32_t D, bool SPLIT>
__device__ __forceinline__ void add_special(const TileView<Shape<KIND, D>>& tile, uint32_t p0, uint32_t base,
                                            uint32_t left, const Seq& seq, const unsigned long long (&bits)[2],
                                            float (&o)[D / 8][4]) {
  using S = Shape<KIND, D>;
  const uint32_t lane = threadIdx.x % 32, t = lane & 3u;
  for (uint32_t p = p0; p < p0 + 16 && p < left; ++p) {
    bool odd = false;
    if constexpr (KIND == KQ_CACHE_F16) {
      for (uint32_t u = lane; u < S::kRow / 16; u += 32) {
        const uint4 v = lds_v4(tile.code(p, 16 * u));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) odd |= finite_or_zero(w[i]) != w[i];
      }
    } else {
      if (lane < S::kScales) odd = lds_u8(tile.scale(p) + lane) >= 0xf8u;
    }
    if (!__any_sync(0xffffffffu, odd)) continue;
#pragma unroll
    for (uint32_t j = 0; j < D / 8; ++j)
#pragma unroll
      for (uint32_t c = 0; c < 2; ++c) {
        const uint32_t e = value_element<S>(j, 2 * t + c);
        float add = 0.f;
        if constexpr (KIND == KQ_CACHE_F16) {
          const uint32_t v = lds_u16(tile.code(p, 2 * e));
          if ((v & 0x7c00u) == 0x7c00u) add = h2f(v);
        } else {
          if (lds_u8(tile.scale(p) + e / 32) >= 0xf8u) add = __int_as_float(0x7fc00000);
        }
        if (sees(bits[0], base + p, seq)) o[j][c] += add;
        if constexpr (!SPLIT) {
          if (sees(bits[1], base + p, seq)) o[j][2 + c] += add;
        }
      }
  }
}

// Weights are kept times 2^kLift of the reference they were taken to, and outputs are rescaled to a new
// reference only when the maximum is more than 2^kSlack above it, which after an item's first tile hardly
// happens: the largest weight is below 2^15, in f16's range, and what f16 loses of a small one (2^-25) is
// 2^-27 of the reference's own weight at most.
constexpr float kLift = 2.f;
constexpr float kSlack = 13.f;

template <uint32_t KIND, uint32_t D, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) tree_kernel(const __grid_constant__ TreeArgs a) {
  using S = Shape<KIND, D>;
  using M = Smem<KIND, D>;
  constexpr uint32_t ROWS = SPLIT ? 8 : 16;
  constexpr uint32_t NS = M::kSlots;
  extern __shared__ __align__(128) uint8_t smem[];
  float* join = reinterpret_cast<float*>(smem + NS * S::kSlot);
  float* join_m = join + kWarps * 8 * M::kJoinRow;  // [warp][16]
  float* join_l = join_m + kWarps * 16;
  uint4* q_smem = reinterpret_cast<uint4*>(join_l + kWarps * 16);
  const uint32_t bars = smem_u32(smem) + NS * S::kSlot + M::kJoin + M::kQ;  // full, empty of each slot
  const uint32_t ring = smem_u32(smem);
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < NS; ++i) {
      mbar_init(bars + 16 * i, 1);
      mbar_init(bars + 16 * i + 8, kWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  const uint64_t total = work_before<ROWS, kTile>(a, a.n_seq);
  const uint32_t ctas = static_cast<uint32_t>(min(uint64_t(gridDim.x), total));
  if (blockIdx.x >= ctas) return;
  uint64_t at = range_start(total, blockIdx.x, ctas);
  const uint64_t end = range_start(total, blockIdx.x + 1, ctas);
  Place p = locate<ROWS, kTile>(a, at);
  uint32_t it = 0;    // slots used so far: tiles of keys and of values in turn
  bool live = true;   // no wait has given up

  if (warp == kWarps) {
    PageWindow window = {0xffffffffu, 0, 0};
    while (at < end) {
      const uint32_t tiles = position_tiles<kTile>(p.seq);
      for (; p.tile < tiles && at < end; ++p.tile, ++at) {
#pragma unroll 1
        for (uint32_t kv = 0; kv < 2; ++kv, ++it) {
          const uint32_t slot = it % NS;
          if (it >= NS && live && !mbar_wait(bars + 16 * slot + 8, (it / NS - 1) & 1)) {
            report_error(a.err, kErrWaitEmpty);
            live = false;
          }
          live = __all_sync(0xffffffffu, live);
          if (live) produce_tile<S, kTile>(a, p, kv ? a.c.v : a.c.k, ring + slot * S::kSlot, bars + 16 * slot, window);
        }
      }
      if (at < end) next_item<ROWS>(a, p);
    }
    return;
  }

  const uint32_t g = lane >> 2, t = lane & 3u;
  const uint32_t seg_log2 = min(a.c.page_log2, 7u);
  while (at < end) {
    // ---- the item's rows as operand A, each row scaled by a power of two to a largest element in
    // [2^7, 2^8), so that f16's range fits any q
    const uint32_t rows = p.seq.drafts * a.group;
    uint32_t r[2], tok[2];
    unsigned long long bits[2];
    float unit[2];  // logits in log2 units a unit of the scaled product
    uint32_t qa[D == 256 ? 1 : S::kSteps][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      r[half] = p.rows * ROWS + g + (SPLIT ? 0 : 8 * half);
      const bool have = r[half] < rows;
      tok[half] = have ? r[half] / a.group : 0;
      bits[half] = have ? mask_bits(a, p.seq, tok[half]) : 0ull;
      if (SPLIT && half == 1) {
        unit[1] = unit[0];
        continue;
      }
      const uint64_t row = (p.seq.first + tok[half]) * a.q_token +
                           uint64_t(p.head * a.group + r[half] % a.group) * a.c.dim;
      float most = 0.f;
#pragma unroll
      for (uint32_t ks = 0; ks < S::kSteps; ++ks)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const uint32_t e = key_element<S>(ks, t) + i;
          if (have && e < a.c.dim) most = fmaxf(most, fabsf(load_one(a.q, row + e, a.type)));
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^(7 - floor(log2(most))), kept inside f32's normal range; 1 for a row of zeros (or infinities)
      const int ex = static_cast<int>(__float_as_uint(most) >> 23) - 127;
      const int sh = most > 0.f && ex < 128 ? min(max(7 - ex, -120), 120) : 0;
      const float up = __int_as_float((127 + sh) << 23);
      unit[half] = __int_as_float((127 - sh) << 23) * a.scale_log2;
#pragma unroll
      for (uint32_t ks = 0; ks < S::kSteps; ++ks) {
        float x[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const uint32_t e = key_element<S>(ks, t) + i;
          x[i] = have && e < a.c.dim ? load_one(a.q, row + e, a.type) * up : 0.f;
        }
        uint32_t hi0, lo0, hi1, lo1;
        split2(x[0], x[1], hi0, lo0);
        split2(x[2], x[3], hi1, lo1);
        if constexpr (D == 256) {
          // every warp writes the same words; the barrier below orders them before the reads
          uint32_t* to = reinterpret_cast<uint32_t*>(q_smem + ks * 32 + lane);
          if constexpr (SPLIT) {
            to[0] = hi0;
            to[1] = lo0;
            to[2] = hi1;
            to[3] = lo1;
          } else {
            to[half] = hi0;
            to[2 + half] = hi1;
          }
        } else if constexpr (SPLIT) {
          qa[ks][0] = hi0;
          qa[ks][1] = lo0;
          qa[ks][2] = hi1;
          qa[ks][3] = lo1;
        } else {
          qa[ks][half] = hi0;
          qa[ks][2 + half] = hi1;
        }
      }
    }
    if constexpr (D == 256) __syncwarp();

    float o[D / 8][4];
#pragma unroll
    for (uint32_t j = 0; j < D / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    const uint32_t tiles = position_tiles<kTile>(p.seq), first_tile = p.tile;
    for (; p.tile < tiles && at < end; ++p.tile, ++at, it += 2) {
      const uint32_t base = p.tile * kTile, left = p.seq.length() - base;  // positions left in the cache
      const uint32_t p0 = warp * 16;
      const bool edge = base + kTile > p.seq.prefix;
      const uint32_t ks_slot = it % NS, v_slot = (it + 1) % NS;
      if (live && !mbar_wait(bars + 16 * ks_slot, (it / NS) & 1)) {
        report_error(a.err, kErrWaitFull);
        live = false;
      }
      live = __all_sync(0xffffffffu, live);
      uint32_t pa[4];
      if (p0 < left) {
        const TileView<S> keys = {ring + ks_slot * S::kSlot, seg_log2};
        float c[2][4];
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
          uint32_t b[S::kSteps][2];
          key_fragments<KIND, D>(keys, p0 + 8 * j + pi8(g), t, b);
#pragma unroll
          for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
#pragma unroll
          for (uint32_t ks = 0; ks < S::kSteps; ++ks) {
            if constexpr (D == 256) {
              const uint4 w = q_smem[ks * 32 + lane];
              const uint32_t qw[4] = {w.x, w.y, w.z, w.w};
              mma16816(c[j], qw, b[ks][0], b[ks][1]);
            } else {
              mma16816(c[j], qa[ks], b[ks][0], b[ks][1]);
            }
          }
        }
        if constexpr (SPLIT) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            c[j][0] += c[j][2];
            c[j][1] += c[j][3];
          }
        }
        // ---- logits in log2 units, masked; the running maximum; the weights
        constexpr int HALVES = SPLIT ? 1 : 2;
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float& v = c[j][2 * half + i];
              v *= unit[half];
              if (edge && !sees(bits[half], base + p0 + 8 * j + 4 * i + t, p.seq)) v = -INFINITY;
              mx = fmaxf(mx, v);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const bool grow = mx > m[half] + kSlack || (m[half] == -INFINITY && mx > m[half]);
          if (__any_sync(0xffffffffu, grow)) {
            const float to = grow ? mx : m[half];
            const float f = grow ? exp2f(m[half] - to) : 1.f;
            m[half] = to;
            l[half] *= f;
#pragma unroll
            for (uint32_t j = 0; j < D / 8; ++j) {
              o[j][2 * half] *= f;
              o[j][2 * half + 1] *= f;
              if constexpr (SPLIT) {
                o[j][2] *= f;
                o[j][3] *= f;
              }
            }
          }
          const float ref = m[half] == -INFINITY ? 0.f : m[half] - kLift;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float w0 = exp2_fast(c[j][2 * half] - ref), w1 = exp2_fast(c[j][2 * half + 1] - ref);
            if constexpr (SPLIT) {
              split2(w0, w1, pa[2 * j], pa[2 * j + 1]);
              l[0] += w0 + w1;
            } else {
              const __half2 h = __floats2half2_rn(w0, w1);
              pa[2 * j + half] = h2(h);
              // the sum of what multiplies the values: rounding the weights then leaves their mean
              // weight exact
              const float2 f = __half22float2(h);
              l[half] += f.x + f.y;
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + 16 * ks_slot + 8);
      if (live && !mbar_wait(bars + 16 * v_slot, ((it + 1) / NS) & 1)) {
        report_error(a.err, kErrWaitFull);
        live = false;
      }
      live = __all_sync(0xffffffffu, live);
      if (p0 < left) {
        const TileView<S> values = {ring + v_slot * S::kSlot, seg_log2};
        if (edge) {
          value_product<KIND, D, true>(values, p0, g, t, left, pa, o);
          add_special<KIND, D, SPLIT>(values, p0, base, left, p.seq, bits, o);
        } else {
          value_product<KIND, D, false>(values, p0, g, t, left, pa, o);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + 16 * v_slot + 8);
    }
    const bool whole = first_tile == 0 && p.tile == tiles;
    float* part = a.part + (uint64_t(blockIdx.x) * 2 + (first_tile ? 0 : 1)) * part_floats(ROWS, D);

    // ---- the warps' maxima, sums and outputs joined, eight rows at a time
#pragma unroll
    for (int half = 0; half < (SPLIT ? 1 : 2); ++half) {
      float sum = l[half];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) {
        join_m[warp * 16 + g] = m[half];
        join_l[warp * 16 + g] = sum;
      }
#pragma unroll
      for (uint32_t j = 0; j < D / 8; ++j)
#pragma unroll
        for (uint32_t c = 0; c < 2; ++c)
          join[(warp * 8 + g) * M::kJoinRow + value_element<S>(j, 2 * t + c)] =
              SPLIT ? o[j][c] + o[j][2 + c] : o[j][2 * half + c];
      named_barrier(1, kWarps * 32);
      const uint32_t row = warp;  // a warp a row now
      float mx = -INFINITY;
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) mx = fmaxf(mx, join_m[w * 16 + row]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      float f[kWarps], den = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) {
        f[w] = exp2f(join_m[w * 16 + row] - ref);
        den = fmaf(f[w], join_l[w * 16 + row], den);
      }
      const uint32_t rr = p.rows * ROWS + 8 * half + row;
      if (rr < rows) {
        const float inv = whole ? (den == 0.f ? 0.f : 1.f / den) : 1.f;
        const uint64_t to = (p.seq.first + rr / a.group) * a.out_token +
                            uint64_t(p.head * a.group + rr % a.group) * a.c.dim;
        for (uint32_t e = lane; e < D; e += 32) {
          float v = 0.f;
#pragma unroll
          for (uint32_t w = 0; w < kWarps; ++w) v = fmaf(f[w], join[(w * 8 + row) * M::kJoinRow + e], v);
          if (!whole) part[(8 * half + row) * D + e] = v;
          else if (e < a.c.dim) store_one(a.out, to + e, v * inv, a.type);
        }
        if (!whole && lane == 0) {
          part[ROWS * D + 8 * half + row] = mx;
          part[ROWS * (D + 1) + 8 * half + row] = den;
        }
      }
      named_barrier(1, kWarps * 32);  // read, before the next item's (or half's) are written
    }
    if (at < end) next_item<ROWS>(a, p);
  }
}

// ---------------------------------------------------------------- the join of split items

// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over an item's parts, in their order. Grid: (items
// of a largest tree a sequence and head, eight rows each); items that one CTA did whole are done.
template <uint32_t ROWS, uint32_t D, uint32_t TW>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ TreeArgs a, uint32_t grid) {
  const uint32_t max_rt = (a.max_drafts * a.group + ROWS - 1) / ROWS;
  const uint32_t rt = blockIdx.x % max_rt, head = blockIdx.x / max_rt % a.c.n_kv;
  const uint32_t s = blockIdx.x / max_rt / a.c.n_kv;
  const Seq seq = load_seq(a, s);
  const uint32_t rts = row_tiles<ROWS>(a, seq), tiles = position_tiles<TW>(seq);
  const uint32_t row = blockIdx.y * 8 + threadIdx.x / 32, rr = rt * ROWS + row;
  if (rr >= seq.drafts * a.group) return;
  uint64_t before = 0, total = 0;
  for (uint32_t i = threadIdx.x % 32; i < a.n_seq; i += 32) {
    const uint64_t w = seq_work<ROWS, TW>(a, load_seq(a, i));
    total += w;
    before += i < s ? w : 0;
  }
  before = warp_sum(before);
  total = warp_sum(total);
  const uint32_t ctas = static_cast<uint32_t>(min(uint64_t(grid), total));
  const uint64_t first = before + (uint64_t(head) * rts + rt) * tiles;
  const uint32_t c0 = range_owner(total, first, ctas), c1 = range_owner(total, first + tiles - 1, ctas);
  if (c0 == c1) return;
  // slot 1 of the CTA the item starts in; slot 0 of the others, which an earlier one began
  const uint64_t stride = part_floats(ROWS, D);
  const auto slot = [&](uint32_t c) { return a.part + (uint64_t(c) * 2 + (c == c0 ? 1 : 0)) * stride; };
  const uint32_t lane = threadIdx.x % 32;
  float mx = -INFINITY;
  for (uint32_t c = c0 + lane; c <= c1; c += 32) mx = fmaxf(mx, slot(c)[ROWS * D + row]);
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float ref = mx == -INFINITY ? 0.f : mx;
  float den = 0.f, v[D / 32] = {};
#pragma unroll 4
  for (uint32_t c = c0; c <= c1; ++c) {
    const float* part = slot(c);
    const float f = exp2f(part[ROWS * D + row] - ref);
    den = fmaf(f, part[ROWS * (D + 1) + row], den);
#pragma unroll
    for (uint32_t i = 0; i < D / 32; ++i) v[i] = fmaf(f, part[row * D + lane + 32 * i], v[i]);
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const uint64_t to = (seq.first + rr / a.group) * a.out_token +
                      uint64_t(head * a.group + rr % a.group) * a.c.dim;
#pragma unroll
  for (uint32_t i = 0; i < D / 32; ++i)
    if (lane + 32 * i < a.c.dim) store_one(a.out, to + lane + 32 * i, v[i] * inv, a.type);
}

// Prepares, and launches, the kernels of one kind of cache.
template <uint32_t KIND>
cudaError_t prepare_kind();
template <uint32_t KIND>
cudaError_t launch_kind(const TreeArgs& a, bool split, bool wide, uint32_t ctas, cudaStream_t s);

template <uint32_t KIND, uint32_t D, bool SPLIT>
cudaError_t prepare_one() {
  return cudaFuncSetAttribute(tree_kernel<KIND, D, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Smem<KIND, D>::kBytes);
}

template <uint32_t KIND, uint32_t D, bool SPLIT>
cudaError_t launch_one(const TreeArgs& a, uint32_t ctas, cudaStream_t s) {
  tree_kernel<KIND, D, SPLIT><<<ctas, kThreads, Smem<KIND, D>::kBytes, s>>>(a);
  return cudaGetLastError();
}

}  // namespace tree
}  // namespace kq
