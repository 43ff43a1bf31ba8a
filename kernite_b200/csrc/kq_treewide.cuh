// kq_treewide.cuh -- attention of drafted tokens, many rows at once: the tcgen05 kernel. Work is cut as
// in kq_tree.cuh, with items of more rows.
//
// The 128 lanes of the tensor core's M are rows (drafted token x query head of the group): 128 of them
// for 16-bit activations; for f32 64 rows twice, as the f16 rounding of the operand and the f16
// rounding of what that left, 16 and 16 in the 32 lanes of a warp, so that the two halves of a row meet
// by a shuffle. S = Q K^T and O += P V accumulate in tensor memory in f32; Q and P are operands there
// too (P over the S it comes from), so that shared memory, which the decoding loads already, gives the
// tensor core K and V alone.
//
// What the tensor core reads has to be f16 in its own layout, so the codes take one more step than in
// the warp-MMA kernel: eight warps turn a copied tile into the operand (each value exactly), once for
// all rows of the item. K and V use the same layout, 8 positions x 8 elements to a 128-byte core matrix:
// K-major for K (positions are N), N-major for V (elements are N).
//
// Roles: warps 0-3 and 4-7 softmax, of even and of odd tiles (warp w has lanes 32 (w mod 4) ..); 8-11
// decode keys, 12-15 values; 16 issues the MMAs; 17 and 18 copy keys and values. A buffer's way round
// (QK, softmax, PV, the next QK) is long against any one of its steps, so tiles are short (64 positions)
// and three or four S buffers are under way at once. Each softmax group has its own maxima, sums and,
// up to a pitch of 128, its own O, joined at an item's end; at 256 there is room for one O, and a tile's
// maximum is passed on to the group that has the next tile.
//
// What bounds it. A tile of 64 positions x 128 elements takes the tensor core 520 cycles (M = 128) and the
// special function unit 512 for its exponentials; it takes 1300 to 1390, whatever number of rows is real: a
// softmax group's way through its tile (read S, maximum, exponentials, P back) is some 2450 cycles of
// latencies, and there is room for two groups (tensor pipe 37 %, issue slots 56 %, 760 instructions a tile and
// scheduler). 4 sequences of 64 drafts x 64 / 8 heads over 11000 positions each of 8-bit keys and values, bf16:
// 128 us, 0.72 PFLOP/s, of 16-bit ones 158 us; 25 f32 drafts over 8191: 46 us. Holding all of S in registers
// instead of reading it twice spilled (149 us against 127), and with registers moved from the other warps was
// no faster (127). MMAs issued by lane 0 instead of an elected thread took 573 us, two S buffers 200.
#pragma once

#include "kq_tc.cuh"
#include "kq_tree.cuh"

namespace kq {
namespace tree {

constexpr uint32_t kSoftWarps = 8, kDecodeWarps = 8;
constexpr uint32_t kMmaWarp = kSoftWarps + kDecodeWarps, kCopyWarp = kMmaWarp + 1;  // and + 2
constexpr uint32_t kWideThreads = (kSoftWarps + kDecodeWarps + 3) * 32;

template <uint32_t KIND, uint32_t D>
struct Wide {
  using S = Shape<KIND, D>;
  static constexpr uint32_t TW = 64;                       // positions a tile
  static constexpr uint32_t kOperand = TW * D * 2;         // bytes of a K or V operand
  static constexpr uint32_t kOperands = D == 256 ? 4 : 8;  // keys and values in turn
  static constexpr uint32_t kRaw = TW * (S::kRow + S::kScales);
  static constexpr uint32_t kFixed = kOperands * kOperand + 4096;
  static constexpr uint32_t kFit = (227 * 1024 - kFixed) / kRaw;
  // keys and values in turn; even, so that a slot is always keys' or values' and the warps of one see every
  // phase of their slots' barriers
  static constexpr uint32_t kRaws = kFit > 8 ? 8 : kFit / 2 * 2;
  static constexpr uint32_t kBytes = kFixed + kRaws * kRaw;
  static_assert(kRaws >= 2 && kBytes <= 227 * 1024, "ring");
  // Flag words (decoder to softmax, a word an item in turn). Values are decoded as far ahead as their operand
  // slots let them, which in items of one tile is that many items: none may come back to the word of the item
  // that is being finished.
  static constexpr uint32_t kFlags = 8;
  static_assert(kFlags > kOperands / 2 && (kFlags & (kFlags - 1)) == 0, "flag words");
  // tensor memory columns: S (then P) buffers, O (one a softmax group where there is room), Q
  static constexpr bool kOwnO = D <= 128;
  static constexpr uint32_t kBufs = D == 256 ? 2 : D == 128 ? 3 : 4;
  static constexpr uint32_t kS = TW;
  static constexpr uint32_t kO = kBufs * TW;
  static constexpr uint32_t kQ = kO + (kOwnO ? 2 : 1) * D;
  static_assert(kQ + D / 2 <= 512, "tensor memory");
};

// Barriers of the wide kernel, 8 bytes each, from `bars`.
struct WideBars {
  uint32_t base;
  __device__ uint32_t raw_full(uint32_t i) const { return base + 8 * i; }
  __device__ uint32_t raw_empty(uint32_t i) const { return base + 64 + 8 * i; }
  __device__ uint32_t op_full(uint32_t i) const { return base + 128 + 8 * i; }
  __device__ uint32_t op_empty(uint32_t i) const { return base + 192 + 8 * i; }
  __device__ uint32_t s_full(uint32_t i) const { return base + 256 + 8 * i; }
  __device__ uint32_t p_full(uint32_t i) const { return base + 288 + 8 * i; }
  __device__ uint32_t pv_done(uint32_t i) const { return base + 320 + 8 * i; }
  __device__ uint32_t q_full() const { return base + 352; }
  __device__ uint32_t drained() const { return base + 360; }
};

// True in one lane of a converged warp. The compiler knows that one thread runs what this guards, which a
// comparison of lane numbers does not tell it: a tcgen05.mma then costs its own time to issue instead
// of about 200 cycles (measured, M = 128, N = 16..128).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b32 r;\n\telect.sync r|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(one));
  return one != 0;
}

// One bounded wait of a warp: false (for good) once any wait of it has given up.
__device__ __forceinline__ void wait_or_die(bool& live, uint32_t bar, uint32_t parity, unsigned* err, unsigned code) {
  if (live && !mbar_wait(bar, parity)) {
    report_error(err, code);
    live = false;
  }
  live = __all_sync(0xffffffffu, live);
}

// Warp-collective: N consecutive 32-bit columns of each thread's own lane, waited for in the same
// statement, so that nothing that uses them can come before the wait.
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16]; tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
      "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
      "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32]; tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
      "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
      "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
      "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
      "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}

// Two runs of 16.
__device__ __forceinline__ void tmem_read(uint32_t ta, uint32_t (&u)[16], uint32_t tb, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%32]; tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33]; "
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
      "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
      "=r"(u[14]), "=r"(u[15]), "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]),
      "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
      "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(ta), "r"(tb)
      : "memory");
}

// Eight consecutive elements (one core-matrix row) of a position from its codes.
template <uint32_t KIND>
__device__ __forceinline__ uint4 decode8(uint32_t w0, uint32_t w1, const Scale2& s) {
  if constexpr (KIND == KQ_CACHE_Q8)
    return make_uint4(decode2(prmt(w0, kMagic, 0x4140), s), decode2(prmt(w0, kMagic, 0x4342), s),
                      decode2(prmt(w1, kMagic, 0x4140), s), decode2(prmt(w1, kMagic, 0x4342), s));
  else  // w0 alone
    return make_uint4(decode2(nibbles(nibble_up(w0, 0)), s), decode2(nibbles(nibble_up(w0, 1)), s),
                      decode2(nibbles(nibble_up(w0, 2)), s), decode2(nibbles(nibble_up(w0, 3)), s));
}

__device__ __forceinline__ void sts_v4(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

__device__ __forceinline__ void sts_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// A decoding thread's share of its group's tiles (keys or values): position p, N units of its row from
// part * N on. row = a power of two above 16, and 16 u < row, so (p row + 16 u) ^ swizzle is
// (p row ^ swizzle) ^ 16 u.
template <uint32_t KIND, uint32_t D>
struct Decoder {
  using W = Wide<KIND, D>;
  using S = Shape<KIND, D>;
  static constexpr uint32_t PARTS = kDecodeWarps / 2 * 32 / W::TW;
  static constexpr uint32_t N = S::kRow / 16 / PARTS;  // 16-byte units of a thread
  static constexpr uint32_t E8 = S::kMost / 8;         // core-matrix rows a unit (f16: 1, Q8: 2, Q4: 4)
  static constexpr uint32_t kStep = W::TW / 8 * 128;   // from one eight elements to the next
  static_assert(PARTS >= 1 && N >= 1, "a thread's share is whole units");
  static constexpr uint32_t kBytes = N * S::kMost / 32;  // scale bytes: 1, 2 or 4
  uint32_t p, part, seg, row, scale, to;

  __device__ explicit Decoder(uint32_t seg_log2) {
    const uint32_t id = (threadIdx.x - kSoftWarps * 32) % (kDecodeWarps / 2 * 32);
    p = id % W::TW;
    part = id / W::TW;
    const uint32_t in = p & ((1u << seg_log2) - 1);
    seg = ((p >> seg_log2) << seg_log2) * (S::kRow + S::kScales);
    row = in * S::kRow ^ cache_swizzle(in, S::kRow) << 4;
    scale = seg + (S::kRow << seg_log2) + in * S::kScales + part * kBytes;
    to = (part * N * E8 * (W::TW / 8) + p / 8) * 128 + (p % 8) * 16;
  }

  // A tile from its copy into the operand's layout. EDGE (values of a tile that reaches past the prefix;
  // left: positions the sequence has from its first on): values past the end, and not finite ones of
  // drafts (positions from drafts_at on), become zero (see value_product); returns the drafts that had
  // such values, as bits.
  template <bool EDGE>
  __device__ __forceinline__ unsigned long long run(uint32_t raw, uint32_t out, uint32_t left, int drafts_at) const {
    const bool gone = EDGE && p >= left;
    const bool draft = EDGE && static_cast<int>(p) >= drafts_at;
    bool special = false;
    uint32_t bytes = 0;
    if constexpr (S::kScales != 0)
      bytes = kBytes == 4 ? lds_u32(raw + scale) : kBytes == 2 ? lds_u16(raw + scale) : lds_u8(raw + scale);
    Scale2 s[kBytes];
    if constexpr (S::kScales != 0) {
#pragma unroll
      for (uint32_t i = 0; i < kBytes; ++i) {
        uint32_t b = bytes >> (8 * i) & 0xffu;
        if constexpr (EDGE) {
          if (draft && b >= 0xf8u) {
            special = true;
            b = 0;
          }
          if (gone) b = 0;
        }
        s[i] = scale2<KIND>(b, b);
      }
    }
    constexpr uint32_t AT_ONCE = N < 4 ? N : 4;
#pragma unroll
    for (uint32_t i0 = 0; i0 < N; i0 += AT_ONCE) {
      uint4 w[AT_ONCE];
#pragma unroll
      for (uint32_t k = 0; k < AT_ONCE; ++k) w[k] = lds_v4(raw + seg + (row ^ 16 * (part * N + i0 + k)));
#pragma unroll
      for (uint32_t k = 0; k < AT_ONCE; ++k) {
        const uint32_t i = i0 + k, at = out + to + i * E8 * kStep;
        if constexpr (KIND == KQ_CACHE_F16) {
          uint4 v = w[k];
          if constexpr (EDGE) {
            if (draft) {
              v = make_uint4(finite_or_zero(v.x), finite_or_zero(v.y), finite_or_zero(v.z), finite_or_zero(v.w));
              special |= v.x != w[k].x || v.y != w[k].y || v.z != w[k].z || v.w != w[k].w;
            }
            if (gone) v = make_uint4(0, 0, 0, 0);
          }
          sts_v4(at, v);
        } else if constexpr (KIND == KQ_CACHE_Q8) {
          const Scale2& z = s[i * S::kMost / 32];
          sts_v4(at, decode8<KIND>(w[k].x, w[k].y, z));
          sts_v4(at + kStep, decode8<KIND>(w[k].z, w[k].w, z));
        } else {
          const Scale2& z = s[i * S::kMost / 32];
          sts_v4(at, decode8<KIND>(w[k].x, 0, z));
          sts_v4(at + kStep, decode8<KIND>(w[k].y, 0, z));
          sts_v4(at + 2 * kStep, decode8<KIND>(w[k].z, 0, z));
          sts_v4(at + 3 * kStep, decode8<KIND>(w[k].w, 0, z));
        }
      }
    }
    return special && !gone ? 1ull << (static_cast<int>(p) - drafts_at) : 0ull;
  }
};

// Element e of the value at position pos, from the cache itself.
template <uint32_t KIND, uint32_t D>
__device__ __forceinline__ float value_at(const TreeArgs& a, const Place& p, uint32_t pos, uint32_t e) {
  using S = Shape<KIND, D>;
  const uint32_t id = static_cast<uint32_t>(a.pages[uint64_t(p.s) * a.max_pages + (pos >> a.c.page_log2)]);
  if (id >= a.c.n_pages) return 0.f;
  const uint8_t* rec = a.c.v + a.c.at(id, p.head);
  const uint32_t in = pos & (a.c.page() - 1);
  if constexpr (KIND == KQ_CACHE_F16)
    return __half2float(*reinterpret_cast<const __half*>(rec + cache_offset(in, 2 * e, S::kRow)));
  return rec[a.c.page() * S::kRow + in * S::kScales + e / 32] >= 0xf8u ? __int_as_float(0x7fc00000) : 0.f;
}

template <uint32_t KIND, uint32_t D, bool SPLIT>
__global__ void __launch_bounds__(kWideThreads, 1) wide_kernel(const __grid_constant__ TreeArgs a) {
  using W = Wide<KIND, D>;
  using S = Shape<KIND, D>;
  constexpr uint32_t ROWS = SPLIT ? 64 : 128;
  constexpr uint32_t TW = W::TW;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t ops = smem_u32(smem), raws = ops + W::kOperands * W::kOperand;
  const uint32_t tail = W::kOperands * W::kOperand + W::kRaws * W::kRaw;
  const WideBars bar = {ops + tail};
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + tail + 384);
  // drafts whose values are not finite, as bits; [W::kFlags]
  unsigned long long* special = reinterpret_cast<unsigned long long*>(smem + tail + 392);
  // what the two softmax groups tell each other
  float* exchange = reinterpret_cast<float*>(smem + tail + 512);
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < W::kRaws; ++i) {
      mbar_init(bar.raw_full(i), 1);
      mbar_init(bar.raw_empty(i), kDecodeWarps / 2);
    }
    for (uint32_t i = 0; i < W::kOperands; ++i) {
      mbar_init(bar.op_full(i), kDecodeWarps / 2);
      mbar_init(bar.op_empty(i), 1);
    }
    for (uint32_t i = 0; i < W::kBufs; ++i) {
      mbar_init(bar.s_full(i), 1);
      mbar_init(bar.p_full(i), kSoftWarps / 2);
      mbar_init(bar.pv_done(i), 1);
    }
    mbar_init(bar.q_full(), kSoftWarps);
    mbar_init(bar.drained(), 1);
    fence_mbar_init();
    for (uint32_t i = 0; i < W::kFlags; ++i) special[i] = 0;
  }
  pdl_wait();
  pdl_launch_dependents();
  const Work<ROWS, TW> work(a);
  const uint64_t total = work.total;
  const uint32_t ctas = static_cast<uint32_t>(min(uint64_t(gridDim.x), total));
  if (blockIdx.x >= ctas) {
    if (threadIdx.x == 0) Split{0, 0, 0, 0, 0}.store(a, blockIdx.x);
    return;
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  uint64_t at = range_start(total, blockIdx.x, ctas);
  const uint64_t end = range_start(total, blockIdx.x + 1, ctas);
  Place p = locate(a, work, at);
  bool live = true;
  const uint32_t seg_log2 = min(a.c.page_log2, 6u);

  if (warp >= kCopyWarp) {
    // ---- copies, from one thread: raw tiles of keys (use 2 i of the ring) or of values (2 i + 1)
    if (elect_one()) {
      const uint32_t kv = warp - kCopyWarp;
      const uint8_t* src = kv ? a.c.v : a.c.k;
      PageIds<TW> ids;
      ids.load(a, p);
      uint32_t it = kv, sent = kv;  // the next use, and the one after the last copied
      while (at < end) {
        const uint32_t tiles = position_tiles<TW>(p.seq);
        while (p.tile < tiles && at < end) {
          const uint32_t slot = it % W::kRaws;
          const Place now = p;
          const PageIds<TW> these = ids;
          // the next tile's pages come in while this one waits for its slot
          ++p.tile;
          ++at;
          if (at < end && p.tile < tiles) ids.load(a, p);
          if (it >= W::kRaws && live && !mbar_wait(bar.raw_empty(slot), (it / W::kRaws - 1) & 1)) {
            report_error(a.err, kErrWaitEmpty);
            live = false;
          }
          if (live) {
            copy_tile<S, TW>(a, now, these, src, raws + slot * W::kRaw, bar.raw_full(slot));
            sent = it + 2;
          }
          it += 2;
        }
        if (at < end) {
          next_item<ROWS>(a, p);
          ids.load(a, p);
        }
      }
      // no copy is in flight when the CTA ends, whatever gave up
      for (uint32_t use = sent > W::kRaws + kv ? sent - W::kRaws : kv; use < sent; use += 2)
        if (!mbar_wait(bar.raw_full(use % W::kRaws), (use / W::kRaws) & 1)) report_error(a.err, kErrWaitFull);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---- MMAs, all from one thread. Tile i's S goes to buffer i % kBufs, its P over it; QK of tile
    // i + kBufs - 1 is issued before PV of tile i, and after PV of tile i - 1, which read the buffer.
    if (elect_one()) {
      constexpr uint32_t idesc_qk = idesc_f16_f32(128, TW);
      constexpr uint32_t idesc_pv = idesc_f16_f32(128, D) | (1u << 16);  // B is N-major
      constexpr uint32_t op_lbo = TW / 8 * 128;
      // an operand's descriptors; another slot or step is an addition to the address field (16 bytes a unit)
      const uint64_t k_desc = smem_desc(ops, op_lbo, 128), v_desc = smem_desc(ops, 128, op_lbo);
      uint32_t n = 0, items = 0;  // tiles, items so far
      const auto wait = [&](uint32_t b, uint32_t parity) {
        if (live && !mbar_wait(b, parity)) {
          report_error(a.err, kErrWaitFull);
          live = false;
        }
      };
      const auto qk = [&](uint32_t i) {
        const uint32_t use = 2 * i, slot = use % W::kOperands;  // operand use 2i: keys of tile i
        wait(bar.op_full(slot), (use / W::kOperands) & 1);
        if (!live) return;
        tc_fence_after();
        const uint32_t d = tmem + i % W::kBufs * W::kS;
        const uint64_t b = k_desc + slot * (W::kOperand >> 4);
#pragma unroll
        for (uint32_t ks = 0; ks < D / 16; ++ks)
          mma_f16_ts(d, tmem + W::kQ + ks * 8, b + ks * (2 * op_lbo >> 4), idesc_qk, ks > 0);
        mma_commit(bar.op_empty(slot));
        mma_commit(bar.s_full(i % W::kBufs));
      };
      while (at < end) {
        const uint32_t tiles = position_tiles<TW>(p.seq);
        const uint32_t count = static_cast<uint32_t>(min(uint64_t(tiles - p.tile), end - at));
        wait(bar.q_full(), items & 1);
        for (uint32_t j = 0; j < min(count, W::kBufs - 1); ++j) qk(n + j);
        for (uint32_t j = 0; j < count; ++j) {
          const uint32_t i = n + j, buf = i % W::kBufs;
          if (j + W::kBufs - 1 < count) qk(i + W::kBufs - 1);
          wait(bar.p_full(buf), (i / W::kBufs) & 1);
          const uint32_t use = 2 * i + 1, slot = use % W::kOperands;
          wait(bar.op_full(slot), (use / W::kOperands) & 1);
          if (!live) continue;
          tc_fence_after();
          const uint32_t pa = tmem + buf * W::kS;
          const uint64_t b = v_desc + slot * (W::kOperand >> 4);
#pragma unroll
          for (uint32_t kp = 0; kp < TW / 16; ++kp)
            mma_f16_ts(tmem + W::kO + (W::kOwnO ? (i & 1) * D : 0), pa + kp * 8, b + kp * (256 >> 4), idesc_pv,
                       kp > 0 || j > (W::kOwnO ? 1 : 0));
          mma_commit(bar.op_empty(slot));
          mma_commit(bar.pv_done(buf));
        }
        n += count;
        at += count;
        p.tile += count;
        ++items;
        if (at < end) next_item<ROWS>(a, p);
      }
      // nothing of this thread's is in flight after this, whatever happened before
      mma_commit(bar.drained());
      if (!mbar_wait(bar.drained(), 0)) report_error(a.err, kErrWaitFull);
    }
    __syncwarp();
  } else if (warp >= kSoftWarps) {
    // ---- decode: copied tiles to operands, use 2 i + kv of both rings for tile i
    const uint32_t kv = (warp - kSoftWarps) / (kDecodeWarps / 2);
    const Decoder<KIND, D> decoder(seg_log2);
    uint32_t it = kv;
    uint32_t items = 0;
    while (at < end) {
      const uint32_t tiles = position_tiles<TW>(p.seq);
      for (; p.tile < tiles && at < end; ++p.tile, ++at, it += 2) {
        const uint32_t base = p.tile * TW, left = p.seq.length() - base;
        const int drafts_at = static_cast<int>(p.seq.prefix) - static_cast<int>(base);
        const uint32_t raw = it % W::kRaws, slot = it % W::kOperands;
        wait_or_die(live, bar.raw_full(raw), (it / W::kRaws) & 1, a.err, kErrWaitFull);
        if (it >= W::kOperands)
          wait_or_die(live, bar.op_empty(slot), (it / W::kOperands - 1) & 1, a.err, kErrWaitEmpty);
        const uint32_t from = raws + raw * W::kRaw, to = ops + slot * W::kOperand;
        if (kv && drafts_at < static_cast<int>(TW)) {
          const unsigned long long odd = decoder.template run<true>(from, to, left, drafts_at);
          if (odd) atomicOr(special + items % W::kFlags, odd);
        } else {
          decoder.template run<false>(from, to, left, drafts_at);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar.raw_empty(raw));
          mbar_arrive(bar.op_full(slot));
        }
      }
      ++items;
      if (at < end) next_item<ROWS>(a, p);
    }
  } else {
    // ---- softmax
    const uint32_t quad = warp % 4, half = warp / 4;  // the group: even or odd tiles, half of Q's and O's columns
    const uint32_t lanes = tmem + ((quad * 32) << 16);
    const uint32_t slot = quad * 32 + lane;
    // a value of this row's for the other group's thread, and the other's
    const auto swap = [&](uint32_t parity, float mine) {
      exchange[(parity * 2 + half) * 128 + slot] = mine;
      named_barrier(2 + quad, 64);
      return exchange[(parity * 2 + 1 - half) * 128 + slot];
    };
    const uint32_t my_o = lanes + W::kO + (W::kOwnO ? half * D : 0);
    float* chain = exchange + 512;  // [group][lane]: a row's maximum after the group's last tile
    uint32_t n = 0, items = 0, swaps = 0;
    while (at < end) {
      // Q as operand A: lane m's row is 16 (m / 32) + m % 16, parts (m % 32) / 16, or row m; scaled
      // (row_scale). This thread: half of its row.
      const uint32_t rows = p.seq.drafts * a.group;
      const uint32_t in_tile = SPLIT ? quad * 16 + lane % 16 : slot;
      const uint32_t my_row = p.rows * ROWS + in_tile;
      const bool have = my_row < rows;
      const bool second = SPLIT && lane >= 16;
      const uint32_t token = have ? token_of(a, my_row) : 0;
      const uint32_t q_head = p.head * a.group + (have ? head_of(a, my_row, token) : 0);
      const uint64_t q_row = (p.seq.first + token) * a.q_token + uint64_t(q_head) * a.c.dim;
      float unit;
      {
        // in chunks that registers hold: the last stays, one before it is read again
        constexpr uint32_t CHUNK = D / 16 < 8 ? D / 16 : 8, CHUNKS = D / 16 / CHUNK;
        float x[CHUNK][8];
        float most = 0.f;
        const auto load = [&](uint32_t c) {
          load_row(a, q_row, have, [&](uint32_t j) { return half * (D / 2) + 8 * (c * CHUNK + j); }, x);
        };
#pragma unroll
        for (uint32_t c = 0; c < CHUNKS; ++c) {
          load(c);
#pragma unroll
          for (uint32_t j = 0; j < CHUNK; ++j)
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) most = fmaxf(most, fabsf(x[j][k]));
        }
        most = fmaxf(most, swap(swaps++ & 1, most));
        const RowScale scale = row_scale<SPLIT>(most, a.scale_log2);
        const float up = scale.up;
        unit = scale.unit;
#pragma unroll
        for (uint32_t c = CHUNKS; c-- > 0;) {
          if (c + 1 < CHUNKS) load(c);
#pragma unroll
          for (uint32_t j0 = 0; j0 < CHUNK; j0 += 4) {
            uint32_t w[16];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
              for (uint32_t k = 0; k < 4; ++k) {
                uint32_t hi, lo;
                split2(x[j0 + j][2 * k] * up, x[j0 + j][2 * k + 1] * up, hi, lo);
                w[4 * j + k] = second ? lo : hi;
              }
            tmem_st16(lanes + W::kQ + half * (D / 4) + 4 * (c * CHUNK + j0), w);
          }
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar.q_full());
      const unsigned long long bits = have ? mask_bits(a, p.seq, token) : 0ull;

      float m = -INFINITY, l = 0.f;
      const uint32_t tiles = position_tiles<TW>(p.seq), first_tile = p.tile;
      constexpr uint32_t COLS = SPLIT ? TW / 2 : TW;  // columns a lane has of its row
      const uint32_t col0 = second ? COLS : 0;
      for (; p.tile < tiles && at < end; ++p.tile, ++at, ++n) {
        if ((n & 1) != half) continue;
        const uint32_t base = p.tile * TW;
        const bool edge = base + TW > p.seq.prefix;
        const uint32_t buf = n % W::kBufs, sbuf = lanes + buf * W::kS;
        // (of three buffers a group passes over every second phase; it cannot take the one before for
        // this one: that was tile n - 3's, done before tile n - 2's, which the group has seen)
        wait_or_die(live, bar.s_full(buf), (n / W::kBufs) & 1, a.err, kErrWaitFull);
        tc_fence_after();
        // the lane's logits (times unit: log2 units), masked in tiles that reach past the prefix
        float s[SPLIT ? COLS : 1];
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const int from = static_cast<int>(base + col0) - static_cast<int>(p.seq.prefix);
        if constexpr (SPLIT) {
#pragma unroll
          for (uint32_t c = 0; c < COLS; c += 16) {
            uint32_t u[16], v[16];
            tmem_read(sbuf + c, u, sbuf + c + COLS, v);
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
              // each of the pair of lanes keeps half of the columns
              const uint32_t keep = second ? v[i] : u[i], send = second ? u[i] : v[i];
              s[c + i] = __uint_as_float(keep) + __uint_as_float(__shfl_xor_sync(0xffffffffu, send, 16));
            }
          }
          if (edge) {
#pragma unroll
            for (uint32_t c = 0; c < COLS; c += 32) {
              const uint32_t seen = seen_word(bits, from + static_cast<int>(c));
#pragma unroll
              for (uint32_t i = 0; i < 32; ++i)
                if (!(seen >> i & 1u)) s[c + i] = -INFINITY;
            }
          }
#pragma unroll
          for (uint32_t c = 0; c < COLS; c += 2) m4[c / 2 & 3] = max3(m4[c / 2 & 3], s[c], s[c + 1]);
        } else {
          const auto largest = [&](uint32_t c, uint32_t seen) {
            uint32_t u[32];
            tmem_read(sbuf + c, u);
#pragma unroll
            for (uint32_t i = 0; i < 32; i += 2)
              m4[i / 2 & 3] = max3(m4[i / 2 & 3], seen >> i & 1u ? __uint_as_float(u[i]) : -INFINITY,
                                   seen >> (i + 1) & 1u ? __uint_as_float(u[i + 1]) : -INFINITY);
          };
          if (!edge) {
#pragma unroll
            for (uint32_t c = 0; c < COLS; c += 32) largest(c, ~0u);
          } else {
#pragma unroll 1
            for (uint32_t c = 0; c < COLS; c += 32) largest(c, seen_word(bits, from + static_cast<int>(c)));
          }
        }
        float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if constexpr (SPLIT) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mx *= unit;
        // the maximum so far: the group's own, or from the group that has the tile before (and this
        // one's for the next)
        float before = m;
        if constexpr (!W::kOwnO) {
          if (p.tile > first_tile) {
            named_barrier(6 + 2 * quad + (1 - half), 64);
            before = chain[(1 - half) * 128 + slot];
          }
        }
        const bool grow = mx > before + kSlack || (before == -INFINITY && mx > before);
        const float now = grow ? mx : before;
        if constexpr (!W::kOwnO) {
          if (p.tile + 1 < tiles && at + 1 < end) {
            chain[half * 128 + slot] = now;
            __syncwarp();
            asm volatile("bar.arrive %0, %1;" ::"r"(6 + 2 * quad + half), "r"(64) : "memory");
          }
        }
        constexpr uint32_t BACK = W::kOwnO ? 2 : 1;  // the tile whose product this one's adds to
        if (__any_sync(0xffffffffu, now != m)) {
          if (now != m) l *= exp2f(m - now);  // (the first time the sum is 0)
          m = now;
          if (__any_sync(0xffffffffu, grow) && p.tile >= first_tile + BACK) {
            // the output so far is rescaled once the product that adds to it is done (its buffer's
            // product before that one was done when this tile's S was)
            const float f = grow ? exp2f(before - now) : 1.f;
            const uint32_t prev = n - BACK;
            wait_or_die(live, bar.pv_done(prev % W::kBufs), (prev / W::kBufs) & 1, a.err, kErrWaitFull);
            tc_fence_after();
#pragma unroll 1
            for (uint32_t c = 0; c < D; c += 16) {
              uint32_t u[16];
              tmem_read(my_o + c, u);
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * f);
              tmem_st16(my_o + c, u);
            }
            tmem_wait_st();
          }
        }
        const float ref = m == -INFINITY ? 0.f : m - kLift;
        const float2 unit2 = make_float2(unit, unit), ref2 = make_float2(-ref, -ref);
        float2 sum = make_float2(0.f, 0.f);
        if constexpr (SPLIT) {
          // weights as two f16; the pair of lanes exchanges so that one has the first parts of all
          // columns, the other the second ones
#pragma unroll
          for (uint32_t c = 0; c < COLS; c += 32) {
            uint32_t first[16], last[16];  // words of columns [c, c + 32) and COLS + the same
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
              const float2 z = fma2(make_float2(s[c + 2 * i], s[c + 2 * i + 1]), unit2, ref2);
              const float w0 = exp2_fast(z.x), w1 = exp2_fast(z.y);
              sum = add2(sum, make_float2(w0, w1));
              uint32_t hi, lo;
              split2(w0, w1, hi, lo);
              const uint32_t got = __shfl_xor_sync(0xffffffffu, second ? hi : lo, 16);
              first[i] = second ? got : hi;
              last[i] = second ? lo : got;
            }
            tmem_st16(sbuf + c / 2, first);
            tmem_st16(sbuf + (COLS + c) / 2, last);
          }
        } else {
          // the columns again; columns [c, c + 32) become words [c / 2, c / 2 + 16), over ones already read
          // For logits in the millions one rounding of product and difference would leave more than a
          // weight's size: the product is rounded first, so that the largest gives the reference's weight.
          const auto weights = [&](uint32_t c, uint32_t seen, bool huge) {
            uint32_t u[32], w[16];
            tmem_read(sbuf + c, u);
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
              const float2 s2 = make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
              const float2 z = huge ? make_float2(__fmul_rn(s2.x, unit) - ref, __fmul_rn(s2.y, unit) - ref)
                                    : fma2(s2, unit2, ref2);
              const float x = seen >> (2 * i) & 1u ? exp2_fast(z.x) : 0.f;
              const float y = seen >> (2 * i + 1) & 1u ? exp2_fast(z.y) : 0.f;
              sum = add2(sum, make_float2(x, y));
              w[i] = h2(__floats2half2_rn(x, y));
            }
            tmem_st16(sbuf + c / 2, w);
          };
          if (!edge && !__any_sync(0xffffffffu, fabsf(m) > 0x1p20f && m != -INFINITY)) {
#pragma unroll
            for (uint32_t c = 0; c < COLS; c += 32) weights(c, ~0u, false);
          } else {
#pragma unroll 1
            for (uint32_t c = 0; c < COLS; c += 32)
              weights(c, edge ? seen_word(bits, from + static_cast<int>(c)) : ~0u, true);
          }
        }
        l += sum.x + sum.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.p_full(buf));
      }

      // ---- the item's output, half of the columns (and for pairs of lanes a quarter) a thread
      const bool whole = first_tile == 0 && p.tile == tiles;
      float* part = a.part + (uint64_t(blockIdx.x) * 2 + (first_tile ? 0 : 1)) * part_floats(ROWS, D);
      // the groups' sums (and outputs) over the larger maximum
      if constexpr (SPLIT) l += __shfl_xor_sync(0xffffffffu, l, 16);
      const float other_m = swap(swaps++ & 1, m);
      const float last_m = fmaxf(m, other_m);
      const float mine = m == last_m ? 1.f : exp2f(m - last_m);
      const float theirs = other_m == last_m ? 1.f : exp2f(other_m - last_m);
      l *= mine;
      l += swap(swaps++ & 1, l);
      m = last_m;
      // the item's last products (after the swaps both groups are past their last tile's S)
      const bool two = W::kOwnO && p.tile - first_tile > 1;
      wait_or_die(live, bar.pv_done((n - 1) % W::kBufs), ((n - 1) / W::kBufs) & 1, a.err, kErrWaitFull);
      if (two) wait_or_die(live, bar.pv_done((n - 2) % W::kBufs), ((n - 2) / W::kBufs) & 1, a.err, kErrWaitFull);
      tc_fence_after();
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
      // the last tile's group's O, and the other's: factors of this thread's row
      const uint32_t last_half = (n - 1) & 1;
      const uint32_t o_last = lanes + W::kO + (W::kOwnO ? last_half * D : 0);
      const uint32_t o_other = lanes + W::kO + (1 - last_half) * D;
      const float f_last = W::kOwnO ? (last_half == half ? mine : theirs) : 1.f;
      const float f_other = last_half == half ? theirs : mine;
      // every tile's values were decoded before their product: the flags are complete, and the items decoded
      // meanwhile have other words
      const unsigned long long odd =
          *reinterpret_cast<volatile unsigned long long*>(special + items % W::kFlags) & bits;
      const uint64_t to = (p.seq.first + token) * a.out_token + uint64_t(q_head) * a.c.dim;
      constexpr uint32_t WIDE = SPLIT ? D / 4 : D / 2;
      const uint32_t o0 = half * (D / 2), e0 = o0 + (second ? WIDE : 0);
#pragma unroll 1
      for (uint32_t c = 0; c < WIDE; c += 16) {
        uint32_t u[16], v[16];
        float y[16];
#pragma unroll
        for (uint32_t g = 0; g < (W::kOwnO ? 2u : 1u); ++g) {
          if (g == 1 && !two) break;
          const uint32_t o = (g ? o_other : o_last) + o0 + c;
          const float f = g ? f_other : f_last;
          if constexpr (SPLIT) tmem_read(o, u, o + WIDE, v);
          else tmem_read(o, u);
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) {
            float z = __uint_as_float(u[i]);
            if constexpr (SPLIT) {
              const float w = __uint_as_float(v[i]);
              z = (second ? w : z) + __shfl_xor_sync(0xffffffffu, second ? z : w, 16);
            }
            y[i] = g ? fmaf(f, z, y[i]) : f * z;
          }
        }
        for (unsigned long long left = odd; left; left &= left - 1) {
          const uint32_t d = __ffsll(left) - 1;
#pragma unroll 1
          for (uint32_t i = 0; i < 16; ++i) {
            const float w = value_at<KIND, D>(a, p, p.seq.prefix + d, e0 + c + i);
            if (!isfinite(w)) {
#pragma unroll
              for (uint32_t k = 0; k < 16; ++k)
                if (k == i) y[k] += w;
            }
          }
        }
        if (have && !whole) {
#pragma unroll
          for (uint32_t i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(part + in_tile * D + e0 + c + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
        } else if (have && e0 + c < a.c.dim) {
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) y[i] *= inv;
          if (a.type == KQ_TYPE_F32) {
#pragma unroll
            for (uint32_t i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(static_cast<float*>(a.out) + to + e0 + c + i) =
                  make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
          } else {
#pragma unroll
            for (uint32_t i = 0; i < 16; i += 8) {
              float z[8];
#pragma unroll
              for (uint32_t k = 0; k < 8; ++k) z[k] = y[i + k];
              if (a.type == KQ_TYPE_F16) store_act<__half, 8>(static_cast<__half*>(a.out) + to + e0 + c + i, z);
              else store_act<__nv_bfloat16, 8>(static_cast<__nv_bfloat16*>(a.out) + to + e0 + c + i, z);
            }
          }
        }
      }
      if (have && !whole && half == 0 && !second) {
        part[ROWS * D + in_tile] = m;
        part[ROWS * (D + 1) + in_tile] = l;
      }
      tc_fence_before();  // O is read before the next item's first product writes it
      named_barrier(1, kSoftWarps * 32);
      if (threadIdx.x == 0) {
        special[items % W::kFlags] = 0;
        if (at == end) leave_split(a, p, first_tile == 0, whole, total, end, p.tile - first_tile, tiles, ctas);
      }
      ++items;
      if (at < end) next_item<ROWS>(a, p);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <uint32_t KIND, uint32_t D, bool SPLIT>
cudaError_t prepare_wide() {
  return cudaFuncSetAttribute(wide_kernel<KIND, D, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Wide<KIND, D>::kBytes);
}

template <uint32_t KIND, uint32_t D, bool SPLIT>
cudaError_t launch_wide(const TreeArgs& a, uint32_t ctas, cudaStream_t s) {
  return launch_pdl(wide_kernel<KIND, D, SPLIT>, dim3(ctas), kWideThreads, Wide<KIND, D>::kBytes, s, a);
}

// Prepares, and launches, the kernels of one kind of cache (pitch 64, 128 or 256).
#define KQ_TREE_KIND(KIND)                                                                                \
  template <>                                                                                             \
  cudaError_t prepare_kind<KIND>() {                                                                      \
    cudaError_t e = cudaSuccess;                                                                          \
    for (auto prepare : {prepare_one<KIND, 64, false>, prepare_one<KIND, 64, true>,                       \
                         prepare_one<KIND, 128, false>, prepare_one<KIND, 128, true>,                     \
                         prepare_one<KIND, 256, false>, prepare_one<KIND, 256, true>,                     \
                         prepare_wide<KIND, 64, false>, prepare_wide<KIND, 64, true>,                     \
                         prepare_wide<KIND, 128, false>, prepare_wide<KIND, 128, true>,                   \
                         prepare_wide<KIND, 256, false>, prepare_wide<KIND, 256, true>})                  \
      if (e == cudaSuccess) e = prepare();                                                                \
    return e;                                                                                             \
  }                                                                                                       \
  template <>                                                                                             \
  cudaError_t launch_kind<KIND>(const TreeArgs& a, bool split, bool wide, uint32_t ctas, cudaStream_t s) { \
    const uint32_t d = a.c.pitch;                                                                         \
    if (wide)                                                                                             \
      return split ? (d == 64    ? launch_wide<KIND, 64, true>                                            \
                      : d == 128 ? launch_wide<KIND, 128, true>                                           \
                                 : launch_wide<KIND, 256, true>)(a, ctas, s)                              \
                   : (d == 64    ? launch_wide<KIND, 64, false>                                           \
                      : d == 128 ? launch_wide<KIND, 128, false>                                          \
                                 : launch_wide<KIND, 256, false>)(a, ctas, s);                            \
    return split ? (d == 64    ? launch_one<KIND, 64, true>                                               \
                    : d == 128 ? launch_one<KIND, 128, true>                                              \
                               : launch_one<KIND, 256, true>)(a, ctas, s)                                 \
                 : (d == 64    ? launch_one<KIND, 64, false>                                              \
                    : d == 128 ? launch_one<KIND, 128, false>                                             \
                               : launch_one<KIND, 256, false>)(a, ctas, s);                               \
  }

}  // namespace tree
}  // namespace kq
