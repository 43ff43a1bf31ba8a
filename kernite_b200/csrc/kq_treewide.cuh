// kq_treewide.cuh -- attention of drafted tokens, many rows at once: the tcgen05 kernel. Work is cut as
// in kq_tree.cuh, with items of more rows.
//
// The 128 lanes of the tensor core's M are rows (drafted token x query head of the group): 128 of them
// for 16-bit activations; for f32 64 rows twice, as the f16 rounding of the operand and the f16
// rounding of what that left, 16 and 16 in the 32 lanes of a warp, so that the two halves of a row meet
// by a shuffle. S = Q K^T (Q and K in shared memory) and O += P V (P in tensor memory, where the
// softmax warps put it over the S they read) accumulate in tensor memory in f32.
//
// What the tensor core reads has to be f16 in its own layout, so the codes take one more step than in
// the warp-MMA kernel: eight warps turn a copied tile into the operand (each value exactly), once for
// all rows of the item. K and V use the same layout, 8 positions x 8 elements to a 128-byte core matrix:
// K-major for K (positions are N), N-major for V (elements are N).
//
// Roles: warps 0-3 softmax (warp w reads lanes 32 w ..), 4-11 decode, 12 copies, 13 issues the MMAs. In
// the steady state QK of the next tile and PV of this one run while the softmax of the next waits only
// for its own S (two S buffers).
#pragma once

#include "kq_tc.cuh"
#include "kq_tree.cuh"

namespace kq {
namespace tree {

constexpr uint32_t kDecodeWarps = 8;
constexpr uint32_t kWideThreads = (4 + kDecodeWarps + 2) * 32;

template <uint32_t KIND, uint32_t D>
struct Wide {
  using S = Shape<KIND, D>;
  static constexpr uint32_t TW = D == 256 ? 64 : 128;      // positions a tile
  static constexpr uint32_t kOperand = TW * D * 2;         // bytes of a K or V operand
  static constexpr uint32_t kOperands = 3;
  static constexpr uint32_t kQ = 128 * D * 2;
  static constexpr uint32_t kRaw = TW * (S::kRow + S::kScales);
  static constexpr uint32_t kFixed = kQ + kOperands * kOperand + 1024;
  static constexpr uint32_t kFit = (227 * 1024 - kFixed) / kRaw;
  static constexpr uint32_t kRaws = kFit > 6 ? 6 : kFit;
  static constexpr uint32_t kBytes = kFixed + kRaws * kRaw;
  static_assert(kRaws >= 2 && kBytes <= 227 * 1024, "ring");
  // tensor memory columns: two S (or one after the other's P), O
  static constexpr uint32_t kS = TW;
  static constexpr uint32_t kO = 256;
};

// Barriers of the wide kernel, 8 bytes each, from `bars`.
struct WideBars {
  uint32_t base;
  __device__ uint32_t raw_full(uint32_t i) const { return base + 8 * i; }
  __device__ uint32_t raw_empty(uint32_t i) const { return base + 64 + 8 * i; }
  __device__ uint32_t op_full(uint32_t i) const { return base + 128 + 8 * i; }
  __device__ uint32_t op_empty(uint32_t i) const { return base + 160 + 8 * i; }
  __device__ uint32_t s_full(uint32_t i) const { return base + 192 + 8 * i; }
  __device__ uint32_t p_full(uint32_t i) const { return base + 208 + 8 * i; }
  __device__ uint32_t q_full() const { return base + 224; }
  __device__ uint32_t pv_done() const { return base + 232; }
  __device__ uint32_t drained() const { return base + 240; }
};

// One bounded wait of a warp: false (for good) once any wait of it has given up.
__device__ __forceinline__ void wait_or_die(bool& live, uint32_t bar, uint32_t parity, unsigned* err, unsigned code) {
  if (live && !mbar_wait(bar, parity)) {
    report_error(err, code);
    live = false;
  }
  live = __all_sync(0xffffffffu, live);
}

// Eight consecutive elements (one core-matrix row) of a position from its codes.
__device__ __forceinline__ uint4 decode_q8(uint32_t w0, uint32_t w1, uint32_t s2) {
  return make_uint4(decode2(prmt(w0, kMagic, 0x4140), kOffset8, s2), decode2(prmt(w0, kMagic, 0x4342), kOffset8, s2),
                    decode2(prmt(w1, kMagic, 0x4140), kOffset8, s2), decode2(prmt(w1, kMagic, 0x4342), kOffset8, s2));
}

__device__ __forceinline__ uint4 decode_q4(uint32_t w, uint32_t s2) {
  constexpr uint32_t m = kMagic & 0xff00ff00u, k = 0x000f000fu;
  return make_uint4(decode2((w & k) | m, kOffset4, s2), decode2((w >> 4 & k) | m, kOffset4, s2),
                    decode2((w >> 8 & k) | m, kOffset4, s2), decode2((w >> 12 & k) | m, kOffset4, s2));
}

__device__ __forceinline__ void sts_v4(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

__device__ __forceinline__ void sts_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// One tile of keys or values from its copy into the operand's layout. left: positions the sequence has
// from the tile's first on. Values past the end, and not finite ones of drafts (from `drafts_at` on),
// become zero (see value_product); returns the drafts that had such values, as bits.
template <uint32_t KIND, uint32_t D>
__device__ __forceinline__ unsigned long long decode_tile(uint32_t raw, uint32_t seg_log2, uint32_t to, bool value,
                                                          uint32_t left, int drafts_at) {
  using W = Wide<KIND, D>;
  using S = Shape<KIND, D>;
  constexpr uint32_t PARTS = kDecodeWarps * 32 / W::TW;
  constexpr uint32_t UNITS = S::kRow / 16;  // 16-byte units of a row
  constexpr uint32_t E8 = S::kMost / 8;     // core-matrix rows a unit (f16: 1, Q8: 2, Q4: 4)
  const uint32_t id = threadIdx.x - 128, p = id % W::TW, part = id / W::TW;
  const TileView<S> tile = {raw, seg_log2};
  const bool gone = value && p >= left;
  const bool draft = value && static_cast<int>(p) >= drafts_at;
  bool special = false;
#pragma unroll
  for (uint32_t i = 0; i < UNITS / PARTS; ++i) {
    const uint32_t u = part * (UNITS / PARTS) + i;
    const uint4 w = lds_v4(tile.code(p, 16 * u));
    const uint32_t at = to + (u * E8 * (W::TW / 8) + p / 8) * 128 + (p % 8) * 16;
    constexpr uint32_t step = W::TW / 8 * 128;
    if constexpr (KIND == KQ_CACHE_F16) {
      uint4 v = w;
      if (draft) {
        v = make_uint4(finite_or_zero(w.x), finite_or_zero(w.y), finite_or_zero(w.z), finite_or_zero(w.w));
        special |= v.x != w.x || v.y != w.y || v.z != w.z || v.w != w.w;
      }
      if (gone) v = make_uint4(0, 0, 0, 0);
      sts_v4(at, v);
    } else {
      uint32_t s = lds_u8(tile.scale(p) + u * S::kMost / 32);
      if (draft && s >= 0xf8u) {
        special = true;
        s = 0;
      }
      if (gone) s = 0;
      const uint32_t s2 = s * 0x00800080u;
      if constexpr (KIND == KQ_CACHE_Q8) {
        sts_v4(at, decode_q8(w.x, w.y, s2));
        sts_v4(at + step, decode_q8(w.z, w.w, s2));
      } else {
        sts_v4(at, decode_q4(w.x, s2));
        sts_v4(at + step, decode_q4(w.y, s2));
        sts_v4(at + 2 * step, decode_q4(w.z, s2));
        sts_v4(at + 3 * step, decode_q4(w.w, s2));
      }
    }
  }
  return special && !gone ? 1ull << (static_cast<int>(p) - drafts_at) : 0ull;
}

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

// E consecutive activations from element i on.
template <uint32_t E>
__device__ __forceinline__ void load_acts(const void* p, uint64_t i, uint32_t type, float (&x)[E]) {
  if (type == KQ_TYPE_F32) {
    if constexpr (E == 2) load_act<float, 2>(static_cast<const float*>(p) + i, x);
    else {
#pragma unroll
      for (uint32_t j = 0; j < E; j += 4) {
        float y[4];
        load_act<float, 4>(static_cast<const float*>(p) + i + j, y);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) x[j + k] = y[k];
      }
    }
  } else if (type == KQ_TYPE_F16) {
    load_act<__half, E>(static_cast<const __half*>(p) + i, x);
  } else {
    load_act<__nv_bfloat16, E>(static_cast<const __nv_bfloat16*>(p) + i, x);
  }
}

template <uint32_t KIND, uint32_t D, bool SPLIT>
__global__ void __launch_bounds__(kWideThreads, 1) wide_kernel(const __grid_constant__ TreeArgs a) {
  using W = Wide<KIND, D>;
  using S = Shape<KIND, D>;
  constexpr uint32_t ROWS = SPLIT ? 64 : 128;
  constexpr uint32_t TW = W::TW;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t q_op = smem_u32(smem), ops = q_op + W::kQ, raws = ops + W::kOperands * W::kOperand;
  const uint32_t tail = W::kQ + W::kOperands * W::kOperand + W::kRaws * W::kRaw;
  const WideBars bar = {q_op + tail};
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + tail + 256);
  unsigned long long* special = reinterpret_cast<unsigned long long*>(smem + tail + 264);  // of the item's drafts
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < W::kRaws; ++i) {
      mbar_init(bar.raw_full(i), 1);
      mbar_init(bar.raw_empty(i), kDecodeWarps);
    }
    for (uint32_t i = 0; i < W::kOperands; ++i) {
      mbar_init(bar.op_full(i), kDecodeWarps);
      mbar_init(bar.op_empty(i), 1);
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(bar.s_full(i), 1);
      mbar_init(bar.p_full(i), 4);
    }
    mbar_init(bar.q_full(), 4);
    mbar_init(bar.pv_done(), 1);
    mbar_init(bar.drained(), 1);
    fence_mbar_init();
    special[0] = special[1] = 0;
  }
  const uint64_t total = work_before<ROWS, TW>(a, a.n_seq);
  const uint32_t ctas = static_cast<uint32_t>(min(uint64_t(gridDim.x), total));
  if (blockIdx.x >= ctas) return;
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
  Place p = locate<ROWS, TW>(a, at);
  bool live = true;
  const uint32_t seg_log2 = min(a.c.page_log2, TW == 128 ? 7u : 6u);

  if (warp == 4 + kDecodeWarps) {
    // ---- copies: raw tiles, keys and values in turn
    PageWindow window = {0xffffffffu, 0, 0};
    uint32_t it = 0;
    while (at < end) {
      const uint32_t tiles = position_tiles<TW>(p.seq);
      for (; p.tile < tiles && at < end; ++p.tile, ++at) {
#pragma unroll 1
        for (uint32_t kv = 0; kv < 2; ++kv, ++it) {
          const uint32_t slot = it % W::kRaws;
          if (it >= W::kRaws) wait_or_die(live, bar.raw_empty(slot), (it / W::kRaws - 1) & 1, a.err, kErrWaitEmpty);
          if (live) produce_tile<S, TW>(a, p, kv ? a.c.v : a.c.k, raws + slot * W::kRaw, bar.raw_full(slot), window);
        }
      }
      if (at < end) next_item<ROWS>(a, p);
    }
  } else if (warp == 5 + kDecodeWarps) {
    // ---- MMAs. Tile i's S goes to buffer i % 2, its P over it; QK of tile i + 1 is issued before PV
    // of tile i, and after PV of tile i - 1, which read the buffer.
    constexpr uint32_t idesc_qk = idesc_f16_f32(128, TW);
    constexpr uint32_t idesc_pv = idesc_f16_f32(128, D) | (1u << 16);  // B is N-major
    constexpr uint32_t q_lbo = 16 * 128, op_lbo = TW / 8 * 128;
    uint32_t n = 0, items = 0;  // tiles, items so far
    const auto qk = [&](uint32_t i) {
      // operand use 2i: keys of tile i
      const uint32_t use = 2 * i, slot = use % W::kOperands;
      wait_or_die(live, bar.op_full(slot), (use / W::kOperands) & 1, a.err, kErrWaitFull);
      tc_fence_after();
      if (live && lane == 0) {
        const uint32_t d = tmem + (i & 1) * W::kS;
#pragma unroll
        for (uint32_t ks = 0; ks < D / 16; ++ks)
          mma_f16_ss(d, smem_desc(q_op + ks * 2 * q_lbo, q_lbo, 128),
                     smem_desc(ops + slot * W::kOperand + ks * 2 * op_lbo, op_lbo, 128), idesc_qk, ks > 0);
        mma_commit(bar.op_empty(slot));
        mma_commit(bar.s_full(i & 1));
      }
      __syncwarp();
    };
    while (at < end) {
      const uint32_t tiles = position_tiles<TW>(p.seq);
      const uint32_t count = static_cast<uint32_t>(min(uint64_t(tiles - p.tile), end - at));
      wait_or_die(live, bar.q_full(), items & 1, a.err, kErrWaitFull);
      tc_fence_after();
      qk(n);
      for (uint32_t j = 0; j < count; ++j) {
        const uint32_t i = n + j;
        if (j + 1 < count) qk(i + 1);
        wait_or_die(live, bar.p_full(i & 1), (i >> 1) & 1, a.err, kErrWaitFull);
        const uint32_t use = 2 * i + 1, slot = use % W::kOperands;
        wait_or_die(live, bar.op_full(slot), (use / W::kOperands) & 1, a.err, kErrWaitFull);
        tc_fence_after();
        if (live && lane == 0) {
          const uint32_t pa = tmem + (i & 1) * W::kS;
#pragma unroll
          for (uint32_t kp = 0; kp < TW / 16; ++kp)
            mma_f16_ts(tmem + W::kO, pa + kp * 8, smem_desc(ops + slot * W::kOperand + kp * 256, 128, op_lbo),
                       idesc_pv, j > 0 || kp > 0);
          mma_commit(bar.op_empty(slot));
          mma_commit(bar.pv_done());
        }
        __syncwarp();
      }
      n += count;
      at += count;
      p.tile += count;
      ++items;
      if (at < end) next_item<ROWS>(a, p);
    }
    // nothing of this thread's is in flight after this, whatever happened before
    if (lane == 0) {
      mma_commit(bar.drained());
      if (!mbar_wait(bar.drained(), 0)) report_error(a.err, kErrWaitFull);
    }
  } else if (warp >= 4) {
    // ---- decode: copied tiles to operands
    uint32_t it = 0;
    uint32_t items = 0;
    while (at < end) {
      const uint32_t tiles = position_tiles<TW>(p.seq);
      for (; p.tile < tiles && at < end; ++p.tile, ++at) {
        const uint32_t base = p.tile * TW, left = p.seq.length() - base;
        const int drafts_at = static_cast<int>(p.seq.prefix) - static_cast<int>(base);
#pragma unroll 1
        for (uint32_t kv = 0; kv < 2; ++kv, ++it) {
          const uint32_t raw = it % W::kRaws, slot = it % W::kOperands;
          wait_or_die(live, bar.raw_full(raw), (it / W::kRaws) & 1, a.err, kErrWaitFull);
          if (it >= W::kOperands)
            wait_or_die(live, bar.op_empty(slot), (it / W::kOperands - 1) & 1, a.err, kErrWaitEmpty);
          const unsigned long long odd = decode_tile<KIND, D>(raws + raw * W::kRaw, seg_log2, ops + slot * W::kOperand,
                                                        kv, left, drafts_at);
          if (odd) atomicOr(special + (items & 1), odd);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bar.raw_empty(raw));
            mbar_arrive(bar.op_full(slot));
          }
        }
      }
      ++items;
      if (at < end) next_item<ROWS>(a, p);
    }
  } else {
    // ---- softmax
    const uint32_t lanes = tmem + ((warp * 32) << 16);
    uint32_t n = 0, items = 0;
    while (at < end) {
      // Q as operand A: lane m's row is 16 (m / 32) + m % 16, parts (m % 32) / 16, or row m; each row
      // scaled by a power of two to a largest element in [2^7, 2^8)
      const uint32_t rows = p.seq.drafts * a.group;
      const uint32_t my_row = p.rows * ROWS + (SPLIT ? warp * 16 + lane % 16 : warp * 32 + lane);
      float unit = a.scale_log2;
      constexpr uint32_t E = D / 32, AHEAD = 4;
#pragma unroll 1
      for (uint32_t r0 = 0; r0 < ROWS / 4; r0 += AHEAD) {
        float x[AHEAD][E];
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
          const uint32_t r = p.rows * ROWS + warp * (ROWS / 4) + r0 + k;
#pragma unroll
          for (uint32_t j = 0; j < E; ++j) x[k][j] = 0.f;
          if (r < rows && lane * E < a.c.dim)
            load_acts<E>(a.q, (p.seq.first + r / a.group) * a.q_token +
                                  uint64_t(p.head * a.group + r % a.group) * a.c.dim + lane * E, a.type, x[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
          float most = 0.f;
#pragma unroll
          for (uint32_t j = 0; j < E; ++j) most = fmaxf(most, fabsf(x[k][j]));
#pragma unroll
          for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          const int ex = static_cast<int>(__float_as_uint(most) >> 23) - 127;
          const int sh = most > 0.f && ex < 128 ? min(max(7 - ex, -120), 120) : 0;
          const float up = __int_as_float((127 + sh) << 23);
          const uint32_t r = r0 + k;  // of the warp's
          if ((SPLIT ? lane % 16 : lane) == r) unit = __int_as_float((127 - sh) << 23) * a.scale_log2;
          const uint32_t m = warp * 32 + r;
#pragma unroll
          for (uint32_t j = 0; j < E; j += 2) {
            const uint32_t e = lane * E + j;
            uint32_t hi, lo;
            split2(x[k][j] * up, x[k][j + 1] * up, hi, lo);
            const uint32_t to = q_op + (e / 8 * 16 + m / 8) * 128 + (m % 8) * 16 + (e % 8) * 2;
            sts_u32(to, hi);
            if constexpr (SPLIT) sts_u32(to + 256, lo);  // lane m + 16
          }
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar.q_full());
      const bool have = my_row < rows;
      const unsigned long long bits = have ? mask_bits(a, p.seq, my_row / a.group) : 0ull;

      float m = -INFINITY, l = 0.f;
      const uint32_t tiles = position_tiles<TW>(p.seq), first_tile = p.tile;
      constexpr uint32_t COLS = SPLIT ? TW / 2 : TW;  // columns a lane has of its row
      const uint32_t col0 = SPLIT && lane >= 16 ? TW / 2 : 0;
      for (; p.tile < tiles && at < end; ++p.tile, ++at, ++n) {
        const uint32_t base = p.tile * TW;
        const bool edge = base + TW > p.seq.prefix;
        const uint32_t sbuf = lanes + (n & 1) * W::kS;
        wait_or_die(live, bar.s_full(n & 1), (n >> 1) & 1, a.err, kErrWaitFull);
        tc_fence_after();
        // the lane's logits (times unit: log2 units), masked
        float s[SPLIT ? COLS : 1];
        float mx = -INFINITY;
        if constexpr (SPLIT) {
#pragma unroll
          for (uint32_t c = 0; c < COLS; c += 16) {
            uint32_t u[16], v[16];
            tmem_ld16(sbuf + c, u);
            tmem_ld16(sbuf + c + TW / 2, v);
            tmem_wait_ld();
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
              // each half of the pair of lanes keeps half of the columns
              const uint32_t keep = lane < 16 ? u[i] : v[i], send = lane < 16 ? v[i] : u[i];
              float x = __uint_as_float(keep) + __uint_as_float(__shfl_xor_sync(0xffffffffu, send, 16));
              if (edge && !sees(bits, base + col0 + c + i, p.seq)) x = -INFINITY;
              s[c + i] = x;
              mx = fmaxf(mx, x);
            }
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        } else {
#pragma unroll 1
          for (uint32_t c = 0; c < COLS; c += 32) {
            uint32_t u[16], v[16];
            tmem_ld16(sbuf + c, u);
            tmem_ld16(sbuf + c + 16, v);
            tmem_wait_ld();
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
              float x = __uint_as_float(u[i]), y = __uint_as_float(v[i]);
              if (edge) {
                if (!sees(bits, base + c + i, p.seq)) x = -INFINITY;
                if (!sees(bits, base + c + 16 + i, p.seq)) y = -INFINITY;
              }
              mx = fmaxf(mx, fmaxf(x, y));
            }
          }
        }
        mx *= unit;
        const bool grow = mx > m + kSlack || (m == -INFINITY && mx > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float to = grow ? mx : m;
          const float f = grow ? exp2f(m - to) : 1.f;
          m = to;
          l *= f;
          if (p.tile > first_tile) {
            // the output so far is rescaled once the product that adds to it is done
            wait_or_die(live, bar.pv_done(), (n - 1) & 1, a.err, kErrWaitFull);
            tc_fence_after();
#pragma unroll 1
            for (uint32_t c = 0; c < D; c += 16) {
              uint32_t u[16];
              tmem_ld16(lanes + W::kO + c, u);
              tmem_wait_ld();
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * f);
              tmem_st16(lanes + W::kO + c, u);
            }
            tmem_wait_st();
          }
        }
        const float ref = m == -INFINITY ? 0.f : m - kLift;
        if constexpr (SPLIT) {
          // weights as two f16; the pair of lanes exchanges so that one has the first parts of all
          // columns, the other the second ones
#pragma unroll
          for (uint32_t c = 0; c < COLS; c += 32) {
            uint32_t first[16], second[16];  // words of columns [c, c + 32) and TW / 2 + the same
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
              const float w0 = exp2f(fmaf(s[c + 2 * i], unit, -ref)), w1 = exp2f(fmaf(s[c + 2 * i + 1], unit, -ref));
              l += w0 + w1;
              uint32_t hi, lo;
              split2(w0, w1, hi, lo);
              const uint32_t got = __shfl_xor_sync(0xffffffffu, lane < 16 ? lo : hi, 16);
              first[i] = lane < 16 ? hi : got;
              second[i] = lane < 16 ? got : lo;
            }
            tmem_st16(sbuf + c / 2, first);
            tmem_st16(sbuf + c / 2 + TW / 4, second);
          }
        } else {
#pragma unroll 1
          for (uint32_t c = 0; c < COLS; c += 32) {
            uint32_t u[16], v[16], w[16];
            tmem_ld16(sbuf + c, u);
            tmem_ld16(sbuf + c + 16, v);
            tmem_wait_ld();
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
              float x = __uint_as_float(i < 8 ? u[2 * i] : v[2 * i - 16]);
              float y = __uint_as_float(i < 8 ? u[2 * i + 1] : v[2 * i - 15]);
              if (edge) {
                if (!sees(bits, base + c + 2 * i, p.seq)) x = -INFINITY;
                if (!sees(bits, base + c + 2 * i + 1, p.seq)) y = -INFINITY;
              }
              const __half2 h = __floats2half2_rn(exp2f(fmaf(x, unit, -ref)), exp2f(fmaf(y, unit, -ref)));
              w[i] = h2(h);
              const float2 f = __half22float2(h);
              l += f.x + f.y;
            }
            // columns [c, c + 32) become words [c / 2, c / 2 + 16): over columns already read
            tmem_st16(sbuf + c / 2, w);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.p_full(n & 1));
      }

      // ---- the item's output
      const bool whole = first_tile == 0 && p.tile == tiles;
      float* part = a.part + (uint64_t(blockIdx.x) * 2 + (first_tile ? 0 : 1)) * part_floats(ROWS, D);
      wait_or_die(live, bar.pv_done(), (n - 1) & 1, a.err, kErrWaitFull);
      tc_fence_after();
      if constexpr (SPLIT) l += __shfl_xor_sync(0xffffffffu, l, 16);
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
      // every tile's values were decoded before their product: the flags are complete, and the next
      // item's go to the other word
      const unsigned long long odd = *reinterpret_cast<volatile unsigned long long*>(special + (items & 1)) & bits;
      const uint32_t in_tile = my_row - p.rows * ROWS;
      const uint64_t to = (p.seq.first + (have ? my_row / a.group : 0)) * a.out_token +
                          uint64_t(p.head * a.group + my_row % a.group) * a.c.dim;
      constexpr uint32_t HALF = SPLIT ? D / 2 : D;
      const uint32_t e0 = SPLIT && lane >= 16 ? HALF : 0;
#pragma unroll 1
      for (uint32_t c = 0; c < HALF; c += 16) {
        uint32_t u[16], v[16];
        tmem_ld16(lanes + W::kO + c, u);
        if constexpr (SPLIT) tmem_ld16(lanes + W::kO + c + HALF, v);
        tmem_wait_ld();
        float y[16];
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
          if constexpr (SPLIT) {
            const uint32_t keep = lane < 16 ? u[i] : v[i], send = lane < 16 ? v[i] : u[i];
            y[i] = __uint_as_float(keep) + __uint_as_float(__shfl_xor_sync(0xffffffffu, send, 16));
          } else {
            y[i] = __uint_as_float(u[i]);
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
      if (have && !whole && (!SPLIT || lane < 16)) {
        part[ROWS * D + in_tile] = m;
        part[ROWS * (D + 1) + in_tile] = l;
      }
      tc_fence_before();  // O is read before the next item's first product writes it
      named_barrier(1, 128);
      if (threadIdx.x == 0) special[items & 1] = 0;
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
  wide_kernel<KIND, D, SPLIT><<<ctas, kWideThreads, Wide<KIND, D>::kBytes, s>>>(a);
  return cudaGetLastError();
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
