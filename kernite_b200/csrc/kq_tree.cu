// kq_tree.cu -- attention of drafted tokens over the paged cache: argument checks, the choice of a
// kernel, the launches (kq_tree.cuh has the kernels).
#include <algorithm>
#include <cmath>
#include <string>

#include "kq_internal.h"
#include "kq_tree.cuh"

namespace kq {

namespace tree {
template <>
cudaError_t prepare_kind<KQ_CACHE_F16>();
template <>
cudaError_t prepare_kind<KQ_CACHE_Q8>();
template <>
cudaError_t prepare_kind<KQ_CACHE_Q4>();
template <>
cudaError_t launch_kind<KQ_CACHE_F16>(const TreeArgs&, bool, bool, uint32_t, cudaStream_t);
template <>
cudaError_t launch_kind<KQ_CACHE_Q8>(const TreeArgs&, bool, bool, uint32_t, cudaStream_t);
template <>
cudaError_t launch_kind<KQ_CACHE_Q4>(const TreeArgs&, bool, bool, uint32_t, cudaStream_t);
}  // namespace tree

namespace {

constexpr uint32_t kMaxTreeGroup = 64;

struct Plan {
  bool split;      // f32 activations: operands as sums of two f16
  bool wide;       // the tcgen05 kernel, else the warp-MMA one
  uint32_t rows;   // rows an item
  uint32_t tile;   // positions a tile
  uint32_t ctas;
  bool many;       // few rows of many parts each: join_kernel's SHARED
  uint64_t parts;  // workspace: bytes of the parts, and all
  uint64_t bytes;
  uint64_t most;   // all, whatever max_len and n_seq are
};

// The logits' scale in log2 units.
float scale_log2(const kq_tree_desc& d, const CacheView& c) {
  const double scale = d.scale > 0.f ? static_cast<double>(d.scale) : 1.0 / std::sqrt(static_cast<double>(c.dim));
  return static_cast<float>(scale * 1.4426950408889634);
}

// What does not depend on addresses: shapes, and the launch they give. KQ_OK or KQ_E_INVALID.
int plan(const kq_ctx* ctx, const kq_tree_desc& d, const CacheView& c, const char* call, Plan* out) {
  if (d.type != KQ_TYPE_F32 && d.type != KQ_TYPE_F16 && d.type != KQ_TYPE_BF16)
    return fail(KQ_E_INVALID, call, "type must be F32, F16 or BF16");
  if (d.n_heads == 0 || d.n_heads % c.n_kv || d.n_heads / c.n_kv > kMaxTreeGroup)
    return fail(KQ_E_INVALID, call, "n_heads must be 1..64 times the cache's n_kv");
  if (d.max_drafts == 0 || d.max_drafts > tree::kMaxDrafts)
    return fail(KQ_E_INVALID, call, "max_drafts must be 1..64");
  if (d.max_len == 0 || d.max_pages == 0) return fail(KQ_E_INVALID, call, "max_len and max_pages must be positive");
  if ((uint64_t(d.max_pages) << c.page_log2) > 0x7fffffffu)
    return fail(KQ_E_INVALID, call, "max_pages pages must hold fewer than 2^31 positions");
  if (d.n_seq > 0x7fffffffu || d.tokens > 0x7fffffffu) return fail(KQ_E_INVALID, call, "too many sequences or tokens");
  // (in log2 units it has to be an f32 too)
  if (!(d.scale >= 0.f) || !std::isfinite(scale_log2(d, c)))
    return fail(KQ_E_INVALID, call, "scale must be 0 to 2^127 and not NaN");
  Plan p = {};
  p.split = d.type == KQ_TYPE_F32;
  const uint32_t group = d.n_heads / c.n_kv;
  // One item of 8 rows fills the warp-MMA kernel's N; more would read the cache again for each, while the
  // tcgen05 kernel's time hardly grows up to 64. 16 sequences of 4000 positions, 8 bits, f32: 8 rows a
  // head 39 us against 62, 16 rows 61 and 64, 24 rows 87 and 64; 4 bits: 42 and 57, 67 and 58, 96 and 59.
  p.wide = d.max_drafts * group > 8u;
  p.rows = p.wide ? (p.split ? 64 : 128) : 8;
  p.tile = p.wide ? 64 : 128;
  const uint64_t row_tiles = (uint64_t(d.max_drafts) * group + p.rows - 1) / p.rows;
  const uint64_t tiles = (uint64_t(d.max_len) + p.tile - 1) / p.tile;
  const uint64_t items = uint64_t(d.n_seq) * c.n_kv * row_tiles;
  if (items > 0x7fffffffu) return fail(KQ_E_INVALID, call, "too many sequences, heads and drafts");
  // kernels number the tiles of one sequence in 32 bits, up to the length that its pages hold
  const uint64_t most = ((uint64_t(d.max_pages) << c.page_log2) + p.tile - 1) / p.tile;
  if (most * c.n_kv * row_tiles > 0xffffffffu)
    return fail(KQ_E_INVALID, call, "too many positions, heads and drafts in one sequence");
  const uint64_t full = uint64_t(ctx->sm_count) * (p.wide ? 1 : tree::narrow_ctas(c.kind, c.pitch));
  p.ctas = static_cast<uint32_t>(std::min<uint64_t>(full, std::max<uint64_t>(1, items * tiles)));
  p.many = !p.wide && p.ctas > 8 * items;  // more parts than a warp loads at once
  const uint64_t part = 2 * tree::part_floats(p.rows, c.pitch) * 4;  // a CTA's
  p.parts = p.ctas * part;
  p.bytes = p.ctas * (part + 2 * sizeof(uint4));
  p.most = full * (part + 2 * sizeof(uint4));
  *out = p;
  return KQ_OK;
}

template <uint32_t ROWS, bool SHARED>
cudaError_t launch_join(const tree::TreeArgs& a, uint32_t ctas, cudaStream_t s) {
  return launch_pdl(a.c.pitch == 64    ? tree::join_kernel<ROWS, 64, SHARED>
                    : a.c.pitch == 128 ? tree::join_kernel<ROWS, 128, SHARED>
                                       : tree::join_kernel<ROWS, 256, SHARED>,
                    dim3(ctas, SHARED ? ROWS : ROWS / 8), 256, 0, s, a);
}

bool on16(uint64_t bytes) { return bytes % 16 == 0; }

}  // namespace

int tree_prepare(kq_ctx*) {
  cudaError_t e = tree::prepare_kind<KQ_CACHE_F16>();
  if (e == cudaSuccess) e = tree::prepare_kind<KQ_CACHE_Q8>();
  if (e == cudaSuccess) e = tree::prepare_kind<KQ_CACHE_Q4>();
  return e == cudaSuccess ? KQ_OK : cuda_fail(e, "cudaFuncSetAttribute", "tree attention kernels");
}

uint64_t tree_workspace_bytes(kq_ctx* ctx, const kq_tree_desc& d) {
  const char* call = "kq_tree_workspace";
  CacheView c;
  Plan p;
  if (!d.cache || cache_view(d.cache, &c) != KQ_OK) {
    fail(KQ_E_INVALID, call, "not a valid cache");
    return 0;
  }
  return plan(ctx, d, c, call, &p) == KQ_OK ? p.most : 0;
}

int attention_tree(kq_ctx* ctx, const kq_tree_desc& d, cudaStream_t s) {
  const char* call = "kq_attention_tree";
  tree::TreeArgs a = {};
  int rc = check_cache(d.cache, call, &a.c);
  if (rc) return rc;
  Plan p;
  rc = plan(ctx, d, a.c, call, &p);
  if (rc) return rc;
  if (d.n_seq == 0 || d.tokens == 0) return KQ_OK;
  if (!d.q || !d.out || !d.starts || !d.prefix || !d.pages || !d.workspace)
    return fail(KQ_E_INVALID, call, "null pointer");
  const uint32_t size = d.type == KQ_TYPE_F32 ? 4 : 2;
  const uint64_t dense = uint64_t(d.n_heads) * a.c.dim;
  a.q_token = d.q_token ? d.q_token : dense;
  a.out_token = d.out_token ? d.out_token : dense;
  if (a.q_token < dense || a.out_token < dense)
    return fail(KQ_E_INVALID, call, "q_token and out_token must be at least n_heads * head_dim");
  if (!on16(d.q) || !on16(d.out) || !on16(a.q_token * size) || !on16(a.out_token * size) || !on16(d.workspace))
    return fail(KQ_E_INVALID, call, "q, out, their token strides and the workspace must be 16-byte aligned");
  if (d.starts % 4 || d.prefix % 4 || d.pages % 4 || d.mask % 8)
    return fail(KQ_E_INVALID, call, "starts, prefix and pages must be 4-byte aligned, mask 8-byte aligned");
  if (d.workspace_bytes < p.bytes)
    return fail(KQ_E_INVALID, call, "workspace of " + std::to_string(d.workspace_bytes) + " bytes; " +
                                        std::to_string(p.bytes) + " needed (kq_tree_workspace)");
  a.q = reinterpret_cast<const void*>(d.q);
  a.out = reinterpret_cast<void*>(d.out);
  a.starts = reinterpret_cast<const int*>(d.starts);
  a.prefix = reinterpret_cast<const int*>(d.prefix);
  a.pages = reinterpret_cast<const int*>(d.pages);
  a.mask = reinterpret_cast<const unsigned long long*>(d.mask);
  a.part = reinterpret_cast<float*>(d.workspace);
  a.splits = reinterpret_cast<uint4*>(d.workspace + p.parts);
  a.scale_log2 = scale_log2(d, a.c);
  a.n_seq = d.n_seq;
  a.n_heads = d.n_heads;
  a.group = d.n_heads / a.c.n_kv;
  a.per_group = a.group == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + a.group - 1) / a.group);
  a.tokens = d.tokens;
  a.max_drafts = d.max_drafts;
  a.max_pages = d.max_pages;
  a.type = d.type;
  a.err = ctx->err;
  const auto launch = a.c.kind == KQ_CACHE_F16  ? tree::launch_kind<KQ_CACHE_F16>
                      : a.c.kind == KQ_CACHE_Q8 ? tree::launch_kind<KQ_CACHE_Q8>
                                                : tree::launch_kind<KQ_CACHE_Q4>;
  cudaError_t e = launch(a, p.split, p.wide, p.ctas, s);
  if (e != cudaSuccess) return cuda_fail(e, "cudaLaunchKernelExC", call);
  if (p.ctas == 1) return KQ_OK;  // nothing is split
  const auto join = p.rows == 8    ? (p.many ? launch_join<8, true> : launch_join<8, false>)
                    : p.rows == 64 ? launch_join<64, false>
                                   : launch_join<128, false>;
  e = join(a, p.ctas, s);
  return e == cudaSuccess ? KQ_OK : cuda_fail(e, "cudaLaunchKernelExC", "tree attention join");
}

}  // namespace kq
