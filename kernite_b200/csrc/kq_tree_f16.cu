// kq_tree_f16.cu -- the attention of drafted tokens over caches of kind F16 (kq_tree.cuh,
// kq_treewide.cuh).
#include "kq_treewide.cuh"

namespace kq {
namespace tree {
KQ_TREE_KIND(KQ_CACHE_F16)
}  // namespace tree
}  // namespace kq
