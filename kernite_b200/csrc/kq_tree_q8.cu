// kq_tree_q8.cu -- the attention of drafted tokens over caches of kind Q8 (kq_tree.cuh,
// kq_treewide.cuh).
#include "kq_treewide.cuh"

namespace kq {
namespace tree {
KQ_TREE_KIND(KQ_CACHE_Q8)
}  // namespace tree
}  // namespace kq
