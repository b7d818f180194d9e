// Tree attention over e4m3 caches.
#include "attention_tree_wide.cuh"

namespace dyn {

int tree_attention_e4m3(const TreeArgs& a, int q_type, cudaStream_t s) { return tree::by_type<TREE_E4M3>(a, q_type, s); }

}  // namespace dyn
