// Tree attention over q8 caches.
#include "attention_tree_wide.cuh"

namespace dyn {

int tree_attention_q8(const TreeArgs& a, int q_type, cudaStream_t s) { return tree::by_type<TREE_Q8>(a, q_type, s); }

}  // namespace dyn
