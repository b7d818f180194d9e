// Tree attention over bf16 caches.
#include "attention_tree_wide.cuh"

namespace dyn {

int tree_attention_bf16(const TreeArgs& a, int q_type, cudaStream_t s) { return tree::by_type<TREE_BF16>(a, q_type, s); }

}  // namespace dyn
