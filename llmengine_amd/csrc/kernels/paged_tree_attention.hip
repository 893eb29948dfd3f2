// paged_tree_attention.hip -- the attention of trees of drafted tokens over the paged KV cache.
#include "../paged.hpp"

namespace mle {
constexpr bool kTrees = true;
}

#include "../paged_attention.hpp"

namespace mle {

SplitKNeed paged_tree_attention_workspace(int head_dim, int64_t rows) {
  return workspace_of(head_dim, rows);
}

hipError_t launch_paged_tree_attention(const AttentionArgs& a, const SplitKWorkspace& ws,
                                       hipStream_t stream) {
  return launch_attention(a, ws, stream);
}

}  // namespace mle
