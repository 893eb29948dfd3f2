// paged_attention.hip -- the attention of runs of new tokens over the paged KV cache.
#include "../paged.hpp"

namespace mle {
constexpr bool kTrees = false;
}

#include "../paged_attention.hpp"

namespace mle {

SplitKNeed paged_attention_workspace(int head_dim, int64_t rows) {
  return workspace_of(head_dim, rows);
}

hipError_t launch_paged_attention(const AttentionArgs& a, const SplitKWorkspace& ws,
                                  hipStream_t stream) {
  return launch_attention(a, ws, stream);
}

}  // namespace mle
