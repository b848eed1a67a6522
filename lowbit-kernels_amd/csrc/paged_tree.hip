// Attention of trees of drafted tokens over a paged KV cache (attention_paged_tree): the kernel of paged_attention.hpp, whose rows
// attend every key before their sequence's new tokens and those of the new tokens that their mask names.
#include "paged_attention.hpp"

namespace lowbit {

hipError_t attention_paged_tree_launch(const PagedAttentionArgs& a, hipStream_t st) {
  if (a.bf16) return a.D == 64 ? pick_paged_attention<bf16, 64, true>(a, st) : pick_paged_attention<bf16, 128, true>(a, st);
  return a.D == 64 ? pick_paged_attention<f16, 64, true>(a, st) : pick_paged_attention<f16, 128, true>(a, st);
}

}  // namespace lowbit
