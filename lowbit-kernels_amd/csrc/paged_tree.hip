// Attention of trees of drafted tokens over a paged KV cache (attention_paged_tree): the kernel of paged_attention.hpp, whose rows
// attend every key before their sequence's new tokens and those of the new tokens that their mask names.
#include "paged_attention.hpp"

namespace lowbit {

size_t attention_paged_tree_workspace(const PagedAttentionArgs& a) {
  const PagedLaunch l = tree_launch(a);
  return l.cap == 1 ? 0 : (l.units + 1) * sizeof(PagedTile) + l.records * paged_record_bytes(l.rg, a.D);
}

hipError_t attention_paged_tree_launch(const PagedAttentionArgs& a, hipStream_t st) {
  if (a.bf16) return a.D == 64 ? pick_tree_attention<bf16, 64>(a, st) : pick_tree_attention<bf16, 128>(a, st);
  return a.D == 64 ? pick_tree_attention<f16, 64>(a, st) : pick_tree_attention<f16, 128>(a, st);
}

}  // namespace lowbit
