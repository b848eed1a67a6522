// Attention of trees of drafted tokens over a paged KV cache (attention_paged_tree): the kernel of paged_attention.hpp, whose rows
// attend every key before their sequence's new tokens and those of the new tokens that their mask names.
// Bound: 16 trees of 31 .. 63 nodes on 300 .. 8000 keys, 28 / 4 heads of 128, 20 GFLOP, 73 MB, 48.7 us, 0.42 PFLOP/s; 2 of 36 on
// 15000 38.5; of 0.2 GFLOP and 1 MB (a tree of 26 on 926, 16 / 2 heads) 13.8. Neither memory (with all keys in the caches 8% less)
// nor a unit: the matrix cores are busy a quarter of the time, the vector unit 28%, and waves wait 38% of it. What counts is a
// wave's chain from a block's scores over its weights to its products, 1.1 us a block with two workgroups a CU (0.76 with one),
// what a call takes beside its blocks, 11 .. 15 us, and the split of the keys, whose records (34 MB) take 5 us to write and 7 to
// join. Measured and not kept: tiles of 64 rows; eight waves on 128 rows and two key groups (16 trees 72 us for then 61); records
// through LDS; a last, shorter part (2 trees on 30000 .. 60000 74 -> 81).
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
