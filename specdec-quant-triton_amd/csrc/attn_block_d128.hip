// Instantiations of paged attention over block-scaled int8 / e4m3 caches, head dim 128: the eager
// launches (1 to 4 row blocks) and the plan-mode launches (runtime row blocks, 2 to 4), and the merge of many splits.
#include "paged_attn.hpp"

namespace specq {

const void* attn_block_fn_d128(int rb, int f8, int plan) {
  switch ((plan ? 8 : 0) + 2 * (rb - 1) + f8) {
    case 0: return reinterpret_cast<const void*>(&paged_attn_kernel<128, 1, BlockI8>);
    case 1: return reinterpret_cast<const void*>(&paged_attn_kernel<128, 1, BlockF8>);
    case 2: return reinterpret_cast<const void*>(&paged_attn_kernel<128, 2, BlockI8>);
    case 3: return reinterpret_cast<const void*>(&paged_attn_kernel<128, 2, BlockF8>);
    case 4: return reinterpret_cast<const void*>(&paged_attn_kernel<128, 3, BlockI8>);
    case 5: return reinterpret_cast<const void*>(&paged_attn_kernel<128, 3, BlockF8>);
    case 6: return reinterpret_cast<const void*>(&paged_attn_kernel<128, 4, BlockI8>);
    case 7: return reinterpret_cast<const void*>(&paged_attn_kernel<128, 4, BlockF8>);
    case 10: return reinterpret_cast<const void*>(&paged_attn_plan_kernel<128, 2, BlockI8>);
    case 11: return reinterpret_cast<const void*>(&paged_attn_plan_kernel<128, 2, BlockF8>);
    case 12: return reinterpret_cast<const void*>(&paged_attn_plan_kernel<128, 3, BlockI8>);
    case 13: return reinterpret_cast<const void*>(&paged_attn_plan_kernel<128, 3, BlockF8>);
    case 14: return reinterpret_cast<const void*>(&paged_attn_plan_kernel<128, 4, BlockI8>);
    case 15: return reinterpret_cast<const void*>(&paged_attn_plan_kernel<128, 4, BlockF8>);
  }
  return nullptr;
}

const void* attn_merge_fn_d128() { return reinterpret_cast<const void*>(&attn_merge_kernel<128>); }

}  // namespace specq
