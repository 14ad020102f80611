// Instantiations of paged attention over block-scaled int8 / e4m3 caches, head dim 64: the eager
// launches (1 to 4 row blocks) and the plan-mode launches (runtime row blocks, 2 to 4), and the merge of many splits.
#include "paged_attn_block.hpp"

namespace specq {

const void* attn_block_fn_d64(int rb, int f8, int plan) {
  switch ((plan ? 8 : 0) + 2 * (rb - 1) + f8) {
    case 0: return reinterpret_cast<const void*>(&attn_block_kernel<64, 1, false>);
    case 1: return reinterpret_cast<const void*>(&attn_block_kernel<64, 1, true>);
    case 2: return reinterpret_cast<const void*>(&attn_block_kernel<64, 2, false>);
    case 3: return reinterpret_cast<const void*>(&attn_block_kernel<64, 2, true>);
    case 4: return reinterpret_cast<const void*>(&attn_block_kernel<64, 3, false>);
    case 5: return reinterpret_cast<const void*>(&attn_block_kernel<64, 3, true>);
    case 6: return reinterpret_cast<const void*>(&attn_block_kernel<64, 4, false>);
    case 7: return reinterpret_cast<const void*>(&attn_block_kernel<64, 4, true>);
    case 10: return reinterpret_cast<const void*>(&attn_block_plan_kernel<64, 2, false>);
    case 11: return reinterpret_cast<const void*>(&attn_block_plan_kernel<64, 2, true>);
    case 12: return reinterpret_cast<const void*>(&attn_block_plan_kernel<64, 3, false>);
    case 13: return reinterpret_cast<const void*>(&attn_block_plan_kernel<64, 3, true>);
    case 14: return reinterpret_cast<const void*>(&attn_block_plan_kernel<64, 4, false>);
    case 15: return reinterpret_cast<const void*>(&attn_block_plan_kernel<64, 4, true>);
  }
  return nullptr;
}

const void* attn_merge_fn_d64() { return reinterpret_cast<const void*>(&attn_merge_kernel<64>); }

}  // namespace specq
