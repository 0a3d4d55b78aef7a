// Attention over a cache, head_dim 64.
#include "attn_tree_mfma.h"

namespace frisk {
hipError_t tree_attn_d64(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s) {
  return tree::tree_mfma_dispatch<64>(a, p, s);
}
}  // namespace frisk
