// Attention over a cache, head_dim 32.
#include "attn_tree_mfma.h"

namespace frisk {
hipError_t tree_attn_d32(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s) {
  return tree::tree_mfma_dispatch<32>(a, p, s);
}
}  // namespace frisk
