// Attention over a cache, head_dim 128.
#include "attn_tree_mfma.h"

namespace frisk {
hipError_t tree_attn_d128(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s) {
  return tree::tree_mfma_dispatch<128>(a, p, s);
}
}  // namespace frisk
