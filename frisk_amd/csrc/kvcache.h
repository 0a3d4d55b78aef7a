// Device side of a cache of keys and values: where a key lies (kv_index.h), and
// the conversions of its 8-bit rows.
#pragma once

#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "kv_index.h"

namespace frisk {
namespace kv {

// (The indexing counts a scale a row for a Cache without this member.)
static_assert(std::is_same<decltype(KvCache::scale_shift), int>::value, "the log2 of the rows that share a scale");

template <Elt C> constexpr float kTop = C == Elt::E4M3 ? 448.0f : 127.0f;

// Eight codes (two words) as f32.
template <Elt C> __device__ __forceinline__ void decode8(i32x2 w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (C == Elt::E4M3) {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false);
      const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
      f[4 * i] = lo[0], f[4 * i + 1] = lo[1], f[4 * i + 2] = hi[0], f[4 * i + 3] = hi[1];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * i + e] = (float)(int8_t)(w[i] >> (8 * e));
    }
  }
}

}  // namespace kv
}  // namespace frisk
