// Device side of a cache of keys and values: where a key lies, and the
// conversions of its 8-bit rows.
#pragma once

#include "common.h"
#include "kernels.h"

namespace frisk {
namespace kv {

// Element and scale offsets of one key's row of head 0; elem < 0: the cache
// does not hold the key.
struct Slot {
  int64_t elem, scale;
};
// The page of key n of sequence b, or -1.
__device__ __forceinline__ int page_of(const KvCache& c, int64_t b, int64_t n) {
  if (n < 0 || n >= c.capacity) return -1;
  int64_t page = b;
  if (c.table) page = c.table[b * c.table_stride + (n >> c.page_shift)];
  return page >= 0 && page < c.pages ? (int)page : -1;
}
__device__ __forceinline__ Slot slot_of(const KvCache& c, int64_t b, int64_t n) {
  const int page = page_of(c, b, n);
  if (page < 0) return {-1, -1};
  const int64_t row = c.table ? n & ((1ll << c.page_shift) - 1) : n;
  return {page * c.sp + row * c.ss, page * c.scp + row * c.scs};
}

// Keys before the call and new tokens of sequence b; ctx < 0: none of its work.
struct Span {
  int64_t ctx;
  int fresh;
};
__device__ __forceinline__ Span span_of(const int32_t* ctx_len, const int32_t* new_len, int tokens,
                                        int64_t b) {
  const int n = new_len ? min(max(new_len[b], 0), tokens) : tokens;
  return {ctx_len[b], n};
}

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
