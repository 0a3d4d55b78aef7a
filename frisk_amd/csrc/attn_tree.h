// Attention of new tokens over a cache of keys and values: what its kernels
// share (attn_tree_rows.hip, attn_tree_mfma.h).
#pragma once

#include "kvcache.h"

namespace frisk {
namespace tree {

constexpr int kBlock = plan::kTreeBlock;  // keys per block
constexpr float kLog2eF = 1.4426950408889634f;
constexpr float kLn2F = 0.6931471805599453f;

// The rows of a launch with several key splits: O (f32, not divided by l),
// then m (exp2 domain) and l, for row (b * heads + h) * tokens + t.
struct Part {
  float* o;   // [rows][splits][head_dim]
  float* ml;  // [rows][splits][2]
  int splits;
  int min_blocks;  // a split has at least so many blocks
  // The Keys kernel, which sums its splits itself, lays o out by tiles of rows
  // (keys_part) and has a word for each behind them.
  unsigned long long* words;
};

__device__ __forceinline__ int blocks_per_split(const Part& p, int blocks) {
  return blocks_per_split(p.splits, p.min_blocks, blocks);
}

// Whether new token t sees draft j.
__device__ __forceinline__ bool sees(const TreeAttnArgs& a, int64_t b, int t, int j) {
  if (!a.mask) return j <= t;
  return (a.mask[b * a.mask_sb + t * a.mask_st + (j >> 6)] >> (j & 63)) & 1;
}

__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
// Natural-log sum from the exp2-domain maximum and the sum.
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.0f ? -__builtin_inff() : (m + __log2f(l)) * kLn2F;
}

template <Elt T> __device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (T == Elt::BF16) {
    return f32x2_to_bf16x2_bits(lo, hi);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
}

// Four dims of an output row, in Q's type or f32.
template <Elt T>
__device__ __forceinline__ void store4(const TreeAttnArgs& a, int64_t at, f32x4 v) {
  if (a.out == Elt::F32) *(f32x4*)((float*)a.o + at) = v;
  else *(i32x2*)((uint16_t*)a.o + at) = i32x2{(int)pack16<T>(v[0], v[1]), (int)pack16<T>(v[2], v[3])};
}

}  // namespace tree

// The matrix-core kernels of one head_dim (attn_tree_d*.hip).
hipError_t tree_attn_d32(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s);
hipError_t tree_attn_d64(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s);
hipError_t tree_attn_d128(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s);
// The launches of attn_tree_rows.hip: any head_dim, and the sum over splits.
hipError_t tree_attn_rows(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s);
hipError_t tree_attn_sum(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s);

}  // namespace frisk
