// Attention of new tokens over a cache, one query row per workgroup, for head
// dims that have no matrix-core kernel (attn_tree_mfma.h); and the sum over key
// splits of either.
//
// Eight lanes take a key, 8 dims (16 B, or 8 B of codes) at a time, so a wave
// has 8 keys and a workgroup 32 streams of keys, each with a running maximum,
// sum and output row of its own that meet once at the end.  A hidden key is not
// loaded.  Vector instructions bound it: each key's row is read and converted
// for one query row only.

#include "attn_tree.h"

namespace frisk {

namespace {

template <Elt E> __device__ __forceinline__ void load8(const void* base, int64_t at, float (&f)[8]) {
  if constexpr (E == Elt::E4M3 || E == Elt::I8) {
    kv::decode8<E>(*(const i32x2*)((const char*)base + at), f);
  } else {
    const i32x4 w = *(const i32x4*)((const uint16_t*)base + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t h = (uint16_t)((uint32_t)w[i / 2] >> (16 * (i & 1)));
      f[i] = E == Elt::BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
    }
  }
}

// NP pieces of 64 dims.
template <Elt T, Elt C, int NP>
__global__ __launch_bounds__(256) void tree_rows_kernel(TreeAttnArgs a, tree::Part part) {
  constexpr bool k8 = C == Elt::E4M3 || C == Elt::I8;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, sub = lane & 7, D = a.cache.head_dim;
  const int64_t row = blockIdx.x;
  const int t = (int)((uint64_t)row % (uint32_t)a.tokens);
  const int64_t bh = (uint64_t)row / (uint32_t)a.tokens;
  const int64_t b = (uint64_t)bh / (uint32_t)a.heads;
  const int h = (int)(bh - b * a.heads), kvh = h / (a.heads / a.cache.kv_heads);
  const kv::Span sp = kv::span_of(a.ctx_len, a.new_len, a.tokens, b);
  if (sp.ctx < 0 || t >= sp.fresh) return;
  const int keys = tree::keys_of(a.cache.capacity, sp), blocks = (keys + tree::kBlock - 1) / tree::kBlock;
  const int per = tree::blocks_per_split(part, blocks), split = blockIdx.y;
  if (split > 0 && split * per >= blocks) return;
  const int end = min(keys, (split + 1) * per * tree::kBlock);

  float q[NP][8], o[NP][8], m = -__builtin_inff(), l = 0.0f;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[p][i] = o[p][i] = 0.0f;
    const int d = p * 64 + sub * 8;
    if (d < D) load8<T>(a.q, b * a.q_sb + h * a.q_sh + t * a.q_ss + d, q[p]);
  }
  const float scale = a.sm_scale * tree::kLog2eF;
  for (int n = split * per * tree::kBlock + wave * 8 + (lane >> 3); n < end; n += 32) {
    if (n >= sp.ctx && !tree::sees(a, b, t, (int)(n - sp.ctx))) continue;
    const kv::Slot at = kv::slot_of(a.cache, b, n);
    if (at.elem < 0) continue;
    const int64_t e = at.elem + kvh * a.cache.sh;
    float s = 0.0f, f[8];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int d = p * 64 + sub * 8;
      if (d >= D) continue;
      load8<C>(a.cache.k, e + d, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = __builtin_fmaf(q[p][i], f[i], s);
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    s += __shfl_xor(s, 4);
    float vs = 1.0f;
    if constexpr (k8) {
      const int64_t sc = at.scale + kvh * a.cache.sch;
      s *= a.cache.k_scale[sc];
      vs = a.cache.v_scale[sc];
    }
    s *= scale;
    const float mn = fmaxf(m, s), nm = mn == -__builtin_inff() ? 0.0f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - nm), w = __builtin_amdgcn_exp2f(s - nm);
    m = mn;
    l = __builtin_fmaf(l, alpha, w);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int d = p * 64 + sub * 8;
      if (d >= D) continue;
      load8<C>(a.cache.v, e + d, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[p][i] = __builtin_fmaf(w * vs, f[i], o[p][i] * alpha);
    }
  }

  // The 8 streams of a wave, then the waves.
  __shared__ float wm[4], wl[4];
  __shared__ __attribute__((aligned(16))) float wo[4][NP * 64];
  float M = m;
#pragma unroll
  for (int x = 8; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
  const float nM = M == -__builtin_inff() ? 0.0f : M;
  const float f = __builtin_amdgcn_exp2f(m - nM);
  l *= f;
#pragma unroll
  for (int x = 8; x < 64; x <<= 1) l += __shfl_xor(l, x);
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = o[p][i] * f;
#pragma unroll
      for (int x = 8; x < 64; x <<= 1) v += __shfl_xor(v, x);
      if (lane < 8) wo[wave][p * 64 + sub * 8 + i] = v;
    }
  if (lane == 0) wm[wave] = M, wl[wave] = l;
  __syncthreads();
  const int d = threadIdx.x * 4;
  if (d >= D) return;
  float top = -__builtin_inff(), L = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, wm[w]);
  const float ntop = top == -__builtin_inff() ? 0.0f : top;
  f32x4 acc = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float g = __builtin_amdgcn_exp2f(wm[w] - ntop);
    L = __builtin_fmaf(wl[w], g, L);
    acc += *(const f32x4*)&wo[w][d] * g;
  }
  if (per < blocks) {  // more than one split of this sequence
    const int64_t r = row * part.splits + split;
    *(f32x4*)(part.o + r * D + d) = acc;
    if (d == 0) part.ml[2 * r] = top, part.ml[2 * r + 1] = L;
    return;
  }
  tree::store4<T>(a, b * a.o_sb + h * a.o_sh + t * a.o_ss + d, acc * tree::inverse_sum(L));
  if (a.lse && d == 0) a.lse[row] = tree::lse_of(top, L);
}

// One lane per 4 dims of a row whose sequence has several splits, summed in
// split order.
template <Elt T>
__global__ __launch_bounds__(256) void tree_sum_kernel(TreeAttnArgs a, tree::Part part, int64_t rows) {
  const int D = a.cache.head_dim, lanes = D / 4;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = (uint64_t)idx / (uint32_t)lanes;
  if (row >= rows) return;
  const int d = (int)(idx - row * lanes) * 4;
  const int t = (int)((uint64_t)row % (uint32_t)a.tokens);
  const int64_t bh = (uint64_t)row / (uint32_t)a.tokens;
  const int64_t b = (uint64_t)bh / (uint32_t)a.heads;
  const int h = (int)(bh - b * a.heads);
  const kv::Span sp = kv::span_of(a.ctx_len, a.new_len, a.tokens, b);
  if (sp.ctx < 0 || t >= sp.fresh) return;
  const int blocks = (tree::keys_of(a.cache.capacity, sp) + tree::kBlock - 1) / tree::kBlock;
  const int per = tree::blocks_per_split(part, blocks);
  if (per >= blocks) return;  // written by its workgroup
  const int n = (blocks + per - 1) / per;
  const float* ml = part.ml + row * part.splits * 2;
  float M = -__builtin_inff(), L = 0.0f;
  for (int s = 0; s < n; ++s) M = fmaxf(M, ml[2 * s]);
  const float nM = M == -__builtin_inff() ? 0.0f : M;
  f32x4 acc = {0, 0, 0, 0};
  for (int s = 0; s < n; ++s) {
    if (ml[2 * s + 1] == 0.0f) continue;  // no key of the split is seen
    const float g = __builtin_amdgcn_exp2f(ml[2 * s] - nM);
    L = __builtin_fmaf(ml[2 * s + 1], g, L);
    acc += *(const f32x4*)(part.o + (row * part.splits + s) * D + d) * g;
  }
  tree::store4<T>(a, b * a.o_sb + h * a.o_sh + t * a.o_ss + d, acc * tree::inverse_sum(L));
  if (a.lse && d == 0) a.lse[row] = tree::lse_of(M, L);
}

template <Elt T, Elt C> hipError_t rows_kind(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s) {
  const int64_t rows = a.batch * a.heads * a.tokens;
  if (rows > UINT32_MAX / 256) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)rows, (unsigned)p.splits);
  const int D = a.cache.head_dim;
  if (D <= 64) hipLaunchKernelGGL((tree_rows_kernel<T, C, 1>), grid, dim3(256), 0, s, a, p);
  else if (D <= 128) hipLaunchKernelGGL((tree_rows_kernel<T, C, 2>), grid, dim3(256), 0, s, a, p);
  else hipLaunchKernelGGL((tree_rows_kernel<T, C, 4>), grid, dim3(256), 0, s, a, p);
  return hipGetLastError();
}

template <Elt T> hipError_t rows_type(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s) {
  switch (a.cache.kind) {
    case Elt::E4M3: return rows_kind<T, Elt::E4M3>(a, p, s);
    case Elt::I8: return rows_kind<T, Elt::I8>(a, p, s);
    default: return rows_kind<T, T>(a, p, s);
  }
}

}  // namespace

hipError_t tree_attn_rows(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s) {
  return a.dtype == Elt::BF16 ? rows_type<Elt::BF16>(a, p, s) : rows_type<Elt::F16>(a, p, s);
}

hipError_t tree_attn_sum(const TreeAttnArgs& a, const tree::Part& p, hipStream_t s) {
  const int64_t rows = a.batch * a.heads * a.tokens, threads = rows * (a.cache.head_dim / 4);
  if (threads > (int64_t)(UINT32_MAX / 256) * 256) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)((threads + 255) / 256));
  if (a.dtype == Elt::BF16) hipLaunchKernelGGL(tree_sum_kernel<Elt::BF16>, grid, dim3(256), 0, s, a, p, rows);
  else hipLaunchKernelGGL(tree_sum_kernel<Elt::F16>, grid, dim3(256), 0, s, a, p, rows);
  return hipGetLastError();
}

hipError_t tree_attn(const TreeAttnArgs& a, hipStream_t s) {
  tree::Part p{nullptr, nullptr, a.splits, a.min_blocks, nullptr};
  const bool keys = a.kernel == plan::TreeKernel::Keys;
  if (a.splits > 1) {
    p.o = (float*)a.workspace;
    if (keys) {
      const int64_t tiles = plan::tree_key_tiles(a.batch, a.heads, a.cache.kv_heads, a.tokens);
      p.words = (unsigned long long*)(p.o + tiles * a.splits * 32 * (a.cache.head_dim + 2));
    } else {
      p.ml = p.o + a.batch * a.heads * a.tokens * a.splits * a.cache.head_dim;
    }
  }
  hipError_t e;
  switch (a.kernel == plan::TreeKernel::Rows ? 0 : a.cache.head_dim) {
    case 32: e = tree_attn_d32(a, p, s); break;
    case 64: e = tree_attn_d64(a, p, s); break;
    case 128: e = tree_attn_d128(a, p, s); break;
    default: e = tree_attn_rows(a, p, s);
  }
  if (e != hipSuccess || a.splits <= 1 || keys) return e;
  return tree_attn_sum(a, p, s);
}

}  // namespace frisk
