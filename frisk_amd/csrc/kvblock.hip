// Rows written into an 8-bit cache whose slots share scales in blocks of 2^s.
//
// A workgroup has the rows of one block, head and tensor: it finds the largest of
// the new ones, and with it the block's scale (include/frisk_hip.h states the
// arithmetic, each step of it one f32 operation), and writes their codes; only
// where the scale grows are the codes before them read and written again.  HBM
// bounds it: 4 x 8192 tokens, 8 heads of 128 in int8, 201 MB in 36 us with 32 slots a scale,
// 32 with 128 (part of it from the last-level cache; with the rows read again 51).  A wave for a block of 32
// slots took 39, rows past the L2s as long as through them.

#include "kvcache.h"

namespace frisk {

namespace {

constexpr int kThreads = 256;

// Eight values as two words of codes.
template <Elt C> __device__ __forceinline__ i32x2 round8(const float (&y)[8]) {
  i32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (C == Elt::E4M3) {
      const int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], p, true);
    } else {
      uint32_t p = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) p |= ((uint32_t)(int)__builtin_rintf(y[4 * i + j]) & 255u) << (8 * j);
      w[i] = (int)p;
    }
  }
  return w;
}

template <Elt T> __device__ __forceinline__ float value_of(i32x4 x, int i) {
  const uint16_t h = (uint16_t)((uint32_t)x[i / 2] >> (16 * (i & 1)));
  return T == Elt::BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
}

// Workgroups in the order (sequence, block, head, k or v).  A block is at most
// HOLD pieces of 8 values a thread, which stay in registers between the passes (0: they are
// read again).
template <Elt T, Elt C, int HOLD>
__global__ __launch_bounds__(kThreads, 4) void kv_block_kernel(KvArgs a, int g, int blocks) {
  constexpr float Q = kv::kTop<C>;
  const KvCache& c = a.cache;
  const int shift = c.scale_shift, size = 1 << shift;
  uint32_t id = blockIdx.x;
  const bool of_v = id & 1;
  id >>= 1;
  const int h = id % c.kv_heads;
  id /= c.kv_heads;
  const int block = id % blocks;
  const int64_t b = id / blocks;
  const kv::Span sp = kv::span_of(a.ctx_len, a.new_len, (int)a.tokens, b);
  if (sp.ctx < 0) return;
  // Keys first .. first + size - 1, of which lo .. hi - 1 are new.
  const int64_t first = ((sp.ctx >> shift) + block) << shift;
  const int64_t lo = first > sp.ctx ? first : sp.ctx;
  int64_t hi = sp.ctx + sp.fresh;
  hi = hi < first + size ? hi : first + size;
  hi = hi < c.capacity ? hi : c.capacity;
  if (lo >= hi) return;
  const int old = (int)(lo - first), end = (int)(hi - first);

  const int sub = threadIdx.x & ((1 << g) - 1), row0 = threadIdx.x >> g, rows = kThreads >> g;
  const bool in = sub * 8 < c.head_dim;
  const uint16_t* x = (const uint16_t*)(of_v ? a.v : a.k) + b * (of_v ? a.vsb : a.ksb) + h * (of_v ? a.vsh : a.ksh) +
                      (first - sp.ctx) * (of_v ? a.vss : a.kss) + sub * 8;
  const int64_t xs = of_v ? a.vss : a.kss;
  // (The new rows' loads are under way while the page is looked up.)
  i32x4 held[HOLD ? HOLD : 1];
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      const int r = row0 + i * rows;
      held[i] = i32x4{0, 0, 0, 0};
      if (in && r >= old && r < end) held[i] = *(const i32x4*)(x + r * xs);
    }
  }
  const kv::Slot at = kv::slot_of(c, b, first);
  if (at.elem < 0) return;
  char* codes = (char*)(of_v ? c.v : c.k) + at.elem + h * c.sh + sub * 8;
  float* scale_at = (of_v ? c.v_scale : c.k_scale) + at.scale + h * c.sch;
  __shared__ uint32_t tops[kThreads / 64];
  __shared__ float before;
  if (threadIdx.x == 0) before = old ? *scale_at : 0.0f;

  // Magnitudes compare as integers, NaN above infinity.
  uint32_t top = 0;
  auto larger = [&](i32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = (uint32_t)v[i] & 0x7fff7fffu;
      top = max(top, max(w & 0xffffu, w >> 16));
    }
  };
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) larger(held[i]);
  } else {
    for (int r = row0; r < end; r += rows)
      if (in && r >= old) larger(*(const i32x4*)(x + r * xs));
  }
  for (int m = 1; m < 64; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) top = max(top, tops[w]);
  const float was = before;

  const float largest = T == Elt::BF16 ? bf16_bits_to_f32((uint16_t)top)
                                       : (float)__builtin_bit_cast(_Float16, (uint16_t)top);
  const bool finite = top < (T == Elt::BF16 ? 0x7f80u : 0x7c00u) && was == was;
  float scale = finite ? fmaxf(largest, Q * 0x1p-126f) / Q : __builtin_nanf("");
  const bool grown = old && scale > was;
  if (finite && old && !grown) scale = was;
  const float inv = finite ? 1.0f / scale : 0.0f;
  auto put = [&](int r, i32x4 v) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = finite ? value_of<T>(v, i) * inv : 0.0f;
    *(i32x2*)(codes + r * c.ss) = round8<C>(y);
  };
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      const int r = row0 + i * rows;
      // (Widened here: all f16 pieces at once took 233 registers.)
      asm volatile("" : "+v"(held[i]));
      if (in && r >= old && r < end) put(r, held[i]);
    }
  } else {
    for (int r = row0; r < end; r += rows)
      if (in && r >= old) put(r, *(const i32x4*)(x + r * xs));
  }
  if (grown) {
    const float ratio = was * inv;
    for (int r = row0; r < old; r += rows) {
      if (!in) continue;
      float f[8];
      kv::decode8<C>(*(const i32x2*)(codes + r * c.ss), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= ratio;
      *(i32x2*)(codes + r * c.ss) = round8<C>(f);
    }
  }
  if (threadIdx.x == 0) *scale_at = scale;
}

template <Elt T, Elt C> hipError_t launch_blocks(const KvArgs& a, hipStream_t stream) {
  int g = 0;
  while ((8 << g) < a.cache.head_dim) ++g;
  const int64_t size = 1ll << a.cache.scale_shift;
  const int64_t blocks = (a.tokens + size - 2) / size + 1;  // that a sequence may touch
  if (blocks > INT32_MAX / 2) return hipErrorInvalidConfiguration;
  const int64_t per = 2 * (int64_t)a.cache.kv_heads * blocks;
  if (a.batch > (int64_t)(UINT32_MAX / kThreads) / per) return hipErrorInvalidConfiguration;
  const int64_t pieces = (size + (kThreads >> g) - 1) / (kThreads >> g);
  auto kern = pieces <= 1 ? kv_block_kernel<T, C, 1> : pieces <= 2 ? kv_block_kernel<T, C, 2>
            : pieces <= 4 ? kv_block_kernel<T, C, 4> : pieces <= 8 ? kv_block_kernel<T, C, 8>
                                                                   : kv_block_kernel<T, C, 0>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.batch * per)), dim3(kThreads), 0, stream, a, g, (int)blocks);
  return hipGetLastError();
}

}  // namespace

hipError_t kv_append_blocks(const KvArgs& a, hipStream_t s) {
  const bool bf = a.dtype == Elt::BF16;
  if (a.cache.kind == Elt::E4M3)
    return bf ? launch_blocks<Elt::BF16, Elt::E4M3>(a, s) : launch_blocks<Elt::F16, Elt::E4M3>(a, s);
  return bf ? launch_blocks<Elt::BF16, Elt::I8>(a, s) : launch_blocks<Elt::F16, Elt::I8>(a, s);
}

}  // namespace frisk
