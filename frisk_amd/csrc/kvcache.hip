// A cache of keys and values written in 16 or 8 bits and read back, and the
// masks of drafted trees.
//
// A row of head_dim values is taken by 2^g lanes of 8 values (16 B) each, for
// k and v together, so a wave has two 16-B loads a lane in flight and its row
// maximum is g exchanges between neighbouring lanes.  HBM bounds both ways.  Rows
// beyond the L2s' 32 MB go past them (read once; and written back at the
// kernel's end otherwise): 4 x 8192 tokens, 8 heads of 128 in e4m3 written and
// read back, 84 -> 75 us.
//
// The code of x is x Q / a rounded to nearest even (a the row's largest
// magnitude, Q the type's), as a correctly rounded quotient would give it:
// with a scaled to [1/2, 1) by a power of two and x by the same, t = x Q has
// at most 18 significant bits and is exact; y0 = t rcp(a) is within 2^-22 of
// the quotient and one step y0 + rcp(a) (t - y0 a), its residual exact in
// fused multiply-adds, makes a representable quotient exact, which the ties of
// the rounding to codes all are (5 or 8 bits), and keeps every other one on
// its side of the ties: |t - m a| for a tie m is at least 2^-19 of t there.

#include "kvcache.h"

namespace frisk {

namespace {

using kv::Slot;
using kv::Span;

// Scale and codes of one row; the row's lanes are the 2^g neighbours.
template <Elt T, Elt C>
__device__ __forceinline__ i32x2 encode8(i32x4 x, int g, float& scale) {
  constexpr float Q = kv::kTop<C>;
  // Magnitudes compare as integers, NaN above infinity.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (uint32_t)x[i] & 0x7fff7fffu;
    top = max(top, max(w & 0xffffu, w >> 16));
  }
  for (int m = 1; m < 1 << g; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
  const bool finite = top < (T == Elt::BF16 ? 0x7f80u : 0x7c00u);
  const float largest = T == Elt::BF16 ? bf16_bits_to_f32((uint16_t)top)
                                       : (float)__builtin_bit_cast(_Float16, (uint16_t)top);
  const float a = fmaxf(finite ? largest : 0.0f, Q * 0x1p-126f);
  scale = finite ? a / Q : __builtin_nanf("");
  const int e = __builtin_amdgcn_frexp_expf(a);
  const float an = __builtin_ldexpf(a, -e), c = __builtin_ldexpf(Q, -e);
  const float r = __builtin_amdgcn_rcpf(an);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t h = (uint16_t)((uint32_t)x[i / 2] >> (16 * (i & 1)));
    const float v = T == Elt::BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
    const float t = finite ? v * c : 0.0f;
    const float y0 = t * r;
    y[i] = __builtin_fmaf(__builtin_fmaf(-y0, an, t), r, y0);
  }
  i32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (C == Elt::E4M3) {
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], p, true);
    } else {
      uint32_t p = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p |= ((uint32_t)(int)__builtin_rintf(y[4 * i + j]) & 255u) << (8 * j);
      w[i] = (int)p;
    }
  }
  return w;
}

template <Elt T, Elt C> __device__ __forceinline__ i32x4 back8(i32x2 w, float scale) {
  float f[8];
  kv::decode8<C>(w, f);
  uint32_t p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = f[2 * i] * scale, hi = f[2 * i + 1] * scale;
    if constexpr (T == Elt::BF16) {
      p[i] = f32x2_to_bf16x2_bits(lo, hi);
    } else {
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      const h2 v = {(_Float16)lo, (_Float16)hi};
      p[i] = __builtin_bit_cast(uint32_t, v);
    }
  }
  return i32x4{(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
}

// Rows in the order (b, head, token), tokens fastest, where the cache's slots
// and its scales are next to each other.
template <Elt T, Elt C, bool WRITE, bool PAST_L2>
__global__ __launch_bounds__(256) void kv_kernel(KvArgs a, int g, int64_t rows) {
  constexpr bool k8 = C == Elt::E4M3 || C == Elt::I8;
  const int lane = threadIdx.x & ((1 << g) - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 >> g) + (threadIdx.x >> g);
  if (row >= rows) return;
  const int tokens = (int)a.tokens;
  const int64_t bh = (uint64_t)row / (uint32_t)tokens;
  const int t = (int)(row - bh * tokens);
  const int64_t b = (uint64_t)bh / (uint32_t)a.cache.kv_heads;
  const int h = (int)(bh - b * a.cache.kv_heads);
  const Span sp = kv::span_of(a.ctx_len, a.new_len, tokens, b);
  if (sp.ctx < 0 || t >= sp.fresh) return;
  const Slot at = kv::slot_of(a.cache, b, sp.ctx + t);
  if (at.elem < 0) return;
  const bool in = lane * 8 < a.cache.head_dim;
  uint16_t* kx = (uint16_t*)a.k + (b * a.ksb + h * a.ksh + t * a.kss + lane * 8);
  uint16_t* vx = (uint16_t*)a.v + (b * a.vsb + h * a.vsh + t * a.vss + lane * 8);
  const int64_t e = at.elem + h * a.cache.sh + lane * 8;
  const int64_t sc = at.scale + h * a.cache.sch;
  auto load = [&](const uint16_t* p) {
    if constexpr (PAST_L2) return __builtin_nontemporal_load((const i32x4*)p);
    else return *(const i32x4*)p;
  };
  auto store = [&](uint16_t* p, i32x4 v) {
    if constexpr (PAST_L2) __builtin_nontemporal_store(v, (i32x4*)p);
    else *(i32x4*)p = v;
  };
  if constexpr (!k8) {
    uint16_t* ck = (uint16_t*)a.cache.k + e;
    uint16_t* cv = (uint16_t*)a.cache.v + e;
    if (!in) return;
    const i32x4 kw = load(WRITE ? kx : ck), vw = load(WRITE ? vx : cv);
    store(WRITE ? ck : kx, kw);
    store(WRITE ? cv : vx, vw);
  } else {
    char* ck = (char*)a.cache.k + e;
    char* cv = (char*)a.cache.v + e;
    if constexpr (WRITE) {
      i32x4 kw = {0, 0, 0, 0}, vw = {0, 0, 0, 0};
      if (in) kw = load(kx), vw = load(vx);
      float ks, vs;
      const i32x2 kc = encode8<T, C>(kw, g, ks), vc = encode8<T, C>(vw, g, vs);
      if (in) *(i32x2*)ck = kc, *(i32x2*)cv = vc;
      if (lane == 0) a.cache.k_scale[sc] = ks, a.cache.v_scale[sc] = vs;
    } else {
      if (!in) return;
      const i32x2 kc = *(const i32x2*)ck, vc = *(const i32x2*)cv;
      const float ks = a.cache.k_scale[sc], vs = a.cache.v_scale[sc];
      store(kx, back8<T, C>(kc, ks));
      store(vx, back8<T, C>(vc, vs));
    }
  }
}

template <Elt T, Elt C, bool WRITE> hipError_t launch_kv(const KvArgs& a, hipStream_t stream) {
  int g = 0;
  while ((8 << g) < a.cache.head_dim) ++g;
  const int64_t rows = a.batch * a.cache.kv_heads * a.tokens;
  const int64_t blocks = (rows + (256 >> g) - 1) / (256 >> g);
  if (blocks > UINT32_MAX / 256) return hipErrorInvalidConfiguration;
  const bool past_l2 = rows * a.cache.head_dim * 4 > (32ll << 20);
  auto kern = past_l2 ? kv_kernel<T, C, WRITE, true> : kv_kernel<T, C, WRITE, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, a, g, rows);
  return hipGetLastError();
}

template <bool WRITE> hipError_t kv_dispatch(const KvArgs& a, hipStream_t s) {
  const bool bf = a.dtype == Elt::BF16;
  switch (a.cache.kind) {
    case Elt::E4M3:
      return bf ? launch_kv<Elt::BF16, Elt::E4M3, WRITE>(a, s) : launch_kv<Elt::F16, Elt::E4M3, WRITE>(a, s);
    case Elt::I8:
      return bf ? launch_kv<Elt::BF16, Elt::I8, WRITE>(a, s) : launch_kv<Elt::F16, Elt::I8, WRITE>(a, s);
    default: return launch_kv<Elt::BF16, Elt::BF16, WRITE>(a, s);  // 16-bit rows as they are
  }
}

// One workgroup per tree; a thread walks its tokens' ancestors, whose numbers
// fall, and writes each token's words from the last to the first.
constexpr int kMaskTokens = 4096;
__global__ __launch_bounds__(256) void tree_mask_kernel(int tokens, const int32_t* __restrict__ parents,
                                                        uint64_t* __restrict__ mask,
                                                        int32_t* __restrict__ depth) {
  __shared__ int16_t up[kMaskTokens];
  const int64_t b = blockIdx.x;
  for (int t = threadIdx.x; t < tokens; t += 256) {
    const int p = parents[b * tokens + t];
    up[t] = (int16_t)(p >= 0 && p < t ? p : -1);
  }
  __syncthreads();
  const int words = (tokens + 63) / 64;
  for (int t = threadIdx.x; t < tokens; t += 256) {
    uint64_t* row = mask + (b * tokens + t) * words;
    int w = words - 1, at = t, n = 0;
    uint64_t bits = 0;
    while (at >= 0) {
      for (; w > at / 64; --w) {
        row[w] = bits;
        bits = 0;
      }
      bits |= 1ull << (at % 64);
      at = up[at];
      ++n;
    }
    for (; w >= 0; --w) {
      row[w] = bits;
      bits = 0;
    }
    if (depth) depth[b * tokens + t] = n - 1;
  }
}

}  // namespace

hipError_t kv_append(const KvArgs& a, hipStream_t s) { return kv_dispatch<true>(a, s); }
hipError_t kv_read(const KvArgs& a, hipStream_t s) { return kv_dispatch<false>(a, s); }

hipError_t tree_mask(int64_t batch, int tokens, const int32_t* parents, uint64_t* mask,
                     int32_t* depth, hipStream_t s) {
  static_assert(kMaskTokens <= 32768, "parents are kept in 16 bits");
  hipLaunchKernelGGL(tree_mask_kernel, dim3((unsigned)batch), dim3(256), 0, s, tokens, parents, mask,
                     depth);
  return hipGetLastError();
}

}  // namespace frisk
