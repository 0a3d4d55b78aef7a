// Rotary positions: pairs of a row's first rot_dim dims turned by the angle of
// the row's position, the other dims copied.
//
// The angle.  F (64-bit) is the pair's turns per position times 2^64, so the
// wrapping product p F is the phase in turns times 2^64 exactly, for any p:
// what is lost is the rounding of F alone (2^-53 of it from a double, 2^-34
// turns at a position of a million).  Its top 32 bits, as a signed fraction of
// a turn, split into a quadrant and a rest of at most an eighth of a turn,
// whose sine and cosine are Taylor polynomials (degrees 9 and 10: the first
// terms left out are 1.8e-9 and 1.1e-10 at pi / 4, below half a step of f32).
//
// The work.  A thread takes 16 B of each half of its pairs, or 16 B of interleaved
// pairs, of several heads, so the angle's ~40 instructions a pair are paid once
// for them and the loads of up to 8 pieces are in flight together.  HBM
// bounds it.  Outputs beyond the L2s' 32 MB are stored past them where a wave
// stores whole 128-B lines (they would be written back at the kernel's end, and
// nobody reads them there): q and k of 8192 tokens, h32/8 d128 bf16, 45 -> 34 us;
// rows of 192 + 128 B, which leave parts of lines, are faster through L2 (11
// against 13 us).

#include "common.h"
#include "kernels.h"

namespace frisk {

namespace {

struct SinCos {
  float s, c;
};

// Sine and cosine of 2 pi phase / 2^64.
__device__ __forceinline__ SinCos sincos_turns(uint64_t phase) {
  const uint32_t u = (uint32_t)((phase + 0x80000000ull) >> 32);
  const uint32_t q = (u + 0x20000000u) >> 30;  // nearest quarter turn
  const int32_t r = (int32_t)(u - (q << 30));
  const float y = (float)r * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = y * y;
  float s = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(z, s, 8.3333333e-3f);
  s = __builtin_fmaf(z, s, -1.6666667e-1f);
  s = __builtin_fmaf(z * s, y, y);
  float c = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(z, c, -1.3888889e-3f);
  c = __builtin_fmaf(z, c, 4.1666667e-2f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.0f);
  const float ss = q & 1 ? c : s, cc = q & 1 ? s : c;
  return {q & 2 ? -ss : ss, (q + 1) & 2 ? -cc : cc};
}

template <Elt E, int P> struct Piece {
  using T = typename EltInfo<E>::T;
  typedef T V __attribute__((ext_vector_type(P)));
};
template <Elt E> struct Piece<E, 1> {
  using V = typename EltInfo<E>::T;
};

template <Elt E, int P> __device__ __forceinline__ float get(const typename Piece<E, P>::V& v, int i) {
  if constexpr (P == 1) return (float)v;
  else return (float)v[i];
}
template <Elt E, int P> __device__ __forceinline__ void put(typename Piece<E, P>::V& v, int i, float f) {
  if constexpr (P == 1) v = (typename EltInfo<E>::T)f;
  else v[i] = (typename EltInfo<E>::T)f;
}

// Pieces of P elements.  Pairs in halves: a chunk is P pairs, a piece of each
// half; interleaved: a chunk is one piece of P / 2 pairs (P == 1: two pieces, one
// pair).  A token has `pair_chunks` of those and `copy_chunks` pieces of dims to
// copy, times `lanes` threads that share its heads.
template <Elt E, int P, bool INTER, bool PAST_L2>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int pair_chunks, int copy_chunks,
                                                   int lanes, int tokens_per_block,
                                                   int blocks_per_token) {
  using V = typename Piece<E, P>::V;
  using T = typename EltInfo<E>::T;
  constexpr int NV = INTER && P > 1 ? 1 : 2;          // pieces of a chunk
  constexpr int NP = INTER && P > 1 ? P / 2 : P;      // pairs of a chunk
  constexpr int HB = 8 / NV;                          // heads in flight
  const int chunks = pair_chunks + copy_chunks, n = chunks * lanes;
  int64_t token;
  int item;
  if (blocks_per_token > 1) {
    token = blockIdx.x / blocks_per_token;
    item = (int)(blockIdx.x - (uint32_t)token * blocks_per_token) * 256 + (int)threadIdx.x;
    if (item >= n) return;
  } else {
    const int t = threadIdx.x / n;
    item = threadIdx.x - t * n;
    token = (int64_t)blockIdx.x * tokens_per_block + t;
    if (t >= tokens_per_block || token >= a.batch * a.seq) return;
  }
  const int chunk = item % chunks, first = item / chunks;
  const int64_t b = (uint64_t)token / (uint64_t)a.seq, s = token - b * a.seq;
  const int h0 = a.t[0].heads, heads = h0 + a.t[1].heads;

  // The token's rows of head 0 of each tensor, and the row of head h.
  const T* in0 = (const T*)a.t[0].x + (b * a.t[0].sb + s * a.t[0].ss);
  const T* in1 = (const T*)a.t[1].x + (b * a.t[1].sb + s * a.t[1].ss);
  T* out0 = (T*)a.t[0].out + (b * a.t[0].osb + s * a.t[0].oss);
  T* out1 = (T*)a.t[1].out + (b * a.t[1].osb + s * a.t[1].oss);
  auto in_row = [&](int h) {
    return h < h0 ? in0 + h * a.t[0].sh : in1 + (h - h0) * a.t[1].sh;
  };
  auto out_row = [&](int h) {
    return h < h0 ? out0 + h * a.t[0].osh : out1 + (h - h0) * a.t[1].osh;
  };
  auto store = [&](T* p, V v) {
    if constexpr (PAST_L2) __builtin_nontemporal_store(v, (V*)p);
    else *(V*)p = v;
  };
  auto load = [&](const T* p) {
    if constexpr (PAST_L2) return __builtin_nontemporal_load((const V*)p);
    else return *(const V*)p;
  };

  if (chunk >= pair_chunks) {  // dims that are not rotated
    const int at = a.rot_dim + (chunk - pair_chunks) * P;
    for (int h = first; h < heads; h += lanes) {
      if (h < h0 ? a.t[0].x == a.t[0].out : a.t[1].x == a.t[1].out) continue;  // in place
      store(out_row(h) + at, load(in_row(h) + at));
    }
    return;
  }
  int64_t p = a.start ? a.start[b] : 0;
  if (!a.positions) p += s;
  else if (a.position_bits == 64) p += ((const int64_t*)a.positions)[b * a.pos_sb + s * a.pos_ss];
  else p += ((const int32_t*)a.positions)[b * a.pos_sb + s * a.pos_ss];
  float cs[NP], sn[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const SinCos r = sincos_turns((uint64_t)p * a.freq[chunk * NP + i]);
    cs[i] = r.c * a.amplitude;
    sn[i] = (a.backward ? -r.s : r.s) * a.amplitude;
  }
  const int at0 = INTER ? chunk * 2 * NP : chunk * NP;
  const int at1 = INTER ? at0 + 1 : at0 + a.rot_dim / 2;  // (the second piece, if any)
  for (int base = first; base < heads; base += HB * lanes) {
    V x[HB][NV];
#pragma unroll
    for (int j = 0; j < HB; ++j) {
      const int h = base + j * lanes;
      if (h < heads) {
        const T* row = in_row(h);
        x[j][0] = load(row + at0);
        if constexpr (NV == 2) x[j][1] = load(row + at1);
      }
    }
#pragma unroll
    for (int j = 0; j < HB; ++j) {
      const int h = base + j * lanes;
      if (h >= heads) continue;
      V y[NV];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int e0 = NV == 1 ? 2 * i : i, e1 = NV == 1 ? 2 * i + 1 : i;
        const float u = get<E, P>(x[j][0], e0), w = get<E, P>(x[j][NV - 1], e1);
        put<E, P>(y[0], e0, __builtin_fmaf(u, cs[i], -(w * sn[i])));
        put<E, P>(y[NV - 1], e1, __builtin_fmaf(u, sn[i], w * cs[i]));
      }
      T* row = out_row(h);
      store(row + at0, y[0]);
      if constexpr (NV == 2) store(row + at1, y[1]);
    }
  }
}

template <Elt E, int P, bool INTER>
hipError_t launch_rope(const RopeArgs& a, hipStream_t stream) {
  constexpr int NP = INTER && P > 1 ? P / 2 : P, es = EltInfo<E>::bytes;
  const int heads = a.t[0].heads + a.t[1].heads;
  const bool copies = a.t[0].x != a.t[0].out || (a.t[1].heads && a.t[1].x != a.t[1].out);
  const int pair_chunks = a.rot_dim / 2 / NP;
  const int copy_chunks = copies ? (a.head_dim - a.rot_dim) / P : 0;
  const int chunks = pair_chunks + copy_chunks;
  // A thread takes as many heads as it has in flight at once, where that leaves
  // two workgroups' threads for every CU.
  constexpr int kMost = INTER && P > 1 ? 8 : 4;
  const int64_t tokens = a.batch * a.seq;
  const int64_t spare = tokens * chunks * heads / ((int64_t)device_cus() * 512);
  const int per = (int)std::min<int64_t>(std::max<int64_t>(spare, 1), kMost);
  const int lanes = (heads + per - 1) / per;
  const int64_t n = (int64_t)chunks * lanes;
  const int tpb = n < 256 ? (int)(256 / n) : 1, bpt = (int)((n + 255) / 256);
  const int64_t blocks = n < 256 ? (tokens + tpb - 1) / tpb : tokens * bpt;
  if (blocks > UINT32_MAX / 256) return hipErrorInvalidConfiguration;
  const int64_t run = INTER ? a.rot_dim : a.rot_dim / 2;  // elements that neighbouring lanes store
  const bool past_l2 = run * es % 128 == 0 && (a.head_dim - a.rot_dim) * es % 128 == 0 &&
                       tokens * heads * a.head_dim * es > (32ll << 20);
  auto kern = rope_kernel<E, P, INTER, false>;
  if constexpr (P * es == 16)
    if (past_l2) kern = rope_kernel<E, P, INTER, true>;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, a, pair_chunks, copy_chunks, lanes,
                     tpb, bpt);
  return hipGetLastError();
}

// The widest pieces, up to 16 B, that divide the rotated dims (in halves: a
// half), the copied dims and every stride, and that the pointers are aligned to.
template <Elt E, bool INTER>
hipError_t rope_type(const RopeArgs& a, hipStream_t stream) {
  constexpr int es = EltInfo<E>::bytes;
  uint64_t bits = (uint64_t)(INTER ? a.rot_dim : a.rot_dim / 2) | (uint64_t)(a.head_dim - a.rot_dim);
  for (int i = 0; i < (a.t[1].heads ? 2 : 1); ++i) {
    const RopeTensor& t = a.t[i];
    bits |= (uint64_t)t.sb | (uint64_t)t.sh | (uint64_t)t.ss | (uint64_t)t.osb | (uint64_t)t.osh |
            (uint64_t)t.oss | (uint64_t)t.x / es | (uint64_t)t.out / es;
  }
  if constexpr (es == 2)
    if (bits % 8 == 0) return launch_rope<E, 8, INTER>(a, stream);
  if (bits % 4 == 0) return launch_rope<E, 4, INTER>(a, stream);
  if (bits % 2 == 0) return launch_rope<E, 2, INTER>(a, stream);
  return launch_rope<E, 1, INTER>(a, stream);
}

}  // namespace

hipError_t rope(const RopeArgs& a, hipStream_t s) {
  switch (a.dtype) {
    case Elt::F32: return a.interleaved ? rope_type<Elt::F32, true>(a, s) : rope_type<Elt::F32, false>(a, s);
    case Elt::F16: return a.interleaved ? rope_type<Elt::F16, true>(a, s) : rope_type<Elt::F16, false>(a, s);
    case Elt::BF16: return a.interleaved ? rope_type<Elt::BF16, true>(a, s) : rope_type<Elt::BF16, false>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace frisk
