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
// The work.  16 B of each half of a pair per lane; a thread takes the same
// pairs of several heads, so the angle's ~40 instructions a pair are paid once
// for them, and the loads of up to four heads are in flight together.  HBM
// bounds it.

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

// P pairs per thread and head: two pieces of P elements.  A token has
// `pair_chunks` of those and `copy_chunks` pieces of dims to copy, times
// `lanes` threads that share its heads.
template <Elt E, int P, bool INTER>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int pair_chunks, int copy_chunks,
                                                   int lanes, int tokens_per_block,
                                                   int blocks_per_token) {
  using V = typename Piece<E, P>::V;
  using T = typename EltInfo<E>::T;
  constexpr int HB = 4;  // heads in flight
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

  if (chunk >= pair_chunks) {  // dims that are not rotated
    const int at = a.rot_dim + (chunk - pair_chunks) * P;
    for (int h = first; h < heads; h += lanes) {
      if (h < h0 ? a.t[0].x == a.t[0].out : a.t[1].x == a.t[1].out) continue;  // in place
      *(V*)(out_row(h) + at) = *(const V*)(in_row(h) + at);
    }
    return;
  }
  int64_t p = a.start ? a.start[b] : 0;
  if (!a.positions) p += s;
  else if (a.position_bits == 64) p += ((const int64_t*)a.positions)[b * a.pos_sb + s * a.pos_ss];
  else p += ((const int32_t*)a.positions)[b * a.pos_sb + s * a.pos_ss];
  float cs[P], sn[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const SinCos r = sincos_turns((uint64_t)p * a.freq[chunk * P + i]);
    cs[i] = r.c * a.amplitude;
    sn[i] = (a.backward ? -r.s : r.s) * a.amplitude;
  }
  const int at0 = INTER ? chunk * 2 * P : chunk * P;
  const int at1 = INTER ? at0 + P : at0 + a.rot_dim / 2;
  for (int base = first; base < heads; base += HB * lanes) {
    V x0[HB], x1[HB];
#pragma unroll
    for (int j = 0; j < HB; ++j) {
      const int h = base + j * lanes;
      if (h < heads) {
        const T* row = in_row(h);
        x0[j] = *(const V*)(row + at0);
        x1[j] = *(const V*)(row + at1);
      }
    }
#pragma unroll
    for (int j = 0; j < HB; ++j) {
      const int h = base + j * lanes;
      if (h >= heads) continue;
      V y0, y1;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        // Pair i is (x0[i], x1[i]), or interleaved elements 2i and 2i + 1 of x0, x1.
        const int e0 = INTER ? 2 * i : i, e1 = INTER ? 2 * i + 1 : i;
        const float u = !INTER || e0 < P ? get<E, P>(x0[j], e0) : get<E, P>(x1[j], e0 - P);
        const float w = !INTER ? get<E, P>(x1[j], e1)
                        : e1 < P ? get<E, P>(x0[j], e1) : get<E, P>(x1[j], e1 - P);
        const float yu = __builtin_fmaf(u, cs[i], -(w * sn[i]));
        const float yw = __builtin_fmaf(u, sn[i], w * cs[i]);
        if (!INTER) {
          put<E, P>(y0, i, yu);
          put<E, P>(y1, i, yw);
        } else {
          if (e0 < P) put<E, P>(y0, e0, yu); else put<E, P>(y1, e0 - P, yu);
          if (e1 < P) put<E, P>(y0, e1, yw); else put<E, P>(y1, e1 - P, yw);
        }
      }
      T* row = out_row(h);
      *(V*)(row + at0) = y0;
      *(V*)(row + at1) = y1;
    }
  }
}

template <Elt E, int P>
hipError_t launch_rope(const RopeArgs& a, hipStream_t stream) {
  const int heads = a.t[0].heads + a.t[1].heads;
  const bool copies = a.t[0].x != a.t[0].out || (a.t[1].heads && a.t[1].x != a.t[1].out);
  const int pair_chunks = a.rot_dim / 2 / P;
  const int copy_chunks = copies ? (a.head_dim - a.rot_dim) / P : 0;
  const int chunks = pair_chunks + copy_chunks;
  // A thread takes up to 8 heads once that leaves two workgroups' threads for
  // every CU.
  const int64_t tokens = a.batch * a.seq;
  const int64_t spare = tokens * chunks * heads / ((int64_t)device_cus() * 512);
  const int per = (int)std::min<int64_t>(std::max<int64_t>(spare, 1), 8);
  const int lanes = (heads + per - 1) / per;
  const int64_t n = (int64_t)chunks * lanes;
  const int tpb = n < 256 ? (int)(256 / n) : 1, bpt = (int)((n + 255) / 256);
  const int64_t blocks = n < 256 ? (tokens + tpb - 1) / tpb : tokens * bpt;
  if (blocks > UINT32_MAX / 256) return hipErrorInvalidConfiguration;
  if (a.interleaved)
    hipLaunchKernelGGL((rope_kernel<E, P, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a,
                       pair_chunks, copy_chunks, lanes, tpb, bpt);
  else
    hipLaunchKernelGGL((rope_kernel<E, P, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a,
                       pair_chunks, copy_chunks, lanes, tpb, bpt);
  return hipGetLastError();
}

// The widest pieces, up to 16 B, that divide the pairs, the copied dims and
// every stride, and that the pointers are aligned to.
template <Elt E>
hipError_t rope_type(const RopeArgs& a, hipStream_t stream) {
  constexpr int es = EltInfo<E>::bytes;
  uint64_t bits = (uint64_t)(a.rot_dim / 2) | (uint64_t)(a.head_dim - a.rot_dim);
  for (int i = 0; i < (a.t[1].heads ? 2 : 1); ++i) {
    const RopeTensor& t = a.t[i];
    bits |= (uint64_t)t.sb | (uint64_t)t.sh | (uint64_t)t.ss | (uint64_t)t.osb | (uint64_t)t.osh |
            (uint64_t)t.oss | (uint64_t)t.x / es | (uint64_t)t.out / es;
  }
  if constexpr (es == 2)
    if (bits % 8 == 0) return launch_rope<E, 8>(a, stream);
  if (bits % 4 == 0) return launch_rope<E, 4>(a, stream);
  if (bits % 2 == 0) return launch_rope<E, 2>(a, stream);
  return launch_rope<E, 1>(a, stream);
}

}  // namespace

hipError_t rope(const RopeArgs& a, hipStream_t s) {
  switch (a.dtype) {
    case Elt::F32: return rope_type<Elt::F32>(a, s);
    case Elt::F16: return rope_type<Elt::F16>(a, s);
    case Elt::BF16: return rope_type<Elt::BF16>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace frisk
