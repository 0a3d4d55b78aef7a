// Attention of new tokens over a cache on the matrix cores, head_dim 32, 64 or
// 128.  attn_tree_d*.hip instantiate the kernels.
//
// The query rows of one kv head (tokens x the heads that share it) form tiles
// of 32; a key block is 64 keys.  A block's arithmetic is that of attn.h: S^T =
// K.Q^T on 32x32x16 MFMAs, so that a lane owns a query row and 32 of its scores;
// online softmax in the exp2 domain with a lazily moving maximum; P rounded
// to q's type feeds O^T += V^T.P^T from the registers it is in, and V^T comes
// from transposing LDS reads in the matching key order.  The row sum is kept
// over the unrounded P, so that the log-sum-exp is exact to f32.
//
// 8-bit rows: codes widen exactly (4 or 8 significant bits), a key's to q's type,
// a value's to bf16.  A key's score is its column of S times the key's scale, and
// P is the weight times the value's scale, in f32; the row sum is of the weights.
// P needs bf16's range: f16 would round a key to nothing whose value scale is 2^-25
// of another's, though it alone may feed a dim.  With q in bf16 P is rounded once,
// as over a 16-bit cache; with q in f16 it is the sum of two bf16 numbers, 16 bits
// (f16 has 11), and the second product is taken twice.
//
// Where a key lies is computed once per key and block (a page number from the
// table, loaded a block ahead), into LDS, as a 64-bit offset; the row loads go
// straight to LDS from 64-bit addresses, so neither pages nor long caches
// limit them.  A key behind the last, or on a page that is none, is loaded from
// the cache's first row and hidden.
//
// Hidden keys must not matter whatever they hold, and 0 * NaN is NaN: in blocks
// with a hidden key a V row that is not finite, or whose scale is not, is taken out
// of the product and added by itself to the rows that see it.
#pragma once

#include "attn_tree.h"

namespace frisk {
namespace tree {

#define TREE_INLINE __device__ __forceinline__

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(1))) const void* global_ptr;

constexpr float kSlack = 8.0f;  // log2 headroom before the running maximum moves

template <Elt T> TREE_INLINE f32x16 mfma(i32x4 a, i32x4 b, f32x16 c) {
  if constexpr (T == Elt::BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Lane l with lane l ^ 32 (both get the result).
TREE_INLINE float pair_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
TREE_INLINE float pair_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

constexpr bool is8(Elt c) { return c == Elt::E4M3 || c == Elt::I8; }
constexpr int bytes_of(Elt c) { return is8(c) ? 1 : 2; }
// Type of the second product, and the parts that P enters it in (pack_p).
template <Elt T, Elt C> constexpr Elt kProduct = is8(C) ? Elt::BF16 : T;
template <Elt T, Elt C> constexpr int kParts = is8(C) && T == Elt::F16 ? 2 : 1;

// LDS geometry of 64 rows (keys) of D elements: rows of kRB bytes, kKC chunks of
// 16 B, chunk c of row r stored at c ^ swz(r).
//  K: the 16 rows that one cycle of ds_read_b128 takes at one logical chunk
//     land in 16 distinct chunks of the 256-B bank window.
//  V: a transposing read takes 4 rows (r & 3) x 64 B in 16 bits, 8 rows (bits
//     0, 1 and 3 of r vary) x 32 B in 8 bits, which land apart (rows of 32 B:
//     two by two).
template <Elt C, int D> struct Geom {
  static constexpr int kRB = D * bytes_of(C), kKC = kRB / 16;
  static constexpr int kShift = kKC == 16 ? 0 : kKC == 8 ? 1 : kKC == 4 ? 2 : 3;
  static constexpr int kTile = kBlock * kRB;
  static constexpr int kLoads = kTile / 1024;  // 1 KiB per load instruction
  static constexpr int kRows = 1024 / kRB;     // rows per load
  __device__ static int swz_k(int r) { return (r >> kShift) & (kKC - 1); }
  __device__ static int swz_v(int r) {
    if constexpr (is8(C)) {
      if constexpr (kKC == 8) return (((r >> 1) & 1) | ((r >> 2) & 2)) << 1;
      else if constexpr (kKC == 4) return ((r >> 3) & 1) << 1;
      else return 0;
    } else {
      if constexpr (kKC == 16) return 4 * (r & 3);
      else if constexpr (kKC == 8) return 2 * ((r >> 1) & 1);
      else return 0;
    }
  }
};

// Eight codes as eight values of T (exact).
template <Elt T, Elt C> TREE_INLINE i32x4 widen8(int w0, int w1) {
  i32x4 out;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int w = i ? w1 : w0;
    if constexpr (C == Elt::E4M3 && T == Elt::BF16) {
      out[2 * i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
      out[2 * i + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    } else if constexpr (C == Elt::E4M3) {
      out[2 * i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
      out[2 * i + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    } else {
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(w >> (8 * e));
      out[2 * i] = (int)pack16<T>(f[0], f[1]);
      out[2 * i + 1] = (int)pack16<T>(f[2], f[3]);
    }
  }
  return out;
}

// Q fragments of one row (B operand of S^T): step ds, lane half h holds dims
// 16 ds + 8 h .. +7; over codes, whose lanes read 16 dims at a time, steps 2 j
// and 2 j + 1 hold dims 16 (2 j + h) .. +7 and +8 .. +15.
template <Elt C, int D> TREE_INLINE void load_q(const char* row, int half, i32x4 (&qf)[D / 16]) {
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) {
    const int d = is8(C) ? 16 * ((ds & ~1) + half) + 8 * (ds & 1) : 16 * ds + 8 * half;
    qf[ds] = *(const i32x4*)(row + d * 2);
  }
}

// K fragments of steps h0 .. h0 + N - 1 (N even over codes) of both 32-key tiles.
template <Elt T, Elt C, int D, int N>
TREE_INLINE void read_k(const char* ks, int h0, int l32, int half, i32x4 (&kf)[2][N]) {
  using G = Geom<C, D>;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int r = kt * 32 + l32;
    if constexpr (is8(C)) {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const i32x4 w = *(const i32x4*)(ks + r * G::kRB + (((h0 + i + half) ^ G::swz_k(r)) << 4));
        kf[kt][i] = widen8<T, C>(w[0], w[1]);
        kf[kt][i + 1] = widen8<T, C>(w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        kf[kt][i] = *(const i32x4*)(ks + r * G::kRB + (((2 * (h0 + i) + half) ^ G::swz_k(r)) << 4));
    }
  }
}

// Lane offset of the transposing reads of V^T (attn.h and gemm_tile.h derive
// them): the fragment of key step kk and dim tile dt holds, in lane (l32,
// half), V[16 kk + (e < 4 ? 4 half + e : 4 + 4 half + e)][32 dt + l32], e = 0 .. 7.
// A dim tile further is another chunk of the row, an XOR above the swizzle.
template <Elt C, int D> TREE_INLINE uint32_t v_offset(int lane) {
  using G = Geom<C, D>;
  const int g = lane >> 4, h = g >> 1, dg = g & 1;
  if constexpr (is8(C)) {
    const int e = (lane >> 1) & 7, b = lane & 1, r = e < 4 ? 4 * h + e : 4 + 4 * h + e;
    return r * G::kRB + ((dg ^ G::swz_v(r)) << 4) + 8 * b;
  } else {
    const int e = (lane >> 2) & 3, q = lane & 3, r = 4 * h + e;
    return r * G::kRB + (((2 * dg + (q >> 1)) ^ G::swz_v(r)) << 4) + 8 * (q & 1);
  }
}
// `at`: v_offset and the offset of V's tile (a multiple of 256 B) in lds.
template <Elt T, Elt C, int D> TREE_INLINE i32x4 read_v(const char* lds, uint32_t at, int kk, int dt) {
  using G = Geom<C, D>;
  const char* p = lds + (at ^ (uint32_t)(dt << (is8(C) ? 5 : 6))) + kk * 16 * G::kRB;
  if constexpr (is8(C)) {
    const i32x2 w = lds_read_tr8(p);
    return widen8<T, C>(w[0], w[1]);
  } else {
    const i32x2 a = __builtin_bit_cast(i32x2, lds_read_tr16(p));
    const i32x2 c = __builtin_bit_cast(i32x2, lds_read_tr16(p + 8 * G::kRB));
    return i32x4{a[0], a[1], c[0], c[1]};
  }
}

// ---- masks -----------------------------------------------------------------------

// seen_bits of token t of sequence b.
TREE_INLINE uint64_t seen_bits(const TreeAttnArgs& a, int64_t b, int t, int64_t ctx, int n0, uint64_t there) {
  return seen_bits(a.mask ? a.mask + (b * a.mask_sb + t * a.mask_st) : nullptr, a.tokens, t, ctx, n0, there);
}
// Key of score register r (of 16) of tile kt, less 4 half.
constexpr int key_of(int kt, int r) { return kt * 32 + 8 * (r >> 2) + (r & 3); }

// ---- softmax of one block -----------------------------------------------------------

// A row's running state.
template <int D> struct State {
  f32x16 o[D / 32];
  float m, l;
};
template <int D> TREE_INLINE void clear(State<D>& st) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) st.o[dt] = f32x16{};
  st.m = -__builtin_inff();
  st.l = 0.0f;
}

// The running maximum of rows whose block's `top`, counted from it (from 0 where it
// is none), is `move` too high; what the block's scores are lowered by.
template <int D> TREE_INLINE float raise(State<D>& st, bool move, float top) {
  const bool none = st.m == -__builtin_inff();
  const float from = none ? 0.0f : st.m, to = from + top;
  const float by = move ? to - from : 0.0f;
  const float alpha = none ? 1.0f : __builtin_amdgcn_exp2f(-by);  // (without a maximum l and o are 0)
  st.m = move ? to : st.m;
  st.l *= alpha;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) st.o[dt] *= alpha;
  return by;
}

// What a block's scales are kept as: the key's times scale_log2, then the value's.
// In a block with a hidden key a value scale that is not finite counts as 0, and
// add_key adds what the rows that see it get: NaN.
TREE_INLINE void put_scale(float* sc, int lane, float value, bool of_key, float scale_log2, bool masked) {
  if (of_key) sc[lane] = value * scale_log2;
  else sc[64 + lane] = masked && !(fabsf(value) < __builtin_inff()) ? 0.0f : value;
}
// Bits of the keys whose value scale is not finite (lane = key).
TREE_INLINE uint64_t nan_scales(float value) {
  return __builtin_amdgcn_ballot_w64(!(fabsf(value) < __builtin_inff()));
}

// Scores s to P (in place, f32): the weights, over codes times the value's scale.
// seen: bits of the row's keys shifted down by 4 half, read if masked (uniform).
// sc: over codes, the block's scales (put_scale).  The row sum and the maximum
// are of the weights alone.
template <Elt C, int D>
TREE_INLINE void softmax(f32x16 (&s)[2], State<D>& st, float scale_log2, const float* sc, int half, bool masked,
                         uint64_t seen) {
  constexpr bool k8 = is8(C);
  // A row that has seen no key keeps m = -inf: p = 0, not NaN.
  float nm = st.m == -__builtin_inff() ? 0.0f : -st.m;
  if constexpr (k8) {  // counted from the maximum, which seldom moves
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 by = *(const f32x4*)(sc + kt * 32 + 8 * g + 4 * half);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[kt][4 * g + i] = __builtin_fmaf(s[kt][4 * g + i], by[i], nm);
      }
  }
  if (masked) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[kt][r] = (seen >> key_of(kt, r)) & 1 ? s[kt][r] : -__builtin_inff();
  }
  float top = -__builtin_inff();
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kt][r]);
  top = pair_max(top);
  if constexpr (k8) {
    const bool move = st.m == -__builtin_inff() ? top > st.m : top > kSlack;
    if (__builtin_amdgcn_ballot_w64(move)) {
      const float by = raise(st, move, top);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kt][r] -= by;
    }
  } else {
    top *= scale_log2;
    const bool move = top > st.m + kSlack;
    if (__builtin_amdgcn_ballot_w64(move)) {
      const float alpha = move ? __builtin_amdgcn_exp2f(st.m - top) : 1.0f;
      st.m = move ? top : st.m;
      st.l *= alpha;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) st.o[dt] *= alpha;
    }
    nm = st.m == -__builtin_inff() ? 0.0f : -st.m;
  }
  float l = st.l;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[kt][r] = __builtin_amdgcn_exp2f(k8 ? s[kt][r] : __builtin_fmaf(s[kt][r], scale_log2, nm));
      l += s[kt][r];
    }
  st.l = l;
  if constexpr (k8) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 by = *(const f32x4*)(sc + 64 + kt * 32 + 8 * g + 4 * half);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[kt][4 * g + i] *= by[i];
      }
  }
}

// P of key step kk as the B operand of the second product.
template <Elt T, Elt C> TREE_INLINE void pack_p(const f32x16 (&s)[2], int kk, i32x4 (&pf)[kParts<T, C>]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = 8 * (kk & 1) + 2 * e;
    const float x = s[kk >> 1][r], y = s[kk >> 1][r + 1];
    const uint32_t w = pack16<kProduct<T, C>>(x, y);
    pf[0][e] = (int)w;
    if constexpr (kParts<T, C> == 2)
      pf[1][e] = (int)pack16<Elt::BF16>(x - __builtin_bit_cast(float, w << 16),
                                        y - __builtin_bit_cast(float, w & 0xffff0000u));
  }
}

// ---- V rows that are not finite ----------------------------------------------------

// Bits of the block's keys whose V row holds an infinity or NaN (lane = key).
template <Elt T, Elt C, int D> TREE_INLINE uint64_t not_finite(const char* vs, int lane) {
  using G = Geom<C, D>;
  if constexpr (C == Elt::I8) return 0;
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < G::kKC; ++i) {
    const i32x4 w = *(const i32x4*)(vs + lane * G::kRB + 16 * ((i + lane) & (G::kKC - 1)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // A carry into the sign bit of each element from a full exponent (codes:
      // from the NaN code).
      const uint32_t x = (uint32_t)w[e];
      if constexpr (C == Elt::E4M3) bad |= ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
      else if constexpr (T == Elt::BF16) bad |= ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
      else bad |= ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    }
  }
  return __builtin_amdgcn_ballot_w64(bad != 0);
}

// o += p V of key `key` alone, for rows that see it; NaN if its scale is.
template <Elt T, Elt C, int D>
TREE_INLINE void add_key(const char* vs, int key, const f32x16 (&p)[2], uint64_t seen, bool nan, int l32, int half,
                         State<D>& st) {
  using G = Geom<C, D>;
  float w = 0.0f;
  // w = p of the key, one condition at a time: 32 at once would take the scalar
  // registers that the loop over keys has.
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      asm("v_cmp_eq_u32_e32 vcc, %1, %2\n\tv_cndmask_b32_e32 %0, %0, %3, vcc"
          : "+v"(w)
          : "n"(key_of(kt, r)), "v"(key & ~4), "v"(p[kt][r])
          : "vcc");
  const int from = l32 + 32 * ((key >> 2) & 1);  // the half that holds the key
  w = nan ? __builtin_nanf("") : __shfl(w, from);
  const bool sees_it = __shfl((int)((seen >> (key & ~4)) & 1), from);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = dt * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
      const int at = key * G::kRB + (((d * bytes_of(C) >> 4) ^ G::swz_v(key)) << 4) + (d * bytes_of(C) & 15);
      float v;
      if constexpr (is8(C)) {
        v = __builtin_amdgcn_cvt_f32_fp8((int)*(const uint8_t*)(vs + at), 0);
      } else {
        const uint16_t h = *(const uint16_t*)(vs + at);
        v = T == Elt::BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
      }
      st.o[dt][r] += sees_it ? w * v : 0.0f;
    }
}
template <Elt C, int D> TREE_INLINE void clear_key(char* vs, int key, int lane) {
  using G = Geom<C, D>;
  if (lane < G::kKC) *(i32x4*)(vs + key * G::kRB + 16 * lane) = i32x4{0, 0, 0, 0};
}

// Workgroup pid as (unit: sequence, kv head and split; tile of its rows).  The
// tiles of a unit run on one XCD (workgroups go round the 8 XCDs), next to each
// other, so that its L2 holds the keys they share.
TREE_INLINE void place_unit(int pid, int units, int tiles, int& unit, int& tile) {
  if (units % 8 == 0) {
    unit = ((pid >> 3) / tiles) * 8 + (pid & 7);
    tile = (pid >> 3) % tiles;
  } else {
    unit = pid / tiles;
    tile = pid % tiles;
  }
}

// ---- few rows: the waves divide the keys ---------------------------------------------

// Waves per workgroup: K and V tiles of all waves in LDS.
template <Elt C, int D> constexpr int kKeyWaves = plan::tree_key_waves(D);
constexpr int kExtra = 1024;  // per wave: 64 row offsets (8 B), 64 scales of K and of V
template <Elt C, int D> constexpr int keys_lds() {
  const int tiles = kKeyWaves<C, D> * (2 * Geom<C, D>::kTile + kExtra);
  const int sum = kKeyWaves<C, D> * 32 * (D + 4 + 2) * 4;
  return tiles > sum ? tiles : sum;
}

// The f32 rows of a tile's splits: per split [32][D] of O (not divided by l),
// then [32][2] of m and l; and the word its splits arrive at.  They are written
// and read past the XCDs' L2 caches (device scope), the arrival is an atomic.
constexpr int kDeviceScope = 0x10;  // SC1 of a buffer access
struct KeysPart {
  __amdgpu_buffer_rsrc_t rs;
  int bytes;  // of a split
  unsigned long long* word;
};
template <int D> TREE_INLINE KeysPart keys_part(const Part& p, int64_t tile) {
  constexpr int kFloats = 32 * (D + 2);
  KeysPart k;
  k.bytes = kFloats * 4;
  k.rs = __builtin_amdgcn_make_buffer_rsrc((void*)(p.o + tile * p.splits * kFloats), (short)0,
                                           p.splits * kFloats * 4, 0x00020000);
  k.word = p.words + tile;
  return k;
}

// Whether this is the last of n arrivals at a word, which is then 0 again.  Any
// value but kArrived + count reads as no arrival yet, so a workspace needs no
// clearing (one never used holds that with probability 2^-56).
constexpr unsigned long long kArrived = 0x7AEE51EC0DE20000ull;
TREE_INLINE int arrive(unsigned long long* word, int n) {
  unsigned long long old = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // An exchange fails only when another arrival changed the word: at most n
  // times.
  for (int attempt = 0; attempt <= n; ++attempt) {
    const int count = (old & ~0xffull) == kArrived ? (int)(old & 0xff) : 0;
    const bool last = count + 1 == n;
    if (__hip_atomic_compare_exchange_strong(word, &old, last ? 0ull : kArrived + count + 1, __ATOMIC_RELAXED,
                                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
      return last;
  }
  return 0;
}

// One tile of 32 rows per workgroup; each wave takes every NW-th key block of
// the split with K and V tiles of its own: no barrier in the loop, and a block's
// bytes of loads in flight per wave.  One token of b16 h32/8 d128 bf16, up to 8192 keys,
// is bound by HBM: 412 MB in 80 us, 5.1 TB/s.  33 tokens of b4 h16/16 d64, f16 over i8, take
// 24.6 us (36 MB): two tiles, which both read and widen all keys, up to 5 blocks a wave whose
// widening, scales and softmax have few products to hide behind.
template <Elt T, Elt C, int D>
__global__ __launch_bounds__((64 * kKeyWaves<C, D>)) void tree_keys_kernel(TreeAttnArgs a, Part part,
                                                                         int row_tiles, int units) {
#if defined(__HIP_DEVICE_COMPILE__)
  using G = Geom<C, D>;
  constexpr int NW = kKeyWaves<C, D>;
  constexpr bool k8 = is8(C);
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int unit, tile;
  place_unit(blockIdx.x, units, row_tiles, unit, tile);
  const int split = unit % part.splits, bk = unit / part.splits;
  const int64_t b = bk / a.cache.kv_heads;
  const int kvh = bk % a.cache.kv_heads;
  const int group = a.heads / a.cache.kv_heads;
  const kv::Span sp = kv::span_of(a.ctx_len, a.new_len, a.tokens, b);
  const int rows = sp.fresh * group;
  if (sp.ctx < 0 || tile * 32 >= rows) return;
  int keys = keys_of(a.cache.capacity, sp);
  const int blocks_all = (keys + kBlock - 1) / kBlock;
  const int per = blocks_per_split(part, blocks_all);
  if (split > 0 && split * per >= blocks_all) return;
  const int row = min(tile * 32 + l32, rows - 1), t = row / group, h = kvh * group + row % group;
  const int end = min(blocks_all, (split + 1) * per);

  i32x4 qf[D / 16];
  load_q<C, D>((const char*)a.q + (b * a.q_sb + h * a.q_sh + t * a.q_ss) * 2, half, qf);
  const float scale_log2 = a.sm_scale * kLog2eF;

  char* ks = smem + wave * (2 * G::kTile + kExtra);
  char* vs = ks + G::kTile;
  int64_t* offs = (int64_t*)(vs + G::kTile);
  float* sc = (float*)(offs + 64);
  const char* kbase = (const char*)a.cache.k;
  const char* vbase = (const char*)a.cache.v;
  const int lrow = lane / G::kKC, lchunk = lane % G::kKC;
  auto issue = [&](const char* base, char* dst, bool is_v) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < G::kLoads; ++i) {
      const int r = i * G::kRows + lrow, c = lchunk ^ (is_v ? G::swz_v(r) : G::swz_k(r));
      __builtin_amdgcn_global_load_lds((global_ptr)(base + offs[r] + (c << 4)), (lds_ptr)(dst + i * 1024),
                                       16, 0, 0);
    }
  };
  const uint32_t v_at = (uint32_t)(vs - smem) + v_offset<C, D>(lane);
  State<D> st;
  clear(st);

  // The table entry of this lane's key of block kb.
  auto my_entry = [&](int kb) { return entry_of(a.cache, a.ctx_len, b, kb * kBlock + lane); };
  int kb = split * per + wave;
  int entry = 0;
  uint64_t there = 0, there_next = 0;
  float ksc = 0.0f, vsc = 0.0f;
  auto place = [&](int block, int e) __attribute__((always_inline)) {
    const Place p = place_of(a.cache, bytes_of(C), b, kvh, block * kBlock + lane, keys, e);
    offs[lane] = p.row;
    if constexpr (k8) {
      ksc = a.cache.k_scale[p.scale];
      vsc = a.cache.v_scale[p.scale];
    }
    return __builtin_amdgcn_ballot_w64(p.there);
  };
  // Table entries of the first two blocks; Q has landed with them, on every
  // path into the loop, so that nothing in it waits for a load by accident.
  const int first = my_entry(max(0, min(kb, end - 1)));
  entry = my_entry(max(0, min(kb + NW, end - 1)));
#pragma unroll
  for (int i = 0; i < D / 16; ++i) asm volatile("" ::"v"(qf[i]), "v"(first), "v"(entry));
  __builtin_amdgcn_s_waitcnt(0);
  if (kb < end) {
    there = place(kb, first);
    __builtin_amdgcn_sched_barrier(0);
    issue(kbase, ks, false);
    issue(vbase, vs, true);
  }
  for (; kb < end; kb += NW) {
    const bool more = kb + NW < end;
    const bool masked = there != ~0ull || (int64_t)(kb + 1) * kBlock > sp.ctx;
    // K landed (V's loads may still be in flight), and with it the scales and
    // the table entry, which were asked for before.
    constexpr int nv = G::kLoads;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((nv & 15) | ((nv >> 4) << 14) | (7 << 4) | (15 << 8));
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (k8) {
      put_scale(sc, lane, ksc, true, scale_log2, masked);
      put_scale(sc, lane, vsc, false, scale_log2, masked);
    }
    const float value_scale = vsc;
    f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int h0 = 0; h0 < D / 16; h0 += 2) {
      i32x4 kf[2][2];
      read_k<T, C, D, 2>(ks, h0, l32, half, kf);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) s[kt] = mfma<T>(kf[kt][i], qf[h0 + i], s[kt]);
    }
    // Every K fragment has been read: the next block's K may land.
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    if (more) {
      there_next = place(kb + NW, entry);
      entry = my_entry(min(kb + 2 * NW, end - 1));
      __builtin_amdgcn_sched_barrier(0);
      issue(kbase, ks, false);
    }
    __builtin_amdgcn_sched_barrier(0);

    constexpr int kp = kParts<T, C>;
    i32x4 pf[4][kp];
    uint64_t seen = 0;
    if (masked) seen = seen_bits(a, b, t, sp.ctx, kb * kBlock, there) >> (4 * half);
    softmax<C, D>(s, st, scale_log2, sc, half, masked, seen);
    // P before the wait; in two parts, which take twice the registers, they are
    // made as the products need them.
    if constexpr (kp == 1) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        pack_p<T, C>(s, kk, pf[kk]);
        asm volatile("" ::"v"(pf[kk][0]));
      }
    } else {
      asm volatile("" ::"v"(s[0]), "v"(s[1]));
    }
    // V landed (only the next block's K may be in flight).
    __builtin_amdgcn_sched_barrier(0);
    if (more) __builtin_amdgcn_s_waitcnt((nv & 15) | ((nv >> 4) << 14) | (7 << 4) | (15 << 8));
    else __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));
    __builtin_amdgcn_sched_barrier(0);
    if (masked) {
      const uint64_t nans = k8 ? nan_scales(value_scale) & there : 0;
      for (uint64_t bad = not_finite<T, C, D>(vs, lane) | nans; bad; bad &= bad - 1) {
        const int key = __builtin_ctzll(bad);
        if ((there >> key) & 1) add_key<T, C, D>(vs, key, s, seen, (nans >> key) & 1, l32, half, st);
        clear_key<C, D>(vs, key, lane);
      }
    }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if constexpr (kp > 1) pack_p<T, C>(s, kk, pf[kk]);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const i32x4 vf = read_v<kProduct<T, C>, C, D>(smem, v_at, kk, dt);
#pragma unroll
        for (int i = 0; i < kp; ++i) st.o[dt] = mfma<kProduct<T, C>>(vf, pf[kk][i], st.o[dt]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    if (more) issue(vbase, vs, true);
    there = there_next;
    __builtin_amdgcn_sched_barrier(0);
  }
  const float l = pair_sum(st.l);

  // Combine the waves: O_w as padded rows, then m and l.
  __syncthreads();
  constexpr int kPitch = D + 4;
  float* po = (float*)smem;
  float* pm = po + NW * 32 * kPitch;
  {
    float* w = po + (wave * 32 + l32) * kPitch;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4*)(w + dt * 32 + 8 * g + 4 * half) =
            f32x4{st.o[dt][4 * g], st.o[dt][4 * g + 1], st.o[dt][4 * g + 2], st.o[dt][4 * g + 3]};
    if (half == 0) {
      pm[(wave * 32 + l32) * 2] = st.m;
      pm[(wave * 32 + l32) * 2 + 1] = l;
    }
  }
  __syncthreads();
  const int live = min(32, rows - tile * 32);
  const int splits = (blocks_all + per - 1) / per;  // of this sequence
  const KeysPart kp = keys_part<D>(part, (int64_t)bk * row_tiles + tile);
  for (int idx = tid; idx < live * (D / 4); idx += 64 * NW) {
    const int q = idx / (D / 4), d = idx % (D / 4) * 4;
    float M = -__builtin_inff(), L = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, pm[(w * 32 + q) * 2]);
    const float nM = M == -__builtin_inff() ? 0.0f : M;
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(pm[(w * 32 + q) * 2] - nM);
      L = __builtin_fmaf(f, pm[(w * 32 + q) * 2 + 1], L);
      acc += *(const f32x4*)(po + (w * 32 + q) * kPitch + d) * f;
    }
    if (splits > 1) {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, acc), kp.rs, (q * D + d) * 4,
                                             split * kp.bytes, kDeviceScope);
      if (d == 0) {
        const i32x2 ml = {__builtin_bit_cast(int, M), __builtin_bit_cast(int, L)};
        __builtin_amdgcn_raw_buffer_store_b64(ml, kp.rs, (32 * D + 2 * q) * 4, split * kp.bytes, kDeviceScope);
      }
      continue;
    }
    const int r = tile * 32 + q, rt = r / group, rh = kvh * group + r % group;
    store4<T>(a, b * a.o_sb + rh * a.o_sh + rt * a.o_ss + d, acc * inverse_sum(L));
    if (a.lse && d == 0) a.lse[(b * a.heads + rh) * a.tokens + rt] = lse_of(M, L);
  }
  if (splits <= 1) return;
  // The last workgroup of the tile's splits to arrive sums them, in split order.
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0): the stores are acknowledged
  __syncthreads();
  int* last = (int*)smem;
  if (tid == 0) *last = arrive(kp.word, splits);
  __syncthreads();
  if (!*last) return;
  for (int idx = tid; idx < live * (D / 4); idx += 64 * NW) {
    const int q = idx / (D / 4), d = idx % (D / 4) * 4;
    float M = -__builtin_inff(), L = 0.0f;
    f32x4 acc = {0, 0, 0, 0};
    for (int s0 = 0; s0 < splits; s0 += 4) {
      f32x2 ml[4];
      f32x4 o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = min(s0 + i, splits - 1) * kp.bytes;
        ml[i] = __builtin_bit_cast(
            f32x2, __builtin_amdgcn_raw_buffer_load_b64(kp.rs, (32 * D + 2 * q) * 4, at, kDeviceScope));
        o[i] = __builtin_bit_cast(
            f32x4, __builtin_amdgcn_raw_buffer_load_b128(kp.rs, (q * D + d) * 4, at, kDeviceScope));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (s0 + i >= splits) continue;
        const float m = ml[i][0], n = fmaxf(M, m);
        const float nn = n == -__builtin_inff() ? 0.0f : n;
        const float fa = __builtin_amdgcn_exp2f(M - nn), fb = __builtin_amdgcn_exp2f(m - nn);
        L = L * fa + ml[i][1] * fb;
        acc = acc * fa + o[i] * fb;
        M = n;
      }
    }
    const int r = tile * 32 + q, rt = r / group, rh = kvh * group + r % group;
    store4<T>(a, b * a.o_sb + rh * a.o_sh + rt * a.o_ss + d, acc * inverse_sum(L));
    if (a.lse && d == 0) a.lse[(b * a.heads + rh) * a.tokens + rt] = lse_of(M, L);
  }
#endif  // __HIP_DEVICE_COMPILE__
}

template <Elt T, Elt C, int D>
static hipError_t launch_keys(const TreeAttnArgs& a, const Part& p, hipStream_t stream) {
  auto kern = tree_keys_kernel<T, C, D>;
  constexpr int lds = keys_lds<C, D>(), threads = 64 * kKeyWaves<C, D>;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  static const hipError_t attr =
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (attr != hipSuccess) return attr;
  const int group = a.heads / a.cache.kv_heads;
  const int64_t tiles = ((int64_t)a.tokens * group + 31) / 32;
  const int64_t units = a.batch * a.cache.kv_heads * p.splits;
  if (units * tiles > UINT32_MAX / threads) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kern, dim3((unsigned)(units * tiles)), dim3(threads), lds, stream, a, p, (int)tiles,
                     (int)units);
  return hipGetLastError();
}

// ---- many rows: the waves share the keys ----------------------------------------------

// NW tiles of 32 rows per workgroup, one a wave; K and V of a key block in LDS
// for all of them, in 16 bits (codes are widened once, on their way), double
// buffered.  Of a block, two waves of a SIMD take 2048 cycles of products and 1800 (8-bit rows:
// 2500) of vector instructions, eight waves 2048 of LDS reads, of 4400 (5600) in all: the
// barrier keeps the waves in step, so they overlap little.  512 tokens of b2 h32/8 d128
// bf16 over 32k keys: 550 us, 990 TFLOP/s, matrix cores busy 48% of the cycles; 64 tokens of b8
// over 16k keys of e4m3: 190 us, 723 TFLOP/s (with f16 queries, two second products: 241).
template <Elt T, Elt C, int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void tree_tile_kernel(TreeAttnArgs a, Part part, int row_blocks,
                                                            int units) {
#if defined(__HIP_DEVICE_COMPILE__)
  using G = Geom<T, D>;
  constexpr bool k8 = is8(C);
  constexpr Elt VT = kProduct<T, C>;  // of V in LDS
  constexpr int kBuf = 2 * G::kTile;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int64_t* offs = (int64_t*)(smem + 2 * kBuf);  // [2][64]
  float* scales = (float*)(offs + 128);         // [2][192]: put_scale's, then the value's as they are
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int unit, rb;
  place_unit(blockIdx.x, units, row_blocks, unit, rb);
  rb = row_blocks - 1 - rb;  // the last rows, which see most keys, first
  const int split = unit % part.splits, bk = unit / part.splits;
  const int64_t b = bk / a.cache.kv_heads;
  const int kvh = bk % a.cache.kv_heads, group = a.heads / a.cache.kv_heads;
  const kv::Span sp = kv::span_of(a.ctx_len, a.new_len, a.tokens, b);
  const int rows = sp.fresh * group;
  if (sp.ctx < 0 || rb * 32 * NW >= rows) return;
  const int keys = keys_of(a.cache.capacity, sp);
  const int blocks_all = (keys + kBlock - 1) / kBlock;
  const int per = blocks_per_split(part, blocks_all);
  if (split > 0 && split * per >= blocks_all) return;
  const int row0 = (rb * NW + wave) * 32;  // this wave's first row
  const int row = min(row0 + l32, rows - 1), t = row / group, h = kvh * group + row % group;
  // Without a mask no row of the workgroup sees past its last token.
  int end = min(blocks_all, (split + 1) * per);
  int t_wave = sp.fresh;  // the last token of this wave
  if (!a.mask) {
    const int t_last = (min(rows, (rb + 1) * 32 * NW) - 1) / group;
    end = min((int64_t)end, (sp.ctx + t_last + kBlock) / kBlock);
    t_wave = min(row0 + 31, rows - 1) / group;
  }
  const int begin = split * per;

  i32x4 qf[D / 16];
  load_q<T, D>((const char*)a.q + (b * a.q_sb + h * a.q_sh + t * a.q_ss) * 2, half, qf);
  const float scale_log2 = a.sm_scale * kLog2eF;
  const char* kbase = (const char*)a.cache.k;
  const char* vbase = (const char*)a.cache.v;

  auto my_entry = [&](int kb) { return entry_of(a.cache, a.ctx_len, b, kb * kBlock + lane); };
  int64_t my_scale = 0;
  // Row offsets of a block, by wave 0 for all; every wave keeps which keys exist.
  auto place = [&](int kb, int entry) __attribute__((always_inline)) {
    const Place p = place_of(a.cache, bytes_of(C), b, kvh, kb * kBlock + lane, keys, entry);
    if (wave == 0) offs[(kb & 1) * 64 + lane] = p.row;
    my_scale = p.scale;
    return __builtin_amdgcn_ballot_w64(p.there);
  };
  // 16 bits: 1 KiB per load instruction to LDS.
  constexpr int kIns = G::kLoads, kPer = (kIns + NW - 1) / NW;
  const int lrow = lane / G::kKC, lchunk = lane % G::kKC;
  auto issue = [&](int kb) __attribute__((always_inline)) {
    char* dst = smem + (kb & 1) * kBuf;
    const int64_t* o = offs + (kb & 1) * 64;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int n = wave * kPer + i;
      if (n >= kIns) continue;  // wave-uniform
      const int r = n * G::kRows + lrow;
      const int64_t at = o[r];
      __builtin_amdgcn_global_load_lds((global_ptr)(kbase + at + ((lchunk ^ G::swz_k(r)) << 4)),
                                       (lds_ptr)(dst + n * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((global_ptr)(vbase + at + ((lchunk ^ G::swz_v(r)) << 4)),
                                       (lds_ptr)(dst + G::kTile + n * 1024), 16, 0, 0);
    }
  };
  // Codes: 16 of them per thread and piece, widened on the way to LDS.
  constexpr int kPieces = 4 * D, kMine = (kPieces + 64 * NW - 1) / (64 * NW), kC8 = D / 16;
  i32x4 kw[kMine], vw[kMine];
  float my_value = 0.0f;
  auto fetch = [&](int kb) __attribute__((always_inline)) {
    const int64_t* o = offs + (kb & 1) * 64;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int p = i * 64 * NW + tid;
      if (kPieces % (64 * NW) && p >= kPieces) continue;
      const int64_t at = o[p / kC8] + (p % kC8) * 16;
      kw[i] = *(const i32x4*)(kbase + at);
      vw[i] = *(const i32x4*)(vbase + at);
    }
    if (wave < 2) my_value = (wave == 0 ? a.cache.k_scale : a.cache.v_scale)[my_scale];
  };
  auto widen = [&](int kb, bool masked) __attribute__((always_inline)) {
    char* dst = smem + (kb & 1) * kBuf;
    // Its LDS addresses are formed here, a block at a time: kept over the loop
    // they would take registers that it does not have.
    int first = tid;
    asm volatile("" : "+v"(first));
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int p = i * 64 * NW + first;
      if (kPieces % (64 * NW) && p >= kPieces) continue;
      const int r = p / kC8, c = 2 * (p % kC8);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        *(i32x4*)(dst + r * G::kRB + (((c + e) ^ G::swz_k(r)) << 4)) =
            widen8<T, C>(kw[i][2 * e], kw[i][2 * e + 1]);
        *(i32x4*)(dst + G::kTile + r * G::kRB + (((c + e) ^ G::swz_v(r)) << 4)) =
            widen8<VT, C>(vw[i][2 * e], vw[i][2 * e + 1]);
      }
    }
    float* sc = scales + (kb & 1) * 192;
    if (wave < 2) put_scale(sc, lane, my_value, wave == 0, scale_log2, masked);
    if (wave == 1) sc[128 + lane] = my_value;
  };

  // Whether some row may not see all keys of a block.
  auto masked_of = [&](int kb, uint64_t there) { return there != ~0ull || (int64_t)(kb + 1) * kBlock > sp.ctx; };

  const uint32_t v_lane = v_offset<T, D>(lane);
  State<D> st;
  clear(st);
  // Table entries of the first blocks; Q has landed with them, on every path
  // into the loop, so that nothing in it waits for a load by accident.
  const int entry0 = my_entry(begin), entry1 = my_entry(begin + 1);
  int entry = my_entry(begin + 2);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) asm volatile("" ::"v"(qf[i]), "v"(entry0), "v"(entry1), "v"(entry));
  __builtin_amdgcn_s_waitcnt(0);
  uint64_t there = 0, there1 = 0;
  if (begin < end) {
    there = place(begin, entry0);
    const int64_t scale0 = my_scale;
    there1 = place(begin + 1, entry1);
    const int64_t scale1 = my_scale;
    __syncthreads();
    if constexpr (k8) {
      my_scale = scale0;
      fetch(begin);
      my_scale = scale1;
      widen(begin, masked_of(begin, there));
    } else {
      issue(begin);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  for (int kb = begin; kb < end; ++kb) {
    const bool more = kb + 1 < end;
    const char* ks = smem + (kb & 1) * kBuf;
    char* vs = smem + (kb & 1) * kBuf + G::kTile;
    const uint32_t v_at = (uint32_t)((kb & 1) * kBuf + G::kTile) + v_lane;
    const bool masked = masked_of(kb, there);
    // The same in every wave: all of them look at the same tile.
    uint64_t bad = 0, nans = 0;
    if (masked) {
      if constexpr (k8) nans = nan_scales(scales[(kb & 1) * 192 + 128 + lane]) & there;
      bad = not_finite<VT, VT, D>(vs, lane) | nans;
    }
    if (more) {
      if constexpr (k8) fetch(kb + 1);
      else issue(kb + 1);
    }
    const bool idle = row0 >= rows || (!a.mask && (int64_t)kb * kBlock > sp.ctx + t_wave);
    if (!idle || bad) {
      // V fragments read ahead of the softmax: as many key steps as registers
      // allow (over codes the staged loads take some).
      constexpr int kEarly = D < 128 ? 4 : k8 ? 0 : 2;
      f32x16 s[2] = {f32x16{}, f32x16{}};
      i32x4 vf[4][D / 32];
      if constexpr (k8 && D == 128) {
#pragma unroll
        for (int h0 = 0; h0 < D / 16; h0 += 2) {
          i32x4 kf[2][2];
          read_k<T, T, D, 2>(ks, h0, l32, half, kf);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) s[kt] = mfma<T>(kf[kt][i], qf[h0 + i], s[kt]);
        }
      } else {
        constexpr int H1 = D / 32;
        i32x4 kf0[2][H1], kf1[2][H1];
        read_k<T, T, D, H1>(ks, 0, l32, half, kf0);
        __builtin_amdgcn_sched_barrier(0);
        read_k<T, T, D, H1>(ks, H1, l32, half, kf1);
#pragma unroll
        for (int i = 0; i < H1; ++i)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) s[kt] = mfma<T>(kf0[kt][i], qf[i], s[kt]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt) vf[kk][dt] = read_v<VT, VT, D>(smem, v_at, kk, dt);
#pragma unroll
        for (int i = 0; i < H1; ++i)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) s[kt] = mfma<T>(kf1[kt][i], qf[H1 + i], s[kt]);
#pragma unroll
        for (int kk = 2; kk < kEarly; ++kk)
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt) vf[kk][dt] = read_v<VT, VT, D>(smem, v_at, kk, dt);
      }
      __builtin_amdgcn_sched_barrier(0);
      constexpr int kp = kParts<T, C>;
      i32x4 pf[4][kp];
      uint64_t seen = 0;
      if (masked) seen = seen_bits(a, b, t, sp.ctx, kb * kBlock, there) >> (4 * half);
      softmax<C, D>(s, st, scale_log2, scales + (kb & 1) * 192, half, masked, seen);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) pack_p<T, C>(s, kk, pf[kk]);
      if (bad) {
        for (uint64_t left = bad & there; left; left &= left - 1)
          add_key<VT, VT, D>(vs, __builtin_ctzll(left), s, seen, (nans >> __builtin_ctzll(left)) & 1, l32, half, st);
        __syncthreads();
        if (wave == 0)
          for (uint64_t left = bad; left; left &= left - 1) clear_key<T, D>(vs, __builtin_ctzll(left), lane);
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kEarly; ++kk)
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt) vf[kk][dt] = read_v<VT, VT, D>(smem, v_at, kk, dt);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = kEarly; kk < 4; ++kk)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) vf[kk][dt] = read_v<VT, VT, D>(smem, v_at, kk, dt);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int i = 0; i < kp; ++i) st.o[dt] = mfma<VT>(vf[kk][dt], pf[kk][i], st.o[dt]);
    }
    if constexpr (k8)
      if (more) widen(kb + 1, masked_of(kb + 1, there1));
    // Offsets of the block after the next, whose place in LDS this block's had.
    there = there1;
    there1 = place(kb + 2, entry);
    entry = my_entry(kb + 3);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }

  // Each lane holds half of its row's dims.
  const float l = pair_sum(st.l);
  if (row0 + l32 >= rows) return;
  const int64_t id = (b * a.heads + h) * a.tokens + t;
  if (per < blocks_all) {
    const int64_t at = id * part.splits + split;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4*)(part.o + at * D + dt * 32 + 8 * g + 4 * half) =
            f32x4{st.o[dt][4 * g], st.o[dt][4 * g + 1], st.o[dt][4 * g + 2], st.o[dt][4 * g + 3]};
    if (half == 0) part.ml[2 * at] = st.m, part.ml[2 * at + 1] = l;
    return;
  }
  const float f = inverse_sum(l);
  const int64_t o_row = b * a.o_sb + h * a.o_sh + t * a.o_ss;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4<T>(a, o_row + dt * 32 + 8 * g + 4 * half,
                f32x4{st.o[dt][4 * g], st.o[dt][4 * g + 1], st.o[dt][4 * g + 2], st.o[dt][4 * g + 3]} * f);
  if (a.lse && half == 0) a.lse[id] = lse_of(st.m, l);
#endif  // __HIP_DEVICE_COMPILE__
}

template <Elt T, Elt C, int D, int NW>
static hipError_t launch_tile(const TreeAttnArgs& a, const Part& p, hipStream_t stream) {
  auto kern = tree_tile_kernel<T, C, D, NW>;
  constexpr int lds = 4 * Geom<T, D>::kTile + 1024 + 1536;
  static const hipError_t attr =
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (attr != hipSuccess) return attr;
  const int group = a.heads / a.cache.kv_heads;
  const int64_t blocks = ((int64_t)a.tokens * group + 32 * NW - 1) / (32 * NW);
  const int64_t units = a.batch * a.cache.kv_heads * p.splits;
  if (units * blocks > UINT32_MAX / (64 * NW)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kern, dim3((unsigned)(units * blocks)), dim3(64 * NW), lds, stream, a, p, (int)blocks,
                     (int)units);
  return hipGetLastError();
}

template <Elt T, Elt C, int D>
static hipError_t launch_mfma(const TreeAttnArgs& a, const Part& p, hipStream_t s) {
  if (a.kernel == plan::TreeKernel::Keys) return launch_keys<T, C, D>(a, p, s);
  if constexpr (D == 128)
    if (a.kernel == plan::TreeKernel::Tile8) return launch_tile<T, C, D, 8>(a, p, s);
  return launch_tile<T, C, D, 4>(a, p, s);
}

template <int D> hipError_t tree_mfma_dispatch(const TreeAttnArgs& a, const Part& p, hipStream_t s) {
  const bool bf = a.dtype == Elt::BF16;
  switch (a.cache.kind) {
    case Elt::E4M3:
      return bf ? launch_mfma<Elt::BF16, Elt::E4M3, D>(a, p, s) : launch_mfma<Elt::F16, Elt::E4M3, D>(a, p, s);
    case Elt::I8:
      return bf ? launch_mfma<Elt::BF16, Elt::I8, D>(a, p, s) : launch_mfma<Elt::F16, Elt::I8, D>(a, p, s);
    default:
      return bf ? launch_mfma<Elt::BF16, Elt::BF16, D>(a, p, s) : launch_mfma<Elt::F16, Elt::F16, D>(a, p, s);
  }
}

}  // namespace tree
}  // namespace frisk
