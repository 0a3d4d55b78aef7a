// Verification of drafted tokens: which branch of a tree the target's
// probabilities accept under given random numbers, and the token after it.
//
// Probabilities are compared with random numbers, so they are computed in 64
// bits: a weight is 2^t, t = (x - max) log2(e) / T, from a polynomial of degree 9
// on the fraction of t, off by 2^-45 of it, and sums are of doubles.  The vector
// unit does as many 64-bit as 32-bit multiply-adds, so a weight costs 17
// instructions, 16 of them of 64 bits.
//
// Three launches.  (1) The rows of nodes that have children, a wave for each
// segment of a row, without a barrier: its maximum and sum.  (2) A workgroup per tree combines
// them, takes every node's probability given its parent, and walks from the root.
// (3) What is left of the probabilities at the last node, by segments: the same kernel as (1);
// segments that no rejected token lies in have their sums from (1).  The tree's last workgroup to
// arrive there finds the segment, then the element, in which the sum passes the last random
// number (a launch of its own took 0.7 us longer).  (2) set the count of arrivals to 0, so that an
// arrival is one addition; exchanges with a word of any content took 1 us each, one after the
// other.  Short rows (plan::kVerifyShort): (3) is a part of (2).  Trees of one node: (3)
// without arrivals and the search as a second launch, or both by one workgroup a row
// (plan::verify_alone).

#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace frisk {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kWalkers = plan::kVerifyTreeThreads;  // threads of a walk
constexpr int kAlone = plan::kVerifyTreeThreads;    // threads of a row in a launch of its own

// A segment's or a row's largest logit, its first place, and the sum of weights
// 2^((x - m) c): NaN if the row gives no probabilities (it holds a NaN or +infinity).
struct Stat {
  double s;
  float m;
  int at;
};
// A segment of the last node's row: sums of what is left there, and of what was left
// before the last rejection; both relative to m.
struct Rest {
  double s, whole;
  float m;
  int at;
};
// Where a walk ended.
struct End {
  double inverse;  // of the sum of the row's weights
  float m;       // its maximum
  int node;      // -1: the tree takes no part, -2: no token
  int rounds;    // children rejected there
  int greedy;    // the token, if the temperature is 0 and it is known; -1: sample, -2: largest
  int arrived;   // workgroups of (3) that have written their rests
};

struct Layout {
  Stat* stats;  // [batch][tokens][segments]
  Rest* rest;   // [batch][segments]
  End* end;     // [batch]
  double* list;  // [batch][tokens] rejected tokens or, of dense drafts, 1 over what their rest summed to
};
__host__ __device__ inline int64_t up16(int64_t n) { return (n + 15) & ~15ll; }
__device__ __forceinline__ Layout layout(const VerifyArgs& a) {
  char* p = (char*)a.workspace;
  Layout l;
  l.stats = (Stat*)p;
  p += up16((int64_t)a.batch * a.tokens * a.segments * sizeof(Stat));
  l.rest = (Rest*)p;
  p += up16((int64_t)a.batch * a.segments * sizeof(Rest));
  l.end = (End*)p;
  p += up16((int64_t)a.batch * sizeof(End));
  l.list = (double*)p;
  return l;
}

constexpr double kPoly[9] = {1.3259165418921631e-06, 1.5252831553412485e-05, 0.000154034371500767,
                             0.0013333557934657732,  0.009618129186021637,   0.055504108666170275,
                             0.2402265069570673,     0.6931471805599285,     1.0};
constexpr double kLead = 1.0175586973078281e-07;  // the polynomial's first coefficient
constexpr double kRound = 0x1.8p52;                // t + kRound has rint(t) in its low bits

// 2^f for |f| <= 1/2: 1 + f p(f), p of degree 8 with the least largest relative
// error of the whole, 2^-45; 1 at f = 0.
__device__ __forceinline__ double pow2_fraction(double f, double lead = kLead) {
  double p = lead;
#pragma unroll
  for (int i = 0; i < 9; ++i) p = __builtin_fma(p, f, kPoly[i]);
  return p;
}
// x 2^k for the k in the low bits of `shifted`.  (Written out, the 32-bit addition to
// the exponent's half became six instructions of a 64-bit one.)
__device__ __forceinline__ double scale_by(double x, double shifted) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, shifted);
  uint32_t hi = (uint32_t)(u >> 32);
  asm("v_lshl_add_u32 %0, %1, 20, %0" : "+v"(hi) : "v"(k));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)u);
}
// 2^t for |t| <= 1000.
__device__ __forceinline__ double pow2_any(double t) {
  const double shifted = t + kRound;
  return scale_by(pow2_fraction(t - (shifted - kRound)), shifted);
}
// 2^t for t <= 0: the exponent is added to the bits of 2^f.  0 below -1000 and for NaN.
__device__ __forceinline__ double pow2(double t) {
  const double w = pow2_any(__builtin_fmax(t, -1000.0));
  return t > -1000.0 ? w : 0.0;
}

// Weights of a segment's elements for their sum: 2^-900 in the place of smaller ones, 16
// instructions of 64 bits.  A v_fma takes one scalar operand, so the other
// constants of an operation are kept in vector registers.
struct Weigh {
  double top, factor, round, lead, least;
  __device__ __forceinline__ Weigh(float m, double f)
      : top((double)m), factor(f), round(kRound), lead(kLead), least(-900.0 / f) {
    asm volatile("" : "+v"(factor), "+v"(round), "+v"(lead));
  }
  // The sum of W elements' weights, step by step for all of them: the steps of one
  // wait for each other.
  template <int W> __device__ __forceinline__ double sum(const float* x) const {
    double f[W], shifted[W], p[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const double d = __builtin_fmax((double)x[k] - top, least);
      shifted[k] = __builtin_fma(d, factor, round);
      f[k] = __builtin_fma(d, factor, round - shifted[k]);
      p[k] = lead;
    }
#pragma unroll
    for (int i = 0; i < 9; ++i) {
#pragma unroll
      for (int k = 0; k < W; ++k) p[k] = __builtin_fma(p[k], f[k], kPoly[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 0; k < W; ++k) p[k] = scale_by(p[k], shifted[k]);
#pragma unroll
    for (int n = W / 2; n; n /= 2)
#pragma unroll
      for (int k = 0; k < n; ++k) p[k] += p[k + n];
    return p[0];
  }
};

// log2(e) / T of a tree; 0: its temperature is 0, the largest logit wins.
__device__ __forceinline__ double factor_of(const VerifyArgs& a, int64_t b) {
  if (!a.temperature) return 1.4426950408889634;
  const float t = a.temperature[b];
  return t > 0.0f ? 1.4426950408889634 / (double)t : 0.0;
}
__device__ __forceinline__ int nodes_of(const VerifyArgs& a, int64_t b) {
  return a.new_len ? min(max(a.new_len[b], 0), a.tokens) : a.tokens;
}
// The end of a tree of one node, which is not walked.
__device__ __forceinline__ End root_end(const VerifyArgs& a, int64_t b) {
  return End{0.0, 0.0f, nodes_of(a, b) < 1 ? -1 : 0, 0, -1, 0};
}

template <Elt E> struct Row {
  using T = typename EltInfo<E>::T;
  static constexpr int N = 16 / EltInfo<E>::bytes;  // elements of 16 B
  const T* p;
  int n, head, full;  // elements; those before the first 16-B boundary; whole pieces behind them
};
template <Elt E> __device__ __forceinline__ Row<E> row_of(const VerifyArgs& a, int64_t b, int64_t t) {
  using R = Row<E>;
  R r;
  r.p = (const typename R::T*)a.logits + (b * a.sb + t * a.st);
  r.n = a.vocab;
  const int off = (int)((uintptr_t)r.p & 15);
  r.head = min(off ? (16 - off) / EltInfo<E>::bytes : 0, r.n);
  r.full = (r.n - r.head) / R::N;
  return r;
}

// A segment's elements are PIECES whole pieces of 16 B a lane, in the order (piece,
// lane, element); the first segment's start with the row's head, the last one's end
// with its tail, one element a lane.
template <Elt E> __device__ __forceinline__ i32x4 raw_piece(const Row<E>& r, int piece) {
  return *(const i32x4*)(r.p + r.head + (int64_t)piece * Row<E>::N);
}
template <Elt E> __device__ __forceinline__ void widen_piece(i32x4 w, float (&x)[Row<E>::N]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t word = (uint32_t)w[i];
    if constexpr (E == Elt::F32) {
      x[i] = __builtin_bit_cast(float, word);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint16_t h = (uint16_t)(word >> (16 * e));
        x[2 * i + e] = E == Elt::BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
      }
    }
  }
}
template <Elt E> __device__ __forceinline__ void load_piece(const Row<E>& r, int piece, float (&x)[Row<E>::N]) {
  widen_piece<E>(raw_piece<E>(r, piece), x);
}
// The loose element of a lane in segment g, or -1: the head's in the first segment
// (lanes 0 ..), the tail's in the last (lanes 32 ..).
template <Elt E> __device__ __forceinline__ int loose_of(const VerifyArgs& a, const Row<E>& r, int g, int lane) {
  if (g == 0 && lane < r.head) return lane;
  const int tail = r.head + r.full * Row<E>::N;
  if (g == a.segments - 1 && lane >= 32 && tail + lane - 32 < r.n) return tail + lane - 32;
  return -1;
}

// ---- sums and so on over a wave ----------------------------------------------------

// The values of two lanes of a pair, the same on both: lanes l ^ 1, l ^ 2, mirrored in
// 8 and in 16, l ^ 16, l ^ 32.
template <int STEP> __device__ __forceinline__ uint2 pair_of(uint32_t x) {
  if constexpr (STEP < 4) {
    constexpr int kControl[4] = {0xB1, 0x4E, 0x141, 0x140};
    return {x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kControl[STEP], 0xf, 0xf, true)};
  } else if constexpr (STEP == 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return {(uint32_t)r[0], (uint32_t)r[1]};
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return {(uint32_t)r[0], (uint32_t)r[1]};
  }
}
template <int STEP = 0> __device__ __forceinline__ double wave_sum(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint2 lo = pair_of<STEP>((uint32_t)u), hi = pair_of<STEP>((uint32_t)(u >> 32));
  x = __builtin_bit_cast(double, (uint64_t)hi.x << 32 | lo.x) + __builtin_bit_cast(double, (uint64_t)hi.y << 32 | lo.y);
  if constexpr (STEP < 5) return wave_sum<STEP + 1>(x);
  else return x;
}
// NaN if one of them is.
template <int STEP = 0> __device__ __forceinline__ float wave_max(float x) {
  const uint2 p = pair_of<STEP>(__builtin_bit_cast(uint32_t, x));
  x = __builtin_elementwise_maximum(__builtin_bit_cast(float, p.x), __builtin_bit_cast(float, p.y));
  if constexpr (STEP < 5) return wave_max<STEP + 1>(x);
  else return x;
}
template <int STEP = 0> __device__ __forceinline__ int wave_min(int x) {
  const uint2 p = pair_of<STEP>((uint32_t)x);
  x = min((int)p.x, (int)p.y);
  if constexpr (STEP < 5) return wave_min<STEP + 1>(x);
  else return x;
}
__device__ __forceinline__ double shfl_d(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)u, lane), hi = (uint32_t)__shfl((int)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The sum over the lanes up to this one.
__device__ __forceinline__ double wave_scan(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double y = shfl_d(x, max(lane - d, 0));
    if (lane >= d) x += y;
  }
  return x;
}
// The value of lane k, the same in all lanes.
__device__ __forceinline__ float lane_f(float x, int k) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), k));
}
__device__ __forceinline__ double lane_d(double x, int k) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, k), hi = __builtin_amdgcn_readlane((int)(u >> 32), k);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// ---- segments of a row --------------------------------------------------------------

// What is left of a probability p after `rounds` children drawn independently from q were
// rejected, whose rests' sums have the inverses z[0 ..]; a rest without mass (0) leaves it as
// it was.  (With divisions in their place a tree of 8 nodes over 47565 bf16 took 41 us, not 37.)
// A pass of the walk calls it for every element, so many rejections at one node cost their square: 50257
// f32 logits 45 us with 2, 222 with 8, 7.4 ms with 64.
__device__ __forceinline__ double left_of(double p, double q, const double* z, int rounds) {
  for (int i = 0; i < rounds; ++i) {
    const double rest = __builtin_fmax(p - q, 0.0), inverse = z[i];
    if (inverse > 0.0) p = rest * inverse;
  }
  return p;
}
// The same, and before the last rejection, whose rest has no sum yet.
struct Left {
  double now, was;
};
__device__ __forceinline__ Left dense_left(double p, float q, const double* z, int rounds) {
  const double was = left_of(p, (double)q, z, rounds - 1);
  return {__builtin_fmax(was - (double)q, 0.0), was};
}

// A segment's elements as they are loaded.
template <Elt E, int PIECES> struct Held {
  i32x4 w[PIECES];
  float extra;
};
template <Elt E, int PIECES>
__device__ __forceinline__ void load_segment(const VerifyArgs& a, const Row<E>& r, int g, Held<E, PIECES>& h) {
  const int lane = threadIdx.x & 63, base = g * PIECES * 64 + lane;
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
    if (base + i * 64 < r.full) h.w[i] = raw_piece<E>(r, base + i * 64);
  const int loose = loose_of<E>(a, r, g, lane);
  h.extra = loose >= 0 ? (float)r.p[loose] : -__builtin_inff();
}

// The statistics of segment g, known to all lanes, without the tokens list[0 .. gone).
template <Elt E, int PIECES>
__device__ __forceinline__ Stat segment_stat(const VerifyArgs& a, const Row<E>& r, int g, const Held<E, PIECES>& h,
                                             double factor, const double* list, int gone) {
  constexpr int N = Row<E>::N;
  const int lane = threadIdx.x & 63, base = g * PIECES * 64 + lane;
  float x[PIECES][N];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    if (base + i * 64 < r.full) {
      widen_piece<E>(h.w[i], x[i]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[i][e] = -__builtin_inff();
    }
  }
  const int loose = loose_of<E>(a, r, g, lane);
  float m = -__builtin_inff(), extra = h.extra;
  for (int k = 0; k < gone; ++k) {
    const int v = (int)list[k];
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (v == r.head + (base + i * 64) * N + e) x[i][e] = m;
    if (v == loose) extra = m;
  }
  // The maximum of a row with a NaN is NaN.
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) m = __builtin_elementwise_maximum(m, x[i][e]);
  m = wave_max(__builtin_elementwise_maximum(m, extra));
  double s = 0.0;
  int at = INT32_MAX;
  if (m > -__builtin_inff()) {
    if (factor == 0.0) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (x[i][e] == m) at = min(at, r.head + (base + i * 64) * N + e);
      if (extra == m) at = min(at, loose);
      at = wave_min(at);
      s = 1.0;
    } else {
      const Weigh weigh(m, factor);
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (base + i * 64 < r.full)
#pragma unroll
          for (int e = 0; e < N; e += 4) s += weigh.template sum<4>(x[i] + e);
      if (loose >= 0) s += weigh.template sum<1>(&extra);
      s = wave_sum(s);
    }
  }
  if (!(m < __builtin_inff())) s = __builtin_nan("");
  return Stat{s, m, at};
}

// Segment g of what dense drafts' rejection left at a tree's last node.
template <Elt E, int PIECES>
__device__ __forceinline__ Rest segment_rest(const VerifyArgs& a, const Row<E>& r, int64_t b, int g, const End& e,
                                             const double* list, double factor) {
  constexpr int N = Row<E>::N;
  const int lane = threadIdx.x & 63;
  const float* q = a.draft_probs + b * a.qb + e.node * a.qt;
  const double top = (double)e.m;
  double s = 0.0, whole = 0.0;
  auto add = [&](float x, int v) {
    const Left w = dense_left(pow2(((double)x - top) * factor) * e.inverse, q[v], list, e.rounds);
    s += w.now;
    whole += w.was;
  };
#pragma unroll 1
  for (int i = 0; i < PIECES; ++i) {
    const int piece = (g * PIECES + i) * 64 + lane;
    if (piece >= r.full) break;
    float x[N];
    load_piece<E>(r, piece, x);
#pragma unroll
    for (int k = 0; k < N; ++k) add(x[k], r.head + piece * N + k);
  }
  const int loose = loose_of<E>(a, r, g, lane);
  if (loose >= 0) add((float)r.p[loose], loose);
  return Rest{wave_sum(s), wave_sum(whole), 0.0f, 0};
}

// ---- the token ---------------------------------------------------------------------

// Rests pass from one workgroup to another inside a launch, so past the L2 caches.
__device__ __forceinline__ void write_rest(Rest* p, const Rest& r) {
  const uint64_t at = (uint64_t)(uint32_t)r.at << 32 | __builtin_bit_cast(uint32_t, r.m);
  __hip_atomic_store((uint64_t*)p, __builtin_bit_cast(uint64_t, r.s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store((uint64_t*)p + 1, __builtin_bit_cast(uint64_t, r.whole), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store((uint64_t*)p + 2, at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Rest read_rest(const Rest* p) {
  const uint64_t s = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t w = __hip_atomic_load((const uint64_t*)p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t at = __hip_atomic_load((const uint64_t*)p + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return {__builtin_bit_cast(double, s), __builtin_bit_cast(double, w), __builtin_bit_cast(float, (uint32_t)at),
          (int)(at >> 32)};
}

// The token of tree b, by a workgroup, from the rests of its last node's segments.
template <Elt E, int PIECES, typename Read>
__device__ __forceinline__ void pick(const VerifyArgs& a, int64_t b, const End& e, double factor, const double* list,
                                     const Read& rest) {
  constexpr int N = Row<E>::N;
  static_assert(PIECES <= kWaves, "a piece of a segment for each wave");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool dense = e.rounds > 0 && a.draft_probs;
  __shared__ int chosen, use_whole;
  __shared__ double before, goal;
  __shared__ float top_at;
  if (wave == 0) {
    // A lane has a run of segments, the first of them held.
    const int per = (a.segments + 63) / 64, c0 = lane * per, c1 = min(c0 + per, a.segments);
    const Rest none = {0.0, 0.0, -__builtin_inff(), INT32_MAX}, held = c0 < c1 ? rest(c0) : none;
    auto of = [&](int c) { return c == c0 ? held : rest(c); };
    float m = held.m;
    for (int c = c0 + 1; c < c1; ++c) m = __builtin_elementwise_maximum(m, of(c).m);
    m = wave_max(m);
    auto scaled = [&](double s, float mc) {
      return s == 0.0 ? 0.0 : dense ? s : s * pow2(((double)mc - (double)m) * factor);
    };
    if (factor == 0.0) {
      int at = INT32_MAX;
      for (int c = c0; c < c1; ++c) {
        const Rest x = of(c);
        if (x.m == m) at = min(at, x.at);
      }
      at = wave_min(at);
      const bool none = !(m > -__builtin_inff() && m < __builtin_inff());
      if (lane == 0) a.token[b] = none ? -1 : at, chosen = -1;
    } else {
      double s = 0.0, w = 0.0;
      for (int c = c0; c < c1; ++c) {
        const Rest x = of(c);
        s += scaled(x.s, x.m), w += scaled(x.whole, x.m);
      }
      const double sums = wave_sum(s), wholes = wave_sum(w);
      const bool whole = dense && !(sums > 0.0);
      const double all = whole ? wholes : sums, want = (double)a.final_uniform[b] * all;
      if (!(all > 0.0) || all == __builtin_inf()) {
        // Nothing is left of one-hot drafts: the last one had it all.  Else the
        // row gives no probabilities.
        if (lane == 0) a.token[b] = all == 0.0 && e.rounds > 0 && !dense ? (int)list[e.rounds - 1] : -1, chosen = -1;
      } else {
        // The first lane, then segment, whose end passes `want`; the last one with any mass, if
        // rounding leaves none.
        const double mine = whole ? w : s, upto = wave_scan(mine);
        const uint64_t some = __builtin_amdgcn_ballot_w64(mine > 0.0);
        const uint64_t past = __builtin_amdgcn_ballot_w64(mine > 0.0 && upto > want);
        const int k = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
        if (lane == k) {
          double base = upto - mine, at = base;
          int g = -1;
          for (int c = c0; c < c1; ++c) {
            const Rest x = of(c);
            const double here = scaled(whole ? x.whole : x.s, x.m);
            if (!(here > 0.0)) continue;
            g = c, at = base;
            base += here;
            if (base > want) break;
          }
          chosen = g, before = at, goal = want, use_whole = whole, top_at = m;
        }
      }
    }
  }
  __syncthreads();
  const int g = chosen;
  if (g < 0) return;
  const Row<E> r = row_of<E>(a, b, e.node);
  const float* q = dense ? a.draft_probs + b * a.qb + e.node * a.qt : nullptr;
  const double top = (double)(dense ? e.m : top_at), want = goal;
  const bool whole = use_whole;
  auto weight = [&](float x) { return pow2(((double)x - top) * factor); };
  auto left = [&](double p, int v) {
    const Left w = dense_left(p * e.inverse, q[v], list, e.rounds);
    return whole ? w.was : w.now;
  };
  // The segment's elements in order: part 0 is the head (the first wave's), 1 + w wave
  // w's piece of each lane, and the last one the tail (the first wave's).
  constexpr int kParts = PIECES + 2;
  __shared__ double parts[kParts];
  const int piece = g * PIECES * 64 + tid, loose = wave == 0 ? loose_of<E>(a, r, g, lane) : -1;
  double w[N];
  float x[N];
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = -__builtin_inff();
  if (wave < PIECES && piece < r.full) load_piece<E>(r, piece, x);
  float extra = -__builtin_inff();
  if (loose >= 0) extra = (float)r.p[loose];
  const int first = r.head + piece * N;
  if (!dense)
    for (int i = 0; i < e.rounds; ++i) {
      const int v = (int)list[i];
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (v == first + k) x[k] = -__builtin_inff();
      if (v == loose) extra = -__builtin_inff();
    }
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = weight(x[k]);  // (0 of -infinity)
  double odd = weight(extra), sum = 0.0;
  if (dense) {
    if (wave < PIECES && piece < r.full)
#pragma unroll
      for (int k = 0; k < N; ++k) w[k] = left(w[k], first + k);
    if (loose >= 0) odd = left(odd, loose);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) sum += w[k];
  const double all = wave_sum(sum);
  const bool in_head = loose >= 0 && loose < r.head;
  const double heads = wave_sum(in_head ? odd : 0.0), tails = wave_sum(in_head ? 0.0 : odd);
  if (lane == 0 && wave < PIECES) parts[1 + wave] = all;
  if (tid == 0) parts[0] = heads, parts[kParts - 1] = tails;
  __syncthreads();
  // The part whose end passes `want` (the last one with a weight, if rounding leaves none).
  double base = before, at = before;
  int part = -1;
  for (int k = 0; k < kParts; ++k) {
    if (!(parts[k] > 0.0)) continue;
    part = k, at = base;
    base += parts[k];
    if (base > want) break;
  }
  const bool ends = part == 0 || part == kParts - 1;
  if (part < 0 || wave != (ends ? 0 : part - 1)) return;
  // Its elements, by lanes: the first that passes, or the last with a weight.
  if (ends) {
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = 0.0;
    if (in_head == (part == 0)) w[0] = odd;
    sum = w[0];
  }
  const int start = ends ? loose : first;
  at += wave_scan(sum) - sum;
  int found = INT32_MAX, last = -1;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    at += w[k];
    if (w[k] > 0.0) {
      last = start + k;
      if (at > want) found = min(found, start + k);
    }
  }
  found = wave_min(found);
  last = -wave_min(-last);
  if (lane == 0) a.token[b] = found != INT32_MAX ? found : last;
}

// Segment g of what is left at a tree's last node.  `held`: the segment, as loaded.
template <Elt E, int PIECES>
__device__ __forceinline__ Rest last_segment(const VerifyArgs& a, const Row<E>& r, int64_t b, int g, const End& e,
                                             const double* list, double factor, const Stat* stats,
                                             const Held<E, PIECES>& held) {
  constexpr int N = Row<E>::N;
  const int lane = threadIdx.x & 63;
  bool reuse = false;
  if (e.rounds > 0) {
    // One-hot drafts: a segment without a rejected token is as it was.
    const int lo = g ? r.head + g * PIECES * 64 * N : 0;
    const int hi = g == a.segments - 1 ? r.n : r.head + (g + 1) * PIECES * 64 * N;
    uint64_t any = 0;
    for (int i0 = 0; i0 < e.rounds && !any; i0 += 64) {
      const int v = i0 + lane < e.rounds ? (int)list[i0 + lane] : -1;
      any = __builtin_amdgcn_ballot_w64(v >= lo && v < hi);
    }
    reuse = !any;
  }
  const Stat st = reuse ? stats[g] : segment_stat<E, PIECES>(a, r, g, held, factor, list, e.rounds);
  return {st.s, st.s, st.m, st.at};
}

// `groups` workgroups have the segments of a row, each wave every (4 groups)-th one, the next
// one's loads under way: of every row whose node has children (last 0), or of the rows that
// the walks ended at.
template <Elt E, int PIECES>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs a, int groups, int last) {
  constexpr int N = Row<E>::N;
  const int lane = threadIdx.x & 63, step = groups * kWaves;
  uint32_t id = blockIdx.x;
  int g = __builtin_amdgcn_readfirstlane((int)(id % groups * kWaves + (threadIdx.x >> 6)));
  if (!last && g >= a.segments) return;
  id /= groups;
  const Layout l = layout(a);
  const int64_t b = last ? id : id / a.tokens;
  const double factor = factor_of(a, b);
  int t = last ? 0 : id % a.tokens, gone = 0;
  const double* list = l.list + b * a.tokens;
  Rest* rests = l.rest + b * a.segments;
  End e = {};
  if (last) {
    e = a.tokens > 1 ? l.end[b] : root_end(a, b);
    if (e.node < 0 || e.greedy >= 0) {
      if (a.tokens > 1 && e.node != -1 && blockIdx.x == b * groups && threadIdx.x == 0)
        a.token[b] = e.node < 0 ? -1 : e.greedy;
      return;
    }
    t = e.node;
    gone = e.rounds;
    if (gone > 0 && a.draft_probs) {
      const Row<E> r = row_of<E>(a, b, t);
      for (; g < a.segments; g += step) {
        const Rest rest = segment_rest<E, PIECES>(a, r, b, g, e, list, factor);
        if (lane == 0) write_rest(rests + g, rest);
      }
    }
  } else {
    // (Every wave looks for itself.)
    const int n = nodes_of(a, b);
    uint64_t child = 0;
    for (int i0 = t + 1; i0 < n && !child; i0 += 64)
      child = __builtin_amdgcn_ballot_w64(i0 + lane < n && a.parents[b * a.tokens + min(i0 + lane, n - 1)] == t);
    if (!child) return;
  }
  const Row<E> r = row_of<E>(a, b, t);
  Stat* stats = l.stats + (b * a.tokens + t) * a.segments;
  Held<E, PIECES> now, next;
  if (g < a.segments) load_segment<E, PIECES>(a, r, g, now);
  for (; g < a.segments; g += step) {
    if (g + step < a.segments) load_segment<E, PIECES>(a, r, g + step, next);
    if (last) {
      const Rest rest = last_segment<E, PIECES>(a, r, b, g, e, list, factor, stats, now);
      if (lane == 0) write_rest(rests + g, rest);
    } else {
      const Stat st = segment_stat<E, PIECES>(a, r, g, now, factor, nullptr, 0);
      if (lane == 0) stats[g] = st;
    }
    now = next;
  }
  // A walked tree's last workgroup to arrive picks the token.
  if (!last || a.tokens == 1) return;
  __shared__ int arrived;
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0): the stores are acknowledged
  __syncthreads();
  if (threadIdx.x == 0)
    arrived = __hip_atomic_fetch_add(&l.end[b].arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived == groups - 1)
    pick<E, PIECES>(a, b, e, factor, list, [&](int c) { return read_rest(rests + c); });
}

// What a walk writes of a tree of one node.
__device__ __forceinline__ void one_node(const VerifyArgs& a, int64_t b) {
  a.path[b] = 0;
  a.count[b] = 1;
  if (a.probs) a.probs[b] = 0.0f;
}
// The tokens of trees of one node.
template <Elt E, int PIECES> __global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
  const Layout l = layout(a);
  const int64_t b = blockIdx.x;
  const double factor = factor_of(a, b);
  const End e = root_end(a, b);
  if (e.node < 0) return;
  if (threadIdx.x == 0) one_node(a, b);
  const Rest* rests = l.rest + b * a.segments;
  pick<E, PIECES>(a, b, e, factor, nullptr, [&](int c) { return read_rest(rests + c); });
}
// ---- rows of bf16 through a table ------------------------------------------------------

// There are few bf16 numbers: the weights 2^(x c) of all of 2^-16 <= |x| < 2^7 are 5888
// doubles (46 KiB, in 55 of LDS: each sign begins a half), which a workgroup computes once, and a logit's is a read of LDS (five 32-bit
// instructions and an addition of 64 bits in the place of 17).  c <= 7, so that they stay
// within a double's range (and x c, up to 900, is off by 2^-44); segments with other numbers are
// summed as the other types' are.  131072 logits of 32 rows of 8 trees: 33 us without the
// table, 20 with it, which the reads of LDS and their conflicts bound (bytes: 11).
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
constexpr int kTableWaves = plan::kVerifyTableWaves, kTableThreads = 64 * kTableWaves;
constexpr uint32_t kTableLeast = (127 - 16) << 7, kTableSize = 23 << 7;  // first magnitude, number of them
constexpr uint32_t kNegative = 0x8000;  // bytes from a number's weight to its negative's
constexpr int kTableBytes = kNegative + kTableSize * 8;
static_assert(kTableSize * 8 <= kNegative, "a half for each sign");
constexpr double kTableSteepest = 7.0;  // c

// Where the magnitudes of two numbers lie in the table.
__device__ __forceinline__ u16x2 place_of(uint32_t w) {
  return __builtin_bit_cast(u16x2, w & 0x7fff7fffu) - (unsigned short)kTableLeast;
}

// The statistics of segment g, if the table has all of its numbers.
template <int PIECES>
__device__ __forceinline__ bool table_stat(const VerifyArgs& a, const Row<Elt::BF16>& r, int g,
                                           const Held<Elt::BF16, PIECES>& h, double factor, const char* table,
                                           Stat& st) {
  // (The first and the last segment may have a head or a tail.)
  if ((g == 0 && r.head > 0) || (g + 1) * PIECES * 64 > r.full ||
      (g == a.segments - 1 && r.head + r.full * Row<Elt::BF16>::N < r.n)) return false;
  // Magnitudes from the table's first on (smaller ones wrap round), and the largest number as an
  // integer: right if it is positive.
  u16x2 most = {0, 0};
  i16x2 top = {-32768, -32768};
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w = (uint32_t)h.w[i][k];
      most = __builtin_elementwise_max(most, place_of(w));
      top = __builtin_elementwise_max(top, __builtin_bit_cast(i16x2, w));
    }
  if (__builtin_amdgcn_ballot_w64(max(most[0], most[1]) >= kTableSize)) return false;
  uint32_t bits = (uint16_t)max(top[0], top[1]);
  if (bits & 0x8000) {  // the lane has negative numbers only: the smallest magnitude
    u16x2 least = {0xffff, 0xffff};
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, (uint32_t)h.w[i][k]));
    bits = min(least[0], least[1]);
  }
  const float m = wave_max(__builtin_bit_cast(float, bits << 16));
  double s[4] = {0.0, 0.0, 0.0, 0.0}, read[2][8];
#pragma unroll
  for (int i = 0; i <= PIECES; ++i) {
    // A piece's reads, then the additions of the one before.
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i == PIECES) continue;
      const uint32_t w = (uint32_t)h.w[i][k];
      const u16x2 at = place_of(w) << (unsigned short)3;
      const uint32_t both = (w & 0x80008000u) | __builtin_bit_cast(uint32_t, at);
      read[i & 1][2 * k] = *(const double*)(table + (both & 0xffff));
      read[i & 1][2 * k + 1] = *(const double*)(table + (both >> 16));
    }
    __builtin_amdgcn_sched_barrier(0);
    if (i == 0) continue;
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] += read[(i + 1) & 1][2 * k] + read[(i + 1) & 1][2 * k + 1];
    __builtin_amdgcn_sched_barrier(0);
  }
  // The sum relative to the maximum, as the other segments' are.
  const double sum = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
  st = Stat{sum * pow2_any(-(double)m * factor), m, INT32_MAX};
  return true;
}

__device__ __forceinline__ void fill_table(char* table, double factor, int threads) {
  for (uint32_t i = threadIdx.x; i < 2 * kTableSize; i += threads) {
    const uint32_t magnitude = kTableLeast + (i >> 1);
    const float x = bf16_bits_to_f32((uint16_t)((i & 1) << 15 | magnitude));
    *(double*)(table + (i & 1) * kNegative + (i >> 1) * 8) = pow2_any((double)x * factor);
  }
}

// As verify_rows_kernel for the rows of nodes that have children.
template <int PIECES>
__global__ __launch_bounds__(kTableThreads) void verify_table_kernel(VerifyArgs a, int groups) {
  __shared__ __attribute__((aligned(16))) char table[kTableBytes];
  const int tid = threadIdx.x, lane = tid & 63, step = groups * kTableWaves;
  uint32_t id = blockIdx.x;
  int g = __builtin_amdgcn_readfirstlane((int)(id % groups * kTableWaves + (tid >> 6)));
  id /= groups;
  const int t = id % a.tokens;
  const int64_t b = id / a.tokens;
  const int n = nodes_of(a, b);
  uint64_t child = 0;  // (every wave looks for itself: all of them find the same)
  for (int i0 = t + 1; i0 < n && !child; i0 += 64)
    child = __builtin_amdgcn_ballot_w64(i0 + lane < n && a.parents[b * a.tokens + min(i0 + lane, n - 1)] == t);
  if (!child) return;
  const double factor = factor_of(a, b);
  const Row<Elt::BF16> r = row_of<Elt::BF16>(a, b, t);
  Stat* stats = layout(a).stats + (b * a.tokens + t) * a.segments;
  Held<Elt::BF16, PIECES> now, next;
  if (g < a.segments) load_segment<Elt::BF16, PIECES>(a, r, g, now);
  const bool tabled = factor > 0.0 && factor <= kTableSteepest;
  if (tabled) {
    fill_table(table, factor, kTableThreads);
  }
  __syncthreads();
  for (; g < a.segments; g += step) {
    if (g + step < a.segments) load_segment<Elt::BF16, PIECES>(a, r, g + step, next);
    Stat st;
    if (!tabled || !table_stat<PIECES>(a, r, g, now, factor, table, st))
      st = segment_stat<Elt::BF16, PIECES>(a, r, g, now, factor, nullptr, 0);
    if (lane == 0) stats[g] = st;
    now = next;
  }
}

// Trees of one node in a launch, a workgroup a row: its latencies and, of long rows, one CU's 64-bit
// arithmetic bound it.  A row of 32000 bf16 9.4 us, of which 1 us less by the table.
template <Elt E, int PIECES> __global__ __launch_bounds__(kAlone) void verify_alone_kernel(VerifyArgs a) {
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const double factor = factor_of(a, b);
  const End e = root_end(a, b);
  if (e.node < 0) return;
  constexpr bool kTable = E == Elt::BF16 && PIECES == 4;
  __shared__ Rest rests[plan::kVerifyAlone];
  __shared__ __attribute__((aligned(16))) char table[kTable ? kTableBytes : 16];
  const Row<E> r = row_of<E>(a, b, 0);
  int g = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  Held<E, PIECES> now;
  if (g < a.segments) load_segment<E, PIECES>(a, r, g, now);
  if (threadIdx.x == 0) one_node(a, b);
  // (A table costs a lane 6 weights: for two waves a SIMD it took 0.5 us longer.)
  const bool tabled = kTable && a.segments > 8 && factor > 0.0 && factor <= kTableSteepest;
  if constexpr (kTable) {
    if (tabled) fill_table(table, factor, kAlone);
    __syncthreads();
  }
  for (; g < a.segments; g += kAlone / 64) {
    Stat st;
    bool found = false;
    if constexpr (kTable) found = tabled && table_stat<PIECES>(a, r, g, now, factor, table, st);
    if (!found) st = segment_stat<E, PIECES>(a, r, g, now, factor, nullptr, 0);
    if (lane == 0) rests[g] = Rest{st.s, st.s, st.m, st.at};
    if (g + kAlone / 64 < a.segments) load_segment<E, PIECES>(a, r, g + kAlone / 64, now);
  }
  __syncthreads();
  pick<E, PIECES>(a, b, e, factor, nullptr, [&](int c) { return rests[c]; });
}

// ---- the walk ----------------------------------------------------------------------

template <Elt E> __device__ __forceinline__ float logit(const VerifyArgs& a, int64_t b, int64_t t, int v) {
  return load_as_f32<E>(a.logits, b * a.sb + t * a.st + v);
}

// LAST: what is left of the last row, and the token, as well.
template <Elt E, int PIECES, bool LAST>
__global__ __launch_bounds__(kWalkers) void verify_walk_kernel(VerifyArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  double* mass = (double*)smem;            // [tokens] sum of a node's row, NaN if it has none
  double* chance = mass + a.tokens;        // [tokens] weight of a node's token in its parent's row
  double* list = chance + a.tokens;        // [tokens]
  float* tops = (float*)(list + a.tokens);  // [tokens]
  int* firsts = (int*)(tops + a.tokens);   // [tokens]
  int* up = firsts + a.tokens;             // [tokens] parent, -1: none that is reached
  float* qs = (float*)(up + a.tokens);     // [tokens]
  int* order = (int*)(qs + a.tokens);      // [tokens] the nodes that have children
  int* tokens = order + a.tokens;          // [tokens] their drafts
  float* us = (float*)(tokens + a.tokens);  // [tokens]
  __shared__ int todo, at_node, at_rounds, inner;
  __shared__ double sums[(kWalkers / 64)];
  const Layout l = layout(a);
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = nodes_of(a, b);
  if (n < 1) {
    if (tid == 0) l.end[b].node = -1;
    return;
  }
  const double factor = factor_of(a, b);
  const bool dense = a.draft_probs != nullptr;
  // A thread has a node; what it loads is under way while the rows are combined.
  static_assert(plan::kVerifyNodes <= kWalkers, "a thread for each node");
  int parent = -1, token = -1;
  float x = 0.0f, q = 1.0f;
  if (tid < a.tokens) {
    if (tid > 0 && tid < n) parent = a.parents[b * a.tokens + tid], token = a.drafts[b * a.tokens + tid];
    if (parent >= tid) parent = -1;
    up[tid] = parent;
    us[tid] = tid < n ? a.uniform[b * a.tokens + tid] : 0.0f;
    tokens[tid] = token;
    if (tid > 0) a.path[b * a.tokens + tid] = -1;
    mass[tid] = __builtin_nan("");
    firsts[tid] = 0;  // (whether the node has a child, for now)
  }
  if (tid == 0) inner = 0;
  const bool known = parent >= 0 && token >= 0 && token < a.vocab;
  if (known) {
    x = logit<E>(a, b, parent, token);
    if (dense) q = a.draft_probs[b * a.qb + parent * a.qt + token];
  }
  __syncthreads();
  if (parent >= 0) firsts[parent] = 1;
  __syncthreads();
  if (tid < n && firsts[tid]) order[atomicAdd(&inner, 1)] = tid;
  __syncthreads();
  // A wave combines the segments of a row.
  for (int i = wave; i < inner; i += kWalkers / 64) {
    const int t = order[i];
    const Stat* st = l.stats + (b * a.tokens + t) * a.segments;
    const Stat none = {0.0, -__builtin_inff(), INT32_MAX}, mine = lane < a.segments ? st[lane] : none;
    float m = mine.m;
    for (int c = lane + 64; c < a.segments; c += 64) m = __builtin_elementwise_maximum(m, st[c].m);
    m = wave_max(m);
    auto scaled = [&](const Stat& x) {
      return x.s == 0.0 ? 0.0 : factor == 0.0 ? x.s : x.s * pow2(((double)x.m - (double)m) * factor);
    };
    double s = scaled(mine);
    int at = mine.m == m ? mine.at : INT32_MAX;
    for (int c = lane + 64; c < a.segments; c += 64) {
      const Stat x = st[c];
      s += scaled(x);
      if (x.m == m) at = min(at, x.at);
    }
    s = wave_sum(s);
    at = wave_min(at);
    if (lane == 0) mass[t] = s > 0.0 && s < __builtin_inf() ? s : __builtin_nan(""), tops[t] = m, firsts[t] = at;
  }
  __syncthreads();
  if (tid < a.tokens) {
    // (A row without probabilities has none for its tokens either.)
    double w = 0.0;
    if (known) w = factor == 0.0 ? token == firsts[parent] ? mass[parent] : 0.0
                                 : pow2(((double)x - (double)tops[parent]) * factor);
    chance[tid] = w;
    qs[tid] = q;
    if (a.probs) a.probs[b * a.tokens + tid] = parent >= 0 ? (float)(w / mass[parent]) : 0.0f;
  }
  __syncthreads();

  // The walk, by the first wave, 64 nodes at a time: children of the current node
  // have higher numbers, and so have those of a child that is taken.  Where
  // another child follows one that was rejected in favour of a dense rest, all
  // waves sum that rest first.
  int cur = 0, count = 1, rounds = 0, base = 1, start = 1;
  bool none = false;
  double left = mass[0];  // of one-hot drafts: the row's sum without the rejected tokens
  if (tid == 0) a.path[b * a.tokens] = 0;
  for (;;) {
    if (wave == 0) {
      bool sum = false;
      for (; base < n && !sum; base += sum ? 0 : 64) {
        const int t = base + lane;
        const bool live = t < n;
        const int parent = live ? up[t] : -1, token = live ? tokens[t] : -1;
        const float u = live ? us[t] : 0.0f;
        double w = live ? chance[t] : 0.0;
        const float q = live ? qs[t] : 0.0f;
        if (!dense)
          for (int i = 0; i < rounds; ++i)
            if (parent == cur && (double)token == list[i]) w = 0.0;
        for (;;) {
          const uint64_t kids = __builtin_amdgcn_ballot_w64(parent == cur && t >= start);
          if (!kids) break;
          const int k = __builtin_ctzll(kids);
          const double whole = mass[cur];
          if (whole != whole) {  // no probabilities: the walk ends here
            none = true;
            base = n;
            break;
          }
          const double wk = lane_d(w, k);
          const float uk = lane_f(u, k), qk = lane_f(q, k);
          const int token_k = __builtin_amdgcn_readlane(token, k);
          bool taken;
          if (dense && factor != 0.0) {
            if (rounds > 0 && list[rounds - 1] < 0.0) {
              sum = true;
              break;
            }
            taken = (double)uk * (double)qk < left_of(wk / whole, (double)qk, list, rounds);
          } else if (factor == 0.0) {
            taken = wk > 0.0;
          } else {
            taken = (double)uk * left < wk;
          }
          start = base + k + 1;
          if (taken) {
            cur = base + k;
            if (lane == 0) a.path[b * a.tokens + count] = cur;
            ++count;
            rounds = 0;
            left = mass[cur];
          } else {
            // One-hot drafts: the token; dense ones: a rest that has no sum yet.
            list[rounds] = dense ? -1.0 : (double)token_k;
            ++rounds;
            if (!dense) {
              left -= wk;
              if (parent == cur && token == token_k) w = 0.0;
            }
          }
          __builtin_amdgcn_wave_barrier();
        }
        if (sum) break;
      }
      if (lane == 0) todo = sum, at_node = cur, at_rounds = rounds;
    }
    __syncthreads();
    if (!todo) break;
    // The sum of what `at_rounds` rejected children left of node at_node's row.
    const int node = at_node, done = at_rounds - 1;
    const double top = (double)tops[node], inverse = 1.0 / mass[node];
    const float* q = a.draft_probs + b * a.qb + node * a.qt;
    double s = 0.0;
    for (int v = tid; v < a.vocab; v += kWalkers) {
      const double p = pow2(((double)logit<E>(a, b, node, v) - top) * factor) * inverse;
      s += __builtin_fmax(left_of(p, (double)q[v], list, done) - (double)q[v], 0.0);
    }
    s = wave_sum(s);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    if (tid == 0) {
      double all = 0.0;
      for (int w = 0; w < (kWalkers / 64); ++w) all += sums[w];
      list[done] = all > 0x1p-1000 ? 1.0 / all : 0.0;
    }
    __syncthreads();
  }
  // (Of the first wave.  A node at which no child was rejected has no `firsts`.)
  End e = {1.0 / mass[cur], tops[cur], none ? -2 : cur, rounds, factor != 0.0 ? -1 : rounds > 0 ? firsts[cur] : -2, 0};
  if constexpr (LAST) {
    __shared__ End end;
    __shared__ Rest rests[plan::kVerifyShort];
    if (tid == 0) end = e, a.count[b] = count;
    __syncthreads();
    e = end;
    if (e.node < 0 || e.greedy >= 0) {
      if (tid == 0) a.token[b] = e.node < 0 ? -1 : e.greedy;
      return;
    }
    const Row<E> r = row_of<E>(a, b, e.node);
    const Stat* stats = l.stats + (b * a.tokens + e.node) * a.segments;
    for (int g = __builtin_amdgcn_readfirstlane(wave); g < a.segments; g += kWalkers / 64) {
      Rest rest;
      if (dense && e.rounds > 0) {
        rest = segment_rest<E, PIECES>(a, r, b, g, e, list, factor);
      } else {
        Held<E, PIECES> held;
        load_segment<E, PIECES>(a, r, g, held);
        rest = last_segment<E, PIECES>(a, r, b, g, e, list, factor, stats, held);
      }
      if (lane == 0) rests[g] = rest;
    }
    __syncthreads();
    pick<E, PIECES>(a, b, e, factor, list, [&](int c) { return rests[c]; });
  } else {
    for (int i = tid; i < at_rounds; i += kWalkers) l.list[b * a.tokens + i] = list[i];
    if (tid == 0) l.end[b] = e, a.count[b] = count;
  }
}

template <Elt E, int PIECES> hipError_t launch_pieces(const VerifyArgs& a, hipStream_t s) {
  const int64_t groups = (a.segments + kWaves - 1) / kWaves;  // a segment a wave
  if (plan::verify_alone(a.batch, a.tokens, a.segments, device_cus())) {
    hipLaunchKernelGGL((verify_alone_kernel<E, PIECES>), dim3((unsigned)a.batch), dim3(kAlone), 0, s, a);
    return hipGetLastError();
  }
  auto rows = verify_rows_kernel<E, PIECES>;
  bool last = true;  // the last rows are still to do
  if (a.tokens > 1) {
    // As many segments a wave as leave 32 waves for a CU.
    const int64_t per = a.batch * a.tokens * groups / (8 * (int64_t)device_cus());
    const int64_t some = (groups + std::max<int64_t>(per, 1) - 1) / std::max<int64_t>(per, 1);
    auto walk = verify_walk_kernel<E, PIECES, false>;
    int64_t tables = 0;
    if constexpr (E == Elt::BF16 && PIECES == 4) {
      tables = plan::verify_tables(a.batch, a.tokens, a.segments, device_cus());
      if (tables)
        hipLaunchKernelGGL(verify_table_kernel<PIECES>, dim3((unsigned)(a.batch * a.tokens * tables)),
                           dim3(kTableThreads), 0, s, a, (int)tables);
    }
    if (!tables)
      hipLaunchKernelGGL(rows, dim3((unsigned)(a.batch * a.tokens * some)), dim3(kThreads), 0, s, a, (int)some, 0);
    if constexpr (PIECES == 1)
      if (a.segments <= plan::kVerifyShort) walk = verify_walk_kernel<E, PIECES, true>, last = false;
    hipLaunchKernelGGL(walk, dim3((unsigned)a.batch), dim3(kWalkers), (unsigned)(a.tokens * 52), s, a);
  }
  if (last)
    hipLaunchKernelGGL(rows, dim3((unsigned)(a.batch * groups)), dim3(kThreads), 0, s, a, (int)groups, 1);
  if (a.tokens == 1) hipLaunchKernelGGL((verify_pick_kernel<E, PIECES>), dim3((unsigned)a.batch), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

template <Elt E> hipError_t launch_type(const VerifyArgs& a, hipStream_t s) {
  switch (a.pieces) {
    case 1: return launch_pieces<E, 1>(a, s);
    case 4: return launch_pieces<E, 4>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

int64_t verify_workspace(int64_t batch, int64_t tokens, int64_t segments) {
  if (plan::verify_alone(batch, tokens, segments, device_cus())) return 0;
  return up16(batch * tokens * segments * (int64_t)sizeof(Stat)) + up16(batch * segments * (int64_t)sizeof(Rest)) +
         up16(batch * (int64_t)sizeof(End)) + batch * tokens * 8;
}

hipError_t tree_verify(const VerifyArgs& a, hipStream_t s) {
  switch (a.dtype) {
    case Elt::F32: return launch_type<Elt::F32>(a, s);
    case Elt::F16: return launch_type<Elt::F16>(a, s);
    default: return launch_type<Elt::BF16>(a, s);
  }
}

}  // namespace frisk
