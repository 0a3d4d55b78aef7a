// Verification of drafted tokens: which branch of a tree the target's
// probabilities accept under given random numbers, and the token after it.
//
// Probabilities are compared with random numbers, so they are computed in 64
// bits: a weight is 2^t, t = (x - max) log2(e) / T, from a polynomial of degree 11
// on the fraction of t, off by 2^-47 of it, and sums are of doubles.  The vector
// unit does as many 64-bit as 32-bit multiply-adds, so a weight costs about 20
// instructions and reading the logits once bounds the work.
//
// Four launches.  (1) The rows of nodes that have children, in chunks: each one's
// maximum and sum.  (2) A workgroup per tree combines them, takes every node's
// probability given its parent, and walks from the root.  (3) What is left of the
// probabilities at the last node, in chunks; chunks that no rejected token lies in
// have their sums from (1).  (4) The chunk, then the element, in which the sum
// passes the last random number.

#include "common.h"
#include "kernels.h"

namespace frisk {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// A chunk's or a row's largest logit, its first place, and the sum of weights
// 2^((x - m) c): NaN if the row gives no probabilities (it holds a NaN or +infinity).
struct Stat {
  double s;
  float m;
  int at;
};
// A chunk of the last node's row: sums of what is left there, and of what was left
// before the last rejection; both relative to m.
struct Rest {
  double s, whole;
  float m;
  int at;
};
// Where a walk ended.
struct End {
  double scale;  // sum of the row's weights
  float m;       // its maximum
  int node;      // -1: the tree takes no part, -2: no token
  int rounds;    // children rejected there
  int greedy;    // the token, if the temperature is 0 and it is known; -1: sample, -2: largest
};

struct Layout {
  Stat* stats;  // [batch][tokens][chunks]
  Rest* rest;   // [batch][chunks]
  End* end;     // [batch]
  double* list;  // [batch][tokens] rejected tokens or, of dense drafts, what their rest summed to
};
__host__ __device__ inline int64_t up16(int64_t n) { return (n + 15) & ~15ll; }
__device__ __forceinline__ Layout layout(const VerifyArgs& a) {
  char* p = (char*)a.workspace;
  Layout l;
  l.stats = (Stat*)p;
  p += up16((int64_t)a.batch * a.tokens * a.chunks * sizeof(Stat));
  l.rest = (Rest*)p;
  p += up16((int64_t)a.batch * a.chunks * sizeof(Rest));
  l.end = (End*)p;
  p += up16((int64_t)a.batch * sizeof(End));
  l.list = (double*)p;
  return l;
}

// 2^t for t <= 0 (0 below -1100).
__device__ __forceinline__ double pow2(double t) {
  t = __builtin_fmax(t, -1100.0);
  const double k = __builtin_rint(t), f = t - k;
  // ln(2)^n / n!: the first term left out is 2^-47 of the result at f = 1/2.
  double p = 4.44553827187081e-10;
  p = __builtin_fma(p, f, 7.054911620801121e-09);
  p = __builtin_fma(p, f, 1.0178086009239696e-07);
  p = __builtin_fma(p, f, 1.3215486790144305e-06);
  p = __builtin_fma(p, f, 1.5252733804059838e-05);
  p = __builtin_fma(p, f, 1.5403530393381606e-04);
  p = __builtin_fma(p, f, 1.3333558146428441e-03);
  p = __builtin_fma(p, f, 9.618129107628477e-03);
  p = __builtin_fma(p, f, 5.5504108664821577e-02);
  p = __builtin_fma(p, f, 2.402265069591007e-01);
  p = __builtin_fma(p, f, 6.931471805599453e-01);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)k);
}

// log2(e) / T of a tree; 0: its temperature is 0, the largest logit wins.
__device__ __forceinline__ double factor_of(const VerifyArgs& a, int64_t b) {
  if (!a.temperature) return 1.4426950408889634;
  const float t = a.temperature[b];
  return t > 0.0f ? 1.4426950408889634 / (double)t : 0.0;
}
__device__ __forceinline__ int nodes_of(const VerifyArgs& a, int64_t b) {
  return a.new_len ? min(max(a.new_len[b], 0), a.tokens) : a.tokens;
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

// A chunk's elements are PIECES whole pieces a thread, in the order (piece, thread,
// element); the first chunk's start with the row's head, the last one's end with
// its tail, one element a thread.
template <Elt E> __device__ __forceinline__ void load_piece(const Row<E>& r, int piece, float (&x)[Row<E>::N]) {
  const i32x4 w = *(const i32x4*)(r.p + r.head + (int64_t)piece * Row<E>::N);
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
// The loose element of a thread in chunk c, or -1: the head's in the first chunk
// (threads 0 ..), the tail's in the last (threads 128 ..).
template <Elt E> __device__ __forceinline__ int loose_of(const VerifyArgs& a, const Row<E>& r, int c) {
  const int tid = threadIdx.x;
  if (c == 0 && tid < r.head) return tid;
  const int tail = r.head + r.full * Row<E>::N;
  if (c == a.chunks - 1 && tid >= 128 && tail + tid - 128 < r.n) return tail + tid - 128;
  return -1;
}

__device__ __forceinline__ double shfl_d(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)u, lane), hi = (uint32_t)__shfl((int)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x += shfl_d(x, lane ^ m);
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x = fmaxf(x, __shfl_xor(x, m));
  return x;
}
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x = min(x, __shfl_xor(x, m));
  return x;
}

// The statistics of chunk c of a row, known to all threads afterwards.  skip(index):
// the element has no weight.
template <Elt E, int PIECES, typename Skip>
__device__ __forceinline__ Stat chunk_stat(const VerifyArgs& a, const Row<E>& r, int c, double factor, Skip skip) {
  constexpr int N = Row<E>::N;
  __shared__ float ms[kWaves];
  __shared__ double ss[kWaves];
  __shared__ int as[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int base = c * PIECES * kThreads + tid;
  float x[PIECES][N];
  float m = -__builtin_inff();
  bool bad = false;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int piece = base + i * kThreads;
    if (piece < r.full) {
      load_piece<E>(r, piece, x[i]);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        bad |= x[i][e] != x[i][e];
        if (skip(r.head + piece * N + e)) x[i][e] = -__builtin_inff();
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[i][e] = -__builtin_inff();
    }
  }
  const int loose = loose_of<E>(a, r, c);
  float extra = -__builtin_inff();
  if (loose >= 0) {
    extra = (float)r.p[loose];
    bad |= extra != extra;
    if (skip(loose)) extra = -__builtin_inff();
  }
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, x[i][e]);
  m = wave_max(fmaxf(m, extra));
  __syncthreads();
  if (lane == 0) ms[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, ms[w]);
  double s = 0.0;
  int at = INT32_MAX;
  if (m > -__builtin_inff()) {
    if (factor == 0.0) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (x[i][e] == m) at = min(at, r.head + (base + i * kThreads) * N + e);
      if (extra == m) at = min(at, loose);
      s = tid == 0 ? 1.0 : 0.0;
    } else {
      const double top = (double)m;
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (base + i * kThreads < r.full)
#pragma unroll
          for (int e = 0; e < N; ++e) s += pow2(((double)x[i][e] - top) * factor);
      if (loose >= 0) s += pow2(((double)extra - top) * factor);
    }
  }
  if (bad || m == __builtin_inff()) s = __builtin_nan("");
  s = wave_sum(s);
  at = wave_min(at);
  if (lane == 0) ss[wave] = s, as[wave] = at;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += ss[w], at = min(at, as[w]);
  return Stat{s, m, at};
}

template <Elt E, int PIECES> __global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
  uint32_t id = blockIdx.x;
  const int c = id % a.chunks;
  id /= a.chunks;
  const int t = id % a.tokens;
  const int64_t b = id / a.tokens;
  const int n = nodes_of(a, b);
  if (t >= n) return;
  // A row is needed if its node has a child.
  bool child = false;
  for (int i = t + 1 + threadIdx.x; i < n; i += kThreads) child |= a.parents[b * a.tokens + i] == t;
  if (!__syncthreads_or(child)) return;
  const Row<E> r = row_of<E>(a, b, t);
  const Stat st = chunk_stat<E, PIECES>(a, r, c, factor_of(a, b), [](int) { return false; });
  if (threadIdx.x == 0) layout(a).stats[(b * a.tokens + t) * a.chunks + c] = st;
}

// What is left of a probability p after `rounds` children drawn from q were
// rejected, whose rests summed to z[0 ..]; a rest without mass leaves it as it was.
__device__ __forceinline__ double left_of(double p, double q, const double* z, int rounds) {
  for (int i = 0; i < rounds; ++i) {
    const double rest = __builtin_fmax(p - q, 0.0), mass = z[i];
    if (mass > 0.0) p = rest / mass;
  }
  return p;
}

template <Elt E> __device__ __forceinline__ float logit(const VerifyArgs& a, int64_t b, int64_t t, int v) {
  return load_as_f32<E>(a.logits, b * a.sb + t * a.st + v);
}

template <Elt E> __global__ __launch_bounds__(kThreads) void verify_walk_kernel(VerifyArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  double* mass = (double*)smem;            // [tokens] sum of a node's row, NaN if it has none
  double* chance = mass + a.tokens;        // [tokens] weight of a node's token in its parent's row
  double* list = chance + a.tokens;        // [tokens]
  float* tops = (float*)(list + a.tokens);  // [tokens]
  int* firsts = (int*)(tops + a.tokens);   // [tokens]
  int* up = firsts + a.tokens;             // [tokens] parent, -1: none that is reached
  float* qs = (float*)(up + a.tokens);     // [tokens]
  __shared__ int todo, at_node, at_rounds;
  __shared__ double sums[kWaves];
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
  for (int t = tid; t < a.tokens; t += kThreads) {
    const int p = t < n ? a.parents[b * a.tokens + t] : -1;
    up[t] = p >= 0 && p < t ? p : -1;
    mass[t] = __builtin_nan("");
    chance[t] = 0.0;
    if (t > 0) a.path[b * a.tokens + t] = -1;
    firsts[t] = 0;  // (whether the node has a child, for now)
  }
  __syncthreads();
  for (int t = tid; t < n; t += kThreads)
    if (up[t] >= 0) firsts[up[t]] = 1;
  __syncthreads();
  for (int t = wave; t < n; t += kWaves) {
    if (!firsts[t]) continue;
    const Stat* st = l.stats + (b * a.tokens + t) * a.chunks;
    float m = -__builtin_inff();
    for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, st[c].m);
    m = wave_max(m);
    double s = 0.0;
    int at = INT32_MAX;
    for (int c = lane; c < a.chunks; c += 64) {
      const Stat x = st[c];
      if (x.m > -__builtin_inff() || x.s != x.s) s += x.s * (factor == 0.0 ? 1.0 : pow2(((double)x.m - (double)m) * factor));
      if (factor == 0.0 && x.m == m) at = min(at, x.at);
    }
    s = wave_sum(s);
    at = wave_min(at);
    if (lane == 0) mass[t] = s > 0.0 && s < __builtin_inf() ? s : __builtin_nan(""), tops[t] = m, firsts[t] = at;
  }
  __syncthreads();
  for (int t = tid; t < a.tokens; t += kThreads) {
    const int p = t < n ? up[t] : -1, v = p >= 0 ? a.drafts[b * a.tokens + t] : -1;
    double w = 0.0;
    float q = 1.0f;
    if (p >= 0 && v >= 0 && v < a.vocab) {
      if (factor == 0.0) w = v == firsts[p] ? mass[p] : 0.0;
      else w = pow2(((double)logit<E>(a, b, p, v) - (double)tops[p]) * factor);
      if (dense) q = a.draft_probs[b * a.qb + p * a.qt + v];
    }
    // (A row without probabilities has none for its tokens either.)
    chance[t] = w;
    qs[t] = q;
    if (a.probs) a.probs[b * a.tokens + t] = p >= 0 ? (float)(w / mass[p]) : 0.0f;
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
        const int parent = live ? up[t] : -1, token = live ? a.drafts[b * a.tokens + t] : -1;
        const float u = live ? a.uniform[b * a.tokens + t] : 0.0f;
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
          const double wk = shfl_d(w, k);
          const float uk = __shfl(u, k), qk = __shfl(q, k);
          const int token_k = __shfl(token, k);
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
    const double top = (double)tops[node], scale = mass[node];
    const float* q = a.draft_probs + b * a.qb + node * a.qt;
    double s = 0.0;
    for (int v = tid; v < a.vocab; v += kThreads) {
      const double p = pow2(((double)logit<E>(a, b, node, v) - top) * factor) / scale;
      s += __builtin_fmax(left_of(p, (double)q[v], list, done) - (double)q[v], 0.0);
    }
    s = wave_sum(s);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    if (tid == 0) {
      double all = 0.0;
      for (int w = 0; w < kWaves; ++w) all += sums[w];
      list[done] = all;
    }
    __syncthreads();
  }
  for (int i = tid; i < at_rounds; i += kThreads) l.list[b * a.tokens + i] = list[i];
  if (tid == 0) {
    End e;
    e.scale = mass[cur];
    e.m = tops[cur];
    e.node = cur;
    e.rounds = rounds;
    e.greedy = -1;
    if (none) e.node = -2;
    // (A node at which no child was rejected has none.)
    if (factor == 0.0) e.greedy = rounds > 0 ? firsts[cur] : -2;
    l.end[b] = e;
    a.count[b] = count;
  }
}

// Weight of what is left of an element, and before the last rejection, for dense
// drafts.
struct Left {
  double now, was;
};
__device__ __forceinline__ Left dense_left(double p, float q, const double* z, int rounds) {
  const double was = left_of(p, (double)q, z, rounds - 1);
  return {__builtin_fmax(was - (double)q, 0.0), was};
}

template <Elt E, int PIECES> __global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs a) {
  constexpr int N = Row<E>::N;
  const Layout l = layout(a);
  const int c = blockIdx.x % a.chunks;
  const int64_t b = blockIdx.x / a.chunks;
  const End e = l.end[b];
  if (e.node < 0 || e.greedy >= 0) return;
  const double factor = factor_of(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Rest* out = l.rest + b * a.chunks + c;
  const Row<E> r = row_of<E>(a, b, e.node);
  const double* list = l.list + b * a.tokens;
  if (e.rounds > 0 && a.draft_probs) {
    __shared__ double ss[kWaves], ws[kWaves];
    const float* q = a.draft_probs + b * a.qb + e.node * a.qt;
    const double top = (double)e.m;
    double s = 0.0, whole = 0.0;
    auto add = [&](float x, int v) {
      const Left w = dense_left(pow2(((double)x - top) * factor) / e.scale, q[v], list, e.rounds);
      s += w.now;
      whole += w.was;
    };
#pragma unroll 1
    for (int i = 0; i < PIECES; ++i) {
      const int piece = (c * PIECES + i) * kThreads + tid;
      if (piece >= r.full) break;
      float x[N];
      load_piece<E>(r, piece, x);
#pragma unroll
      for (int k = 0; k < N; ++k) add(x[k], r.head + piece * N + k);
    }
    const int loose = loose_of<E>(a, r, c);
    if (loose >= 0) add((float)r.p[loose], loose);
    s = wave_sum(s);
    whole = wave_sum(whole);
    if (lane == 0) ss[wave] = s, ws[wave] = whole;
    __syncthreads();
    if (tid == 0) {
      Rest o = {0.0, 0.0, 0.0f, 0};
      for (int w = 0; w < kWaves; ++w) o.s += ss[w], o.whole += ws[w];
      *out = o;
    }
    return;
  }
  // One-hot drafts: without the rejected tokens.
  const int lo = c * PIECES * kThreads * N + (c ? r.head : 0);
  const int hi = c == a.chunks - 1 ? r.n : min(r.head + (c + 1) * PIECES * kThreads * N, r.n);
  __shared__ uint32_t gone[PIECES * kThreads * N / 32 + 1];
  bool any = false;
  if (e.rounds > 0) {
    for (int i = tid; i < PIECES * kThreads * N / 32 + 1; i += kThreads) gone[i] = 0;
    __syncthreads();
    for (int i = tid; i < e.rounds; i += kThreads) {
      const int v = (int)list[i];
      if (v >= lo && v < hi) atomicOr(&gone[(v - lo) >> 5], 1u << ((v - lo) & 31)), any = true;
    }
    any = __syncthreads_or(any);
    if (!any) {
      const Stat st = l.stats[(b * a.tokens + e.node) * a.chunks + c];
      if (tid == 0) *out = Rest{st.s, st.s, st.m, st.at};
      return;
    }
  }
  const Stat st = chunk_stat<E, PIECES>(a, r, c, factor, [&](int v) {
    return any && (gone[(v - lo) >> 5] >> ((v - lo) & 31)) & 1u;
  });
  if (tid == 0) *out = Rest{st.s, st.s, st.m, st.at};
}

template <Elt E, int PIECES> __global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
  constexpr int N = Row<E>::N;
  const Layout l = layout(a);
  const int64_t b = blockIdx.x;
  const End e = l.end[b];
  if (e.node == -1) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const double factor = factor_of(a, b);
  if (e.node < 0 || e.greedy >= 0) {
    if (tid == 0) a.token[b] = e.node < 0 ? -1 : e.greedy;
    return;
  }
  const Rest* rest = l.rest + b * a.chunks;
  const double* list = l.list + b * a.tokens;
  const bool dense = e.rounds > 0 && a.draft_probs;
  __shared__ int chosen, found, use_whole, token_at, last_at[kWaves];
  __shared__ double before, goal, sums[kWaves];
  __shared__ float top_at;
  if (wave == 0) {
    float m = -__builtin_inff();
    for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, rest[c].m);
    m = wave_max(m);
    auto scaled = [&](double s, float mc) {
      return s == 0.0 ? 0.0 : dense ? s : s * pow2(((double)mc - (double)m) * factor);
    };
    if (factor == 0.0) {
      int at = INT32_MAX;
      bool bad = false;
      for (int c = lane; c < a.chunks; c += 64) {
        if (rest[c].m == m) at = min(at, rest[c].at);
        bad |= rest[c].s != rest[c].s;
      }
      at = wave_min(at);
      bad = __builtin_amdgcn_ballot_w64(bad) != 0;
      if (lane == 0) a.token[b] = bad || at == INT32_MAX ? -1 : at, chosen = -1;
    } else {
      double s = 0.0, w = 0.0;
      for (int c = lane; c < a.chunks; c += 64) s += scaled(rest[c].s, rest[c].m), w += scaled(rest[c].whole, rest[c].m);
      s = wave_sum(s);
      w = wave_sum(w);
      const bool whole = dense && !(s > 0.0);
      const double all = whole ? w : s, want = (double)a.final_uniform[b] * all;
      if (!(all > 0.0) || all == __builtin_inf()) {
        // Nothing is left of one-hot drafts: the last one had it all.  Else the
        // row gives no probabilities.
        if (lane == 0) a.token[b] = all == 0.0 && e.rounds > 0 && !dense ? (int)list[e.rounds - 1] : -1, chosen = -1;
      } else {
        // The first chunk whose end passes `want`; the last one with any mass, if rounding
        // leaves none.
        double base = 0.0, at_base = 0.0, last_base = 0.0;
        int at = -1, last = -1;
        for (int c0 = 0; c0 < a.chunks && at < 0; c0 += 64) {
          const int c = c0 + lane;
          const double mine = c < a.chunks ? scaled(whole ? rest[c].whole : rest[c].s, rest[c].m) : 0.0;
          double sum = mine;
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) {
            const double y = shfl_d(sum, max(lane - d, 0));
            if (lane >= d) sum += y;
          }
          const uint64_t some = __builtin_amdgcn_ballot_w64(mine > 0.0);
          const uint64_t past = __builtin_amdgcn_ballot_w64(mine > 0.0 && base + sum > want);
          if (past) {
            const int k = __builtin_ctzll(past);
            at = c0 + k;
            at_base = base + shfl_d(sum, k) - shfl_d(mine, k);
          } else if (some) {
            const int k = 63 - __builtin_clzll(some);
            last = c0 + k;
            last_base = base + shfl_d(sum, k) - shfl_d(mine, k);
          }
          base += shfl_d(sum, 63);
        }
        if (lane == 0) {
          chosen = at >= 0 ? at : last;
          before = at >= 0 ? at_base : last_base;
          goal = want;
          use_whole = whole;
          top_at = m;
        }
      }
    }
  }
  if (tid == 0) found = INT32_MAX, token_at = -1;
  __syncthreads();
  const int c = chosen;
  if (c < 0) return;
  // The chunk's elements in order: the head, the pieces, the tail.
  const Row<E> r = row_of<E>(a, b, e.node);
  const float* q = dense ? a.draft_probs + b * a.qb + e.node * a.qt : nullptr;
  const double top = (double)(dense ? e.m : top_at), want = goal;
  const bool whole = use_whole;
  auto weight = [&](float x, int v) {
    const double p = pow2(((double)x - top) * factor);
    if (dense) {
      const Left w = dense_left(p / e.scale, q[v], list, e.rounds);
      return whole ? w.was : w.now;
    }
    for (int i = 0; i < e.rounds; ++i)
      if (v == (int)list[i]) return 0.0;
    return p;
  };
  double base = before;
  int last = -1;
  // Step 0: the head, an element a thread; then the pieces; then the tail.
  const int tail = r.head + r.full * N;
  for (int step = 0; step < PIECES + 2; ++step) {
    double w[N], mine = 0.0;
    int first = 0, n = 0;
    if (step == 0 || step == PIECES + 1) {
      first = (step ? tail : 0) + tid;
      n = (step ? c == a.chunks - 1 && first < r.n : c == 0 && tid < r.head) ? 1 : 0;
      if (n) mine = w[0] = weight((float)r.p[first], first);
    } else {
      const int piece = (c * PIECES + step - 1) * kThreads + tid;
      if (piece < r.full) {
        n = N;
        first = r.head + piece * N;
        float x[N];
        load_piece<E>(r, piece, x);
#pragma unroll
        for (int k = 0; k < N; ++k) w[k] = weight(x[k], first + k), mine += w[k];
      }
    }
    double sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double y = shfl_d(sum, max(lane - d, 0));
      if (lane >= d) sum += y;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    double at = base + sum - mine, all = base;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      if (k < wave) at += sums[k];
      all += sums[k];
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < n && w[k] > 0.0) {
        last = first + k;
        at += w[k];
        if (at > want) {
          atomicMin(&found, first + k);
          break;
        }
      }
    base = all;
    __syncthreads();
    if (found != INT32_MAX) break;
  }
  if (found == INT32_MAX) {  // rounding: the last element with a weight
    for (int m = 1; m < 64; m <<= 1) last = max(last, __shfl_xor(last, m));
    if (lane == 0) last_at[wave] = last;
    __syncthreads();
    last = max(max(last_at[0], last_at[1]), max(last_at[2], last_at[3]));
  }
  if (tid == 0) a.token[b] = found != INT32_MAX ? found : last;
}

template <Elt E, int PIECES> hipError_t launch_pieces(const VerifyArgs& a, hipStream_t s) {
  const int64_t rows = a.batch * a.tokens * a.chunks, ends = a.batch * a.chunks;
  if (rows > UINT32_MAX / kThreads) return hipErrorInvalidConfiguration;
  if (a.tokens > 1)
    hipLaunchKernelGGL((verify_stats_kernel<E, PIECES>), dim3((unsigned)rows), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL((verify_walk_kernel<E>), dim3((unsigned)a.batch), dim3(kThreads),
                     (unsigned)(a.tokens * 40), s, a);
  hipLaunchKernelGGL((verify_rest_kernel<E, PIECES>), dim3((unsigned)ends), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL((verify_pick_kernel<E, PIECES>), dim3((unsigned)a.batch), dim3(kThreads), 0, s, a);
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

int64_t verify_workspace(int64_t batch, int64_t tokens, int64_t chunks) {
  return up16(batch * tokens * chunks * (int64_t)sizeof(Stat)) + up16(batch * chunks * (int64_t)sizeof(Rest)) +
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
