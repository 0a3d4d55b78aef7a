// Pages of a cache: the rows of accepted drafts moved behind their context, pages
// copied, and the tables of sequences that fork, end and grow.

#include "kvcache.h"

namespace frisk {

namespace {

using kv::Slot;

// One wave per sequence and head.  A lane has 16 B of each row of k or v (or a
// scale of each), so what it moves is its own: a move reads row path[i] >= i
// and writes row i, and the moves go up in i, kAhead loads before their stores;
// none of those rows has been written by an earlier move.
constexpr int kAhead = 8;
__global__ __launch_bounds__(64) void kv_compact_kernel(KvCompactArgs a) {
  const KvCache& c = a.cache;
  const int lane = threadIdx.x, h = blockIdx.x % c.kv_heads;
  const int64_t b = blockIdx.x / c.kv_heads;
  const int64_t ctx = a.ctx_len[b];
  const int n = min(a.count[b], a.tokens);
  if (ctx < 0) return;
  const int es = c.kind == Elt::E4M3 || c.kind == Elt::I8 ? 1 : 2;
  const int chunks = c.head_dim * es / 16, scales = es == 1 ? 1 : 0;
  // Items: the chunks of k, of v, then the scales of each (at most 64).
  const bool of_scale = lane >= 2 * chunks;
  const bool of_v = of_scale ? lane > 2 * chunks : lane >= chunks;
  const bool in = lane < 2 * (chunks + scales);
  char* base = of_scale ? (char*)((of_v ? c.v_scale : c.k_scale) + h * c.sch)
                        : (char*)(of_v ? c.v : c.k) + h * c.sh * es + (of_v ? lane - chunks : lane) * 16;
  __shared__ int64_t from[64], to[64], from_scale[64], to_scale[64];
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = i0 + lane, live = min(64, n - i0);
    const int64_t p = i < n ? a.path[b * a.path_stride + i] : i;
    // The path ends before an entry that is none.
    const uint64_t wrong = __builtin_amdgcn_ballot_w64(p < i);
    const int last = wrong ? min(live, (int)__builtin_ctzll(wrong)) : live;
    Slot src = {-1, -1}, dst = {-1, -1};
    if (i < n && p > i) src = kv::slot_of(c, b, ctx + p), dst = kv::slot_of(c, b, ctx + i);
    const bool moves = src.elem >= 0 && dst.elem >= 0;
    __syncthreads();
    from[lane] = moves ? src.elem * es : -1;
    to[lane] = dst.elem * es;
    from_scale[lane] = src.scale * 4;
    to_scale[lane] = dst.scale * 4;
    __syncthreads();
    for (int j0 = 0; j0 < last; j0 += kAhead) {
      i32x4 row[kAhead];
      int scale[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int k = j0 + j;
        if (k >= last || from[k] < 0 || !in) continue;
        if (of_scale) scale[j] = *(const int*)(base + from_scale[k]);
        else row[j] = *(const i32x4*)(base + from[k]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int k = j0 + j;
        if (k >= last || from[k] < 0 || !in) continue;
        if (of_scale) *(int*)(base + to_scale[k]) = scale[j];
        else *(i32x4*)(base + to[k]) = row[j];
      }
    }
    if (last < live) return;
  }
}

// A workgroup per pair of pages and head: 16 B of k and of v a thread at a time.
__global__ __launch_bounds__(256) void kv_copy_pages_kernel(KvCopyPagesArgs a) {
  const KvCache& c = a.cache;
  const int h = blockIdx.x % c.kv_heads;
  const int64_t pair = blockIdx.x / c.kv_heads;
  const int src = a.src[pair], dst = a.dst[pair];
  if (src < 0 || src >= c.pages || dst < 0 || dst >= c.pages || src == dst) return;
  int64_t rows = a.page_size;
  if (a.rows) rows = min(rows, (int64_t)max(a.rows[pair], 0));
  const int es = c.kind == Elt::E4M3 || c.kind == Elt::I8 ? 1 : 2;
  const int chunks = c.head_dim * es / 16;
  const int64_t items = rows * chunks;
  const bool whole = c.ss == c.head_dim;  // rows next to each other
  const char* k0 = (const char*)c.k + (src * c.sp + h * c.sh) * es;
  const char* v0 = (const char*)c.v + (src * c.sp + h * c.sh) * es;
  char* k1 = (char*)c.k + (dst * c.sp + h * c.sh) * es;
  char* v1 = (char*)c.v + (dst * c.sp + h * c.sh) * es;
  auto offset = [&](int64_t i) {
    if (whole) return i * 16;
    const int64_t r = (uint64_t)i / (uint32_t)chunks;
    return r * c.ss * es + (i - r * chunks) * 16;
  };
  constexpr int kAtOnce = 4;
  for (int64_t i0 = threadIdx.x; i0 < items; i0 += 256 * kAtOnce) {
    i32x4 k[kAtOnce], v[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t i = i0 + 256 * j;
      if (i >= items) continue;
      const int64_t at = offset(i);
      k[j] = *(const i32x4*)(k0 + at);
      v[j] = *(const i32x4*)(v0 + at);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t i = i0 + 256 * j;
      if (i >= items) continue;
      const int64_t at = offset(i);
      *(i32x4*)(k1 + at) = k[j];
      *(i32x4*)(v1 + at) = v[j];
    }
  }
  if (es == 2) return;
  const int64_t scales = (rows + (1 << c.scale_shift) - 1) >> c.scale_shift;
  for (int64_t i = threadIdx.x; i < scales; i += 256) {
    const int64_t s = src * c.scp + h * c.sch + i * c.scs, d = dst * c.scp + h * c.sch + i * c.scs;
    c.k_scale[d] = c.k_scale[s];
    c.v_scale[d] = c.v_scale[s];
  }
}

// ---- tables ------------------------------------------------------------------------

constexpr int kTableThreads = 1024, kTableWaves = kTableThreads / 64;
constexpr int kListed = 1024;  // new pages that are looked up
constexpr int kPieces = 8;  // pieces of four entries that a lane has at once
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Sum of `x` over the threads before this one; `all`: over all.  wave_sums: LDS.
__device__ __forceinline__ int before(int x, int* wave_sums, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(sum, d);
    if (lane >= d) sum += y;
  }
  __syncthreads();
  if (lane == 63) wave_sums[wave] = sum;
  __syncthreads();
  int base = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kTableWaves; ++w) {
    if (w < wave) base += wave_sums[w];
    all += wave_sums[w];
  }
  return base + sum - x;
}

// What a row of the new table takes over and has room for, in pages.
struct Span {
  int parent;  // row of the old table
  int kept, wanted;
  int part;  // keys of the last page kept, 0: it is full (or none)
};
__device__ __forceinline__ Span span_of(const KvPagesArgs& a, int b) {
  Span s = {a.parent ? a.parent[b] : b, 0, 0, 0};
  const int64_t most = (int64_t)a.max_pages << a.page_shift, page = 1ll << a.page_shift;
  int64_t keep = a.keep[b], want = a.want ? a.want[b] : keep;
  if (s.parent < 0 || s.parent >= a.batch || keep < 0) {
    s.parent = -1;
    return s;
  }
  keep = min(keep, most);
  want = max(min(want, most), keep);
  s.kept = (int)((keep + page - 1) >> a.page_shift);
  s.wanted = (int)((want + page - 1) >> a.page_shift);
  s.part = (int)(keep & (page - 1));
  return s;
}

// One workgroup.  `used`, a bit a page, is what the new table holds: first the
// pages kept whole, which nobody writes, then the last pages that sequences go
// on writing: one stays with its sequence if nobody else keeps it, else with
// the first of those that would write it; the others get a copy.  Free pages
// are then counted off by number to the entries that lack one, by place.
__global__ __launch_bounds__(kTableThreads) void kv_pages_kernel(KvPagesArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  const int words = (a.pages + 31) / 32, room = (words + 3) & ~3;
  uint32_t* used = lds;              // [words]
  uint32_t* twice = used + room;     // [words] pages that several sequences would write
  int* last = (int*)(twice + room);  // [batch] the page that a row would write, -1: none; then -2 - it: a copy
  int* need = last + a.batch;        // [batch] entries without a page; then the sum before
  int* ranks = need + a.batch;       // [kTableThreads + 1] free pages before a thread's words
  int* list = ranks + kTableThreads + 1;  // [kListed] the first free pages
  int* sums = list + kListed;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int w = tid; w < words; w += kTableThreads) {
    uint32_t bits = 0;
    if (a.held)
      for (int i = 0; i < 32 && w * 32 + i < a.pages; ++i) bits |= (uint32_t)(a.held[w * 32 + i] != 0) << i;
    used[w] = bits;
    twice[w] = 0;
  }
  __syncthreads();
  auto bit = [](const uint32_t* m, int p) { return (m[p >> 5] >> (p & 31)) & 1u; };
  // Sixteen lanes have a row, 512 of its entries at a time (entry i0 + 64 j + 4 sub + e is
  // element e of piece j), so that the loads of four rows are under way together.  An
  // entry costs the one CU an instruction for every 64 of them: pieces that a row keeps whole are taken
  // as they are, others and the rest of the row an entry a lane.
  const int sub = lane & 15;
  const uint64_t group = 0xffffull << (lane & 48);
  auto for_rows = [&](auto piece, auto rest) {
    for (int b0 = wave * 4; b0 < a.batch; b0 += kTableWaves * 4) {
      const int b = b0 + (lane >> 4);
      Span s = {-1, 0, 0, 0};
      if (b < a.batch) s = span_of(a, b);
      const int whole = s.part ? s.kept - 1 : s.kept;  // pages kept whole
      const int32_t* row = a.table + (int64_t)max(s.parent, 0) * a.table_stride;
      bool clean = true;
      for (int i0 = 0; i0 < a.max_pages; i0 += 64 * kPieces) {
        i32x4 p[kPieces];
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
          const int i = i0 + 64 * j + 4 * sub;
          if (i + 4 <= whole) p[j] = *(const i32x4_any*)(row + i);
        }
#pragma unroll
        for (int j = 0; j < kPieces; ++j) clean &= piece(b, s, whole, i0 + 64 * j + 4 * sub, p[j]);
      }
      const bool all = !(__builtin_amdgcn_ballot_w64(!clean) & group);
      rest(b, s, whole, row, all);
    }
  };
  auto valid = [&](int p) { return (uint32_t)p < (uint32_t)a.pages; };
  auto mark = [&](int p) { atomicOr(&used[p >> 5], 1u << (p & 31)); };
  // Pages kept whole; entries that lack one.
  int lack = 0;
  for_rows(
      [&](int, const Span&, int whole, int i, const i32x4& p) {
        if (i + 4 > whole) return true;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (valid(p[e])) mark(p[e]);
          else ++lack;
        }
        return true;
      },
      [&](int b, const Span& s, int whole, const int32_t* row, bool) {
        const int i = (whole & ~3) + sub;  // the entries behind the pieces, and the row's last
        int p = -1;
        if (i < s.kept && sub < 4) {
          p = row[i];
          p = valid(p) ? p : -1;
          lack += p < 0;
          if (i < whole && p >= 0) mark(p);
        }
        if (b < a.batch && i == whole) last[b] = s.part ? p : -1;
        int all = lack;
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) all += __shfl_xor(all, d);
        if (b < a.batch && sub == 0) need[b] = all + s.wanted - s.kept;
        lack = 0;
      });
  __syncthreads();
  // Last pages that a sequence keeps whole are copied ...
  for (int b = tid; b < a.batch; b += kTableThreads)
    if (last[b] >= 0 && bit(used, last[b])) last[b] = -2 - last[b];
  __syncthreads();
  for (int b = tid; b < a.batch; b += kTableThreads) {
    const int p = last[b];
    if (p >= 0 && (atomicOr(&used[p >> 5], 1u << (p & 31)) >> (p & 31)) & 1u) atomicOr(&twice[p >> 5], 1u << (p & 31));
  }
  __syncthreads();
  // ... and those of several writers by all but the first.
  for (int b0 = 0; b0 < a.batch; b0 += kTableThreads) {
    const int b = b0 + tid;
    bool copies = false;
    if (b < a.batch) {
      const int p = last[b];
      if (p >= 0 && bit(twice, p))
        for (int i = 0; i < b && !copies; i += 4) {
          const i32x4 four = *(const i32x4*)(last + i);  // (what lies behind the last row: of `need`)
#pragma unroll
          for (int e = 0; e < 4; ++e) copies |= i + e < b && (four[e] == p || four[e] == -2 - p);
        }
    }
    __syncthreads();
    if (copies) last[b] = -2 - last[b];
    __syncthreads();
  }
  // Entries that lack a page before each row's.
  int total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kTableThreads) {
    const int b = b0 + tid;
    const int mine = b < a.batch ? need[b] + (last[b] < -1 ? 1 : 0) : 0;
    int all;
    const int at = before(mine, sums, all);
    if (b < a.batch) need[b] = total + at;
    total += all;
  }
  // Free pages before each thread's words.
  const int per = (words + kTableThreads - 1) / kTableThreads;
  auto free_of = [&](int w) {
    const uint32_t rest = (w + 1) * 32 <= a.pages ? ~0u : (1u << (a.pages & 31)) - 1;
    return ~used[w] & rest;
  };
  int mine = 0, have;
  for (int w = tid * per; w < min(words, (tid + 1) * per); ++w) mine += __popc(free_of(w));
  const int rank = before(mine, sums, have);
  ranks[tid] = rank;
  if (tid == 0) {
    ranks[kTableThreads] = have;
    if (a.lacking) *a.lacking = max(0, total - have);
  }
  __syncthreads();
  // The first of them, in order.
  for (int first = 0; first < a.pages; first += kTableThreads) {
    const int page = first + tid, w = page >> 5, owner = w / per;
    if (ranks[(first >> 5) / per] >= min(total, kListed)) break;  // (the same in all threads)
    if (page >= a.pages || !((free_of(w) >> (page & 31)) & 1)) continue;
    int n = ranks[owner] + __popc(free_of(w) & ((1u << (page & 31)) - 1));
    for (int before_w = owner * per; before_w < w; ++before_w) n += __popc(free_of(before_w));
    if (n < kListed) list[n] = page;
  }
  __syncthreads();
  // The n-th free page, or -1.
  auto nth = [&](int n) {
    if (n >= have) return -1;
    if (n < kListed) return list[n];
    int lo = 0, hi = kTableThreads;  // ranks[lo] <= n < ranks[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (ranks[mid] <= n) lo = mid;
      else hi = mid;
    }
    n -= ranks[lo];
    for (int w = lo * per; w < min(words, (lo + 1) * per); ++w) {
      uint32_t bits = free_of(w);
      const int here = __popc(bits);
      if (n < here) {
        for (; n > 0; --n) bits &= bits - 1;
        return w * 32 + __ffs((int)bits) - 1;
      }
      n -= here;
    }
    return -1;
  };
  for_rows(
      [&](int b, const Span& s, int whole, int i, const i32x4& p) {
        int32_t* out = a.out + (int64_t)b * a.out_stride + i;
        if (b >= a.batch) return true;
        if (i + 4 <= whole) {
          if (!valid(p[0]) || !valid(p[1]) || !valid(p[2]) || !valid(p[3])) return false;
          *(i32x4_any*)out = p;
        } else if (i >= s.wanted && i + 4 <= a.max_pages) {
          *(i32x4_any*)out = i32x4{-1, -1, -1, -1};
        }
        return true;
      },
      [&](int b, const Span& s, int whole, const int32_t* row, bool clean) {
        if (b >= a.batch) return;
        const int page = last[b], end = s.part ? whole : -1;  // the entry that the row writes
        int32_t* out = a.out + (int64_t)b * a.out_stride;
        int lacks = need[b];
        if (sub == 0 && (end < 0 || page >= -1)) {
          if (a.src) a.src[b] = -1;
          if (a.dst) a.dst[b] = -1;
          if (a.rows) a.rows[b] = 0;
        }
        const int stop = min((s.wanted + 3) & ~3, a.max_pages);
        for (int i0 = clean ? whole & ~3 : 0; i0 < stop; i0 += 16) {
          const int i = i0 + sub;
          int p = -1;
          if (i < s.kept) p = i == end ? max(page, -1) : row[i];
          const bool without = i < s.wanted && !valid(p);
          const uint64_t ask = __builtin_amdgcn_ballot_w64(without) & group;
          if (without) p = nth(lacks + __popcll(ask & ((1ull << lane) - 1)));
          lacks += __popcll(ask);
          if (i < stop) out[i] = i < s.wanted ? p : -1;
          if (i == end && page < -1) {
            if (a.src) a.src[b] = p >= 0 ? -2 - page : -1;
            if (a.dst) a.dst[b] = p;
            if (a.rows) a.rows[b] = p >= 0 ? s.part : 0;
          }
        }
        const int i = (a.max_pages & ~3) + sub;  // a last piece that is none
        if (i >= stop && i < a.max_pages) out[i] = -1;
      });
}

}  // namespace

hipError_t kv_compact(const KvCompactArgs& a, hipStream_t s) {
  const int64_t waves = a.batch * a.cache.kv_heads;
  if (waves > UINT32_MAX / 64) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kv_compact_kernel, dim3((unsigned)waves), dim3(64), 0, s, a);
  return hipGetLastError();
}

hipError_t kv_copy_pages(const KvCopyPagesArgs& a, hipStream_t s) {
  const int64_t blocks = a.pairs * a.cache.kv_heads;
  if (blocks > UINT32_MAX / 256) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kv_copy_pages_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
  return hipGetLastError();
}

int64_t kv_pages_lds(int64_t batch, int64_t pages) {
  return (((pages + 31) / 32 + 3) / 4 * 8 + 2 * batch + kTableThreads + 1 + kListed + kTableWaves) * 4;
}

hipError_t kv_pages(const KvPagesArgs& a, hipStream_t s) {
  const int64_t lds = kv_pages_lds(a.batch, a.pages);
  if (lds > kMaxLds) return hipErrorInvalidConfiguration;
  static const hipError_t attr =
      hipFuncSetAttribute((const void*)kv_pages_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLds);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL(kv_pages_kernel, dim3(1), dim3(kTableThreads), (size_t)lds, s, a);
  return hipGetLastError();
}

}  // namespace frisk
