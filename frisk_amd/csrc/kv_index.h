// Where the keys of a cache lie and which of them a new token sees: the indexing
// of the cache's kernels, without HIP, so that a host program can run it too.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define FRISK_INDEX __device__ __forceinline__
#else
#define FRISK_INDEX inline
#endif

namespace frisk {
namespace kv {

// Keys before the call and new tokens of sequence b; ctx < 0: none of its work.
struct Span {
  int64_t ctx;
  int fresh;
};
FRISK_INDEX Span span_of(const int32_t* ctx_len, const int32_t* new_len, int tokens, int64_t b) {
  int n = tokens;
  if (new_len) n = new_len[b] < 0 ? 0 : new_len[b] < tokens ? new_len[b] : tokens;
  return {ctx_len[b], n};
}

// The scale of row `row` of a page: each one's own, or one for 2^scale_shift rows
// (a Cache without that member has one for each).
template <typename Cache> FRISK_INDEX auto scale_row(const Cache& c, int64_t row, int) -> decltype(c.scale_shift, int64_t()) {
  return row >> c.scale_shift;
}
template <typename Cache> FRISK_INDEX int64_t scale_row(const Cache&, int64_t row, long) { return row; }

// Element and scale offsets of one key's row of head 0; elem < 0: the cache
// does not hold the key.
struct Slot {
  int64_t elem, scale;
};
// The page of key n of sequence b, or -1.  (Cache: KvCache's fields.)
template <typename Cache> FRISK_INDEX int page_of(const Cache& c, int64_t b, int64_t n) {
  if (n < 0 || n >= c.capacity) return -1;
  int64_t page = b;
  if (c.table) page = c.table[b * c.table_stride + (n >> c.page_shift)];
  return page >= 0 && page < c.pages ? (int)page : -1;
}
template <typename Cache> FRISK_INDEX Slot slot_of(const Cache& c, int64_t b, int64_t n) {
  const int page = page_of(c, b, n);
  if (page < 0) return {-1, -1};
  const int64_t row = c.table ? n & ((1ll << c.page_shift) - 1) : n;
  return {page * c.sp + row * c.ss, page * c.scp + scale_row(c, row, 0) * c.scs};
}

}  // namespace kv

namespace tree {

// Keys of a sequence that exist: up to the last new one, and the capacity.
FRISK_INDEX int keys_of(int64_t capacity, const kv::Span& sp) {
  const int64_t n = sp.ctx + sp.fresh;
  return (int)(n < capacity ? n : capacity);
}

// Key blocks per split of a sequence with `blocks` of them: the launch's
// splits, or fewer where they would fall short.
FRISK_INDEX int blocks_per_split(int splits, int min_blocks, int blocks) {
  const int even = (blocks + splits - 1) / splits;
  return min_blocks > even ? min_blocks : even;
}

// The table entry that names key n's page (any value without a table); n is
// held inside the capacity.
template <typename Cache>
FRISK_INDEX int entry_of(const Cache& c, const int32_t* ctx_len, int64_t b, int n) {
  const int last = (int)c.capacity - 1;  // (the capacity fits)
  n = n < 0 ? 0 : n < last ? n : last;
  return c.table ? c.table[b * c.table_stride + (n >> c.page_shift)] : ctx_len[b];
}

// Byte offset of a key's row and element offset of its scale, for one head; a
// key that does not exist has those of the cache's first row.
struct Place {
  int64_t row;
  int64_t scale;
  bool there;
};
template <typename Cache>
FRISK_INDEX Place place_of(const Cache& c, int bytes, int64_t b, int kvh, int n, int keys, int entry) {
  const int page = c.table ? entry : (int)b;
  const int slot = c.table ? n & ((1 << c.page_shift) - 1) : n;
  Place p;
  p.there = n < keys && page >= 0 && page < c.pages;
  const int64_t pg = p.there ? page : 0, sl = p.there ? slot : 0;
  p.row = (pg * c.sp + sl * c.ss + kvh * c.sh) * bytes;
  p.scale = pg * c.scp + kv::scale_row(c, sl, 0) * c.scs + kvh * c.sch;
  return p;
}

// Which keys of the block of 64 from key n0 a token sees, as bits: all of the
// context, drafts by the token's mask words (null: up to its own), of those
// that exist (`there`).
FRISK_INDEX uint64_t seen_bits(const uint64_t* words, int tokens, int t, int64_t ctx, int n0, uint64_t there) {
  const int64_t j0 = n0 - ctx;  // draft number of the first key
  if (j0 + 64 <= 0) return there;
  uint64_t bits;
  if (!words) {
    const int64_t n = t - j0 + 1;  // the first n keys
    bits = n >= 64 ? ~0ull : n <= 0 ? 0 : (1ull << n) - 1;
  } else {
    const int count = (tokens + 63) >> 6;
    if (j0 < 0) {
      const int n = (int)-j0;  // context keys in front, 1 .. 63
      bits = ((1ull << n) - 1) | (words[0] << n);
    } else {
      const int64_t i = j0 >> 6;
      const int s = (int)(j0 & 63);
      bits = i < count ? words[i] >> s : 0;
      if (s && i + 1 < count) bits |= words[i + 1] << (64 - s);
    }
  }
  return bits & there;
}

}  // namespace tree
}  // namespace frisk
