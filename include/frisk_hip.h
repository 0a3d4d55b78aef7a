/*
 * frisk_hip.h — C-ABI of the MI355X (gfx950) GEMM, attention and tile-op
 * kernels.
 *
 * The reference (guoqiao7/frisk) has no execute entry in its FFI: the
 * pass/execute bindings are commented out at ffi/ffi.h:14 and ffi/ffi.cpp:6,
 * and the only GPU path is the out-of-process harness
 * benchmark/layout/execution/run_execution.py:23-95 (frisk-opt -> JSON ->
 * Triton).  These entry points are what that FFI would bind for the GEMM and
 * attention tile programs and the tile ops around them:
 *
 *   frisk_gemm      <- the semantics of frisk.gemm
 *                      (include/Dialect/Frisk/IR/FriskOps.td:252-292;
 *                      shape/type contract lib/Dialect/Frisk/IR/
 *                      LegacyImportSemantics.cpp:11-46, extended to
 *                      int8->int32 and fp8-e4m3->f32/bf16/f16),
 *                      replacing the wgmma emission of
 *                      benchmark/layout/execution/backend.py:383-431.
 *   frisk_attn_fwd  <- the attention tile program (tmp/ir.mlir:89-157,
 *                      benchmark/layout/execution/tiled_attention.py:210-728),
 *                      with online softmax instead of three passes.
 *   frisk_reduce    <- frisk.reduce (include/Dialect/Frisk/IR/FriskOps.td:
 *                      425-453; clear/merge lowering LegacyFragmentNormalization
 *                      .cpp:522-555) and frisk.reduce_tensor (FriskLayoutOps.td:
 *                      17-30) in the canonical_fiber_tree_v1 order
 *                      (lib/Dialect/Frisk/Analysis/ReductionLayoutProof.cpp:
 *                      108-140).
 *   frisk_copy      <- frisk.copy (FriskOps.td:351-397) of a whole tile,
 *                      including the element-type change of a fragment stored
 *                      to global memory (tmp/ir.mlir:154).
 *   frisk_fill      <- frisk.fill (FriskOps.td:400-422; builder ffi/ir.cpp:
 *                      439-454).
 *
 * Beside attention, for serving and training around it (no counterpart in the
 * reference): frisk_rope (rotary positions), frisk_kv_append / frisk_kv_read
 * (a cache of keys and values in 16 or 8 bits), frisk_tree_mask and
 * frisk_tree_attn (attention of new or drafted tokens over that cache).
 *
 * Conventions: plain pointers and sizes only; every pointer is a device
 * pointer owned by the caller; `stream` is a hipStream_t (NULL = the null
 * stream).  Calls are stream-ordered and reentrant.  Every entry returns 0
 * on success or a negative FRISK_E* code; a failed call launches nothing and
 * writes no output, and frisk_last_error() (thread-local) describes why.
 */
#ifndef FRISK_HIP_H
#define FRISK_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FRISK_ABI_VERSION 9

/* Element types (the dtype strings of ffi/ir.cpp:399-411 plus bf16/i8/i32). */
typedef enum frisk_dtype {
  FRISK_F32 = 0,
  FRISK_F16 = 1,
  FRISK_BF16 = 2,
  FRISK_E4M3 = 3, /* OCP float8 e4m3fn */
  FRISK_I8 = 4,
  FRISK_I32 = 5,
  FRISK_F64 = 6
} frisk_dtype;

/* Error codes. */
#define FRISK_OK 0
#define FRISK_EINVAL (-1)   /* bad shape, stride, dtype combination or pointer */
#define FRISK_EUNSUP (-2)   /* valid request this build has no kernel for */
#define FRISK_EHIP (-3)     /* the HIP runtime reported an error */

/*
 * C[m, n] = op(A)[m, k] . op(B)[k, n]   (clear_accum != 0)
 * C[m, n] += op(A)[m, k] . op(B)[k, n]  (clear_accum == 0)
 *
 * op(A) = A (stored [m, k], row stride lda)        when trans_a == 0
 *       = A^T (A stored [k, m], row stride lda)    when trans_a != 0
 * op(B) = B (stored [k, n], row stride ldb)        when trans_b == 0
 *       = B^T (B stored [n, k], row stride ldb)    when trans_b != 0
 * C is stored [m, n] with row stride ldc.  Strides are in elements.
 *
 * Type contract (a_type must equal b_type):
 *   f32  x f32  -> f32
 *   f16  x f16  -> f16 | f32        (f32 accumulation)
 *   bf16 x bf16 -> bf16 | f32       (f32 accumulation)
 *   e4m3 x e4m3 -> bf16 | f16 | f32 (f32 accumulation, then * scale_a*scale_b)
 *   i8   x i8   -> i32              (exact int32 accumulation)
 * scale_a/scale_b are the per-tensor dequantisation factors of fp8 inputs
 * and must be 1.0 for every other type.
 *
 * workspace / workspace_bytes: optional device scratch (16-byte aligned)
 * owned by the caller.  A small-M bf16/f16/f32 GEMM given at least
 * frisk_gemm_workspace_size() bytes splits K over the whole GPU (f32
 * partial tiles, added in a fixed order, so the result does not depend on
 * timing); without it, or when the size is 0, the unsplit kernels run.
 * Two slices are summed inside the GEMM launch, through partials and
 * arrival words in the workspace; its contents before the call do not
 * matter, and nothing needs clearing between calls.  Calls that share a
 * workspace must not overlap.
 */
typedef struct frisk_gemm_desc {
  int64_t m, n, k;
  int32_t trans_a, trans_b;
  int32_t a_type, b_type, c_type; /* frisk_dtype */
  int32_t clear_accum;
  const void* a;
  int64_t lda;
  const void* b;
  int64_t ldb;
  void* c;
  int64_t ldc;
  float scale_a, scale_b;
  void* workspace; /* optional, may be NULL */
  int64_t workspace_bytes;
  /* Optional kernel variant; all zero: the library chooses.  tile = 256:
   * the 256x256 kernel (four waves in a 2x2 grid); tile = 128: the 128x128
   * kernel with a wave_m x wave_n wave grid, one of 2x2, 4x1, 1x4 (256
   * threads) or 2x1, 1x2 (128 threads), 0x0 meaning 2x2.  A requested
   * variant runs unsplit, or with slices > 1 in that many K slices (2x2
   * grid, bf16/f16/f32, N % 4 == 0; placed on stage boundaries as the
   * library's own split; it needs the workspace frisk_gemm_workspace_size
   * reports for the request, and runs unsplit without it).  It returns
   * FRISK_EUNSUP when the descriptor does not meet the matrix-core
   * conditions below.  variant_flags must be 0.  This is how a tile
   * program's instruction contract (its #frisk.mma_contract: MFMA atom and
   * wave grid of the workgroup tile) and the launch contract layout
   * inference gives a whole-matrix GEMM select the kernel that runs. */
  int32_t tile, wave_m, wave_n, variant_flags;
  int32_t slices; /* K slices of a requested variant; 0 or 1: unsplit */
} frisk_gemm_desc;

int frisk_gemm(const frisk_gemm_desc* desc, void* stream);

/* Every storage order of A and B runs on the matrix cores (f32/bf16/f16/fp8/
 * i8; f32 on v_mfma_f32_32x32x2_f32) when the operands have 16-byte aligned
 * bases and row pitches, K * esize is a multiple of 16 for an operand stored
 * K-contiguous (A without trans_a, B with trans_b), C's row pitch is a
 * multiple of 16 bytes, and every buffer a tile addresses spans less than
 * 2^31 bytes.  Anything else ("gemm_generic" in frisk_gemm_plan) runs a
 * matrix-core kernel that takes any alignment and pitch and stages through
 * registers, at about half the rate; it splits K over a workspace like the
 * others, and runs unsplit where a given workspace is short or misaligned. */

/* frisk_gemm without any device allocation by the library or the caller:
 * no hipMalloc, hipFree or allocating library routine is called.  No
 * counterpart in the reference; it is for callers that cannot allocate
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * allocation).  It runs the same kernels as frisk_gemm given a workspace of
 * frisk_gemm_workspace_size(desc) bytes, with the split-K partials in a
 * device array of FRISK_GEMM_NOALLOC_SCRATCH_BYTES that the library holds on
 * every GPU it runs on until the process ends.  desc->workspace must be NULL
 * and workspace_bytes 0.  A GEMM whose split needs more scratch than that is
 * rejected with FRISK_EUNSUP (call frisk_gemm with a workspace instead).
 * Calls on one GPU share that array: calls that overlap in time on one GPU
 * (different streams, or host threads) race on it and must be serialised by
 * the caller; calls ordered on one stream are safe.  The first call on a
 * device looks the array up there (hipGetSymbolAddress): make it outside
 * graph capture (one warm-up call), then capture freely. */
#define FRISK_GEMM_NOALLOC_SCRATCH_BYTES (64ll << 20)
int frisk_gemm_noalloc(const frisk_gemm_desc* desc, void* stream);

/* Workspace bytes that make frisk_gemm(desc) split K (0: none is used), or
 * a negative FRISK_E* code for an invalid descriptor.  Pointers in desc are
 * not read.  No counterpart in the reference (its GEMM ops take no
 * scratch); callers that have none keep calling frisk_gemm unchanged. */
int64_t frisk_gemm_workspace_size(const frisk_gemm_desc* desc);

/* The launch frisk_gemm(desc) makes, as one line of JSON written to buf
 * (len bytes including the terminating NUL): "kernel" (gemm_w4 = 256x256
 * tiles, gemm_128 = 128x128 tiles, gemm_skinny = small M, gemm_generic),
 * "tile_m"/"tile_n", the MFMA "atom", "waves" and "wave_tile" (the wave
 * grid and each wave's sub-tile), "stage_bytes" (K bytes per LDS stage),
 * "a_major"/"b_major" ("k" = K-contiguous storage, "m"/"n" otherwise), the
 * LDS fragment read of each operand ("lds_read_a"/"lds_read_b":
 * ds_read_b128, or ds_read_b64_tr_b16 / _tr_b8 for an M/N-major operand),
 * "slices" (split-K), "slice_sum" ("none", "in_launch": summed by the GEMM
 * kernel itself, "second_launch": by a slice-sum kernel) and
 * "workspace_bytes".  desc->workspace_bytes is taken
 * as the workspace a call would pass; pointers are never read, but when all
 * of a, b and c are given their alignment counts as in frisk_gemm (so a
 * requested variant the tensors cannot run is refused here too).  No
 * counterpart in the reference, whose execution packet records the chosen
 * instruction contract instead (ExportExecution.cpp:46-295): this reports
 * the contract of the kernel the C-ABI selects, for layout checks and
 * tests. */
int frisk_gemm_plan(const frisk_gemm_desc* desc, char* buf, int64_t len);

/*
 * Flash-attention forward over [batch, heads, seq, head_dim] tensors:
 *   O[b,h,i,:] = softmax_j(sm_scale * Q[b,h,i,:].K[b,h,j,:]) . V[b,h,j,:]
 * with j <= i (plus seq_k - seq_q) when causal != 0.  Q/K/V are bf16 or f16
 * (one dtype); O is that dtype or f32 (o_dtype; the reference's tiled
 * attention writes f32 O, tiled_attention.py:658-683).  head_dim is 16, 32,
 * 64 or 128.  The softmax statistics are f32.  Strides are in elements; the
 * innermost (head_dim) stride is 1.  lse, if non-NULL, receives the f32
 * natural-log row log-sum-exp of the scaled scores, laid out
 * [batch, heads, seq_q] contiguous.
 *
 * k_transposed = 1 takes K stored [batch, heads, head_dim, seq_k] with unit
 * key stride (the layout of the reference's FA tile program, K as
 * memref<1x32x128x4096>, tmp/ir.mlir:89-92); k_stride_s is then the stride
 * between head_dim rows (at least seq_k), and seq_k must be even (odd:
 * FRISK_EUNSUP).  The kernel reads it in place.
 */
typedef struct frisk_attn_desc {
  int64_t batch, heads, seq_q, seq_k, head_dim;
  int32_t dtype; /* frisk_dtype: FRISK_BF16 or FRISK_F16 */
  int32_t causal;
  float sm_scale;
  const void* q;
  int64_t q_stride_b, q_stride_h, q_stride_s;
  const void* k;
  int64_t k_stride_b, k_stride_h, k_stride_s;
  const void* v;
  int64_t v_stride_b, v_stride_h, v_stride_s;
  void* o;
  int64_t o_stride_b, o_stride_h, o_stride_s;
  float* lse;
  int32_t o_dtype;      /* frisk_dtype: equal to dtype, or FRISK_F32 */
  int32_t k_transposed; /* 0: K [b, h, seq_k, head_dim]; 1: K [b, h, head_dim, seq_k] */
  /* Waves per workgroup (32 queries each): 0, the library chooses (the
   * launch contract layout inference gives an attention program); 4 or 8
   * (8 needs head_dim 128).  A call that the few-query kernel takes (up to
   * 32 queries and more than 64 to 704 keys, by head_dim, the number of heads
   * and K's storage; "attn_fewq" in the launch contract), whose 4, 8 or 16 waves divide
   * the keys, is checked for it and runs the same with any.  The result bits
   * do not depend on it. */
  int32_t waves;
} frisk_attn_desc;

int frisk_attn_fwd(const frisk_attn_desc* desc, void* stream);

/* frisk_attn_fwd with optional device scratch (16-byte aligned) owned by the
 * caller.  A call with few queries (seq_q <= 32, a decode step) and few heads,
 * given at least frisk_attn_workspace_size() bytes, splits the keys over the
 * whole GPU (f32 partial rows, combined in split order by a second launch, so
 * the same inputs give the same bits); without it, or when the size is 0, it
 * is frisk_attn_fwd.  The contents before a call do not matter; calls that
 * share a workspace must not overlap. */
int frisk_attn_fwd_ws(const frisk_attn_desc* desc, void* workspace, int64_t workspace_bytes,
                      void* stream);

/* Workspace bytes that make frisk_attn_fwd_ws(desc) split the keys (0: none
 * is used), or a negative FRISK_E* code for an invalid descriptor.  Pointers
 * in desc are not read. */
int64_t frisk_attn_workspace_size(const frisk_attn_desc* desc);

/* Reduction kinds (frisk.reduce "add"/"max"/"min", reduce_tensor "sum"/...). */
typedef enum frisk_reduce_kind {
  FRISK_REDUCE_SUM = 0,
  FRISK_REDUCE_MAX = 1,
  FRISK_REDUCE_MIN = 2
} frisk_reduce_kind;

/*
 * Reduction of src[rows, cols] (row stride ld_src) along `axis`:
 *   axis 1:  dst[r * dst_stride] = reduce over c of src[r, c]   (rows outputs)
 *   axis 0:  dst[c * dst_stride] = reduce over r of src[r, c]   (cols outputs)
 * clear == 0 merges with the destination's old value:
 *   dst = combine(dst, reduction)   (frisk.reduce with clear = false).
 * dtype is f32, f16 or bf16 for both src and dst, and every combine is done
 * in it: a sum is rounded to dtype after each addition.  Sums associate as
 * the canonical pairwise tree over the reduced index in ascending order
 * (adjacent pairs first, an odd last node carried up), so results are
 * deterministic and independent of the launch shape.  max / min propagate
 * NaN and order -0.0 below +0.0.  src and dst must not overlap; pointers are
 * element-aligned.  Limits: rows, cols < 2^31; axis 0 needs rows < 2^23.
 *
 * leaf_order_bits > 0 selects another leaf order, that of a distributed
 * layout whose reduced-axis bits sit on single carrier bits (the fibers of
 * canonical_fiber_tree_v1, ReductionLayoutProof.cpp:119-124): the reduced
 * extent must be 2^leaf_order_bits, leaf_order[0..bits) is a permutation of
 * 0..bits-1, and leaf position p holds reduced index
 * sum_j ((p >> j) & 1) << leaf_order[j].  This path runs one thread per
 * output and is meant for tile-sized reductions.
 *
 * workspace / workspace_bytes: optional device scratch (16-byte aligned)
 * owned by the caller.  An axis-0 reduction of many rows with at least
 * frisk_reduce_workspace_size() bytes splits the rows over the whole GPU
 * in two passes (same tree, same result); without it, or when the size is
 * 0, one pass runs.  Calls that share a workspace must not overlap.
 */
typedef struct frisk_reduce_desc {
  int64_t rows, cols;
  int32_t dtype; /* frisk_dtype: FRISK_F32, FRISK_F16 or FRISK_BF16 */
  int32_t kind;  /* frisk_reduce_kind */
  int32_t axis;  /* 0 or 1 */
  int32_t clear;
  const void* src;
  int64_t ld_src;
  void* dst;
  int64_t dst_stride;
  int32_t leaf_order_bits; /* 0: ascending index order */
  uint8_t leaf_order[32];
  void* workspace;         /* optional, may be NULL */
  int64_t workspace_bytes;
} frisk_reduce_desc;

int frisk_reduce(const frisk_reduce_desc* desc, void* stream);

/* Workspace bytes that make frisk_reduce(desc) take its two-pass path (0:
 * none is used), or a negative FRISK_E* code for an invalid descriptor.
 * Pointers in desc are not read. */
int64_t frisk_reduce_workspace_size(const frisk_reduce_desc* desc);

/*
 * dst[r, c] = convert(src[r, c]) for a [rows, cols] tile (row strides
 * ld_src, ld_dst in elements).  Equal types copy the elements unchanged (any
 * frisk_dtype).  Otherwise src_type and dst_type are f32, f16, bf16 or e4m3:
 * widening is exact and narrowing rounds to nearest even (arith.truncf);
 * f16 and bf16 overflow to infinity, e4m3 (no infinity) to NaN.  src and dst
 * must not overlap.
 */
typedef struct frisk_copy_desc {
  int64_t rows, cols;
  int32_t src_type, dst_type; /* frisk_dtype */
  const void* src;
  int64_t ld_src;
  void* dst;
  int64_t ld_dst;
} frisk_copy_desc;

int frisk_copy(const frisk_copy_desc* desc, void* stream);

/*
 * dst[r, c] = value for a [rows, cols] tile (row stride ld).  For float
 * dtypes `value` is rounded to nearest even in dtype (e4m3: values past 464
 * in magnitude become NaN); for i8 / i32 it must be an integer in range.
 */
typedef struct frisk_fill_desc {
  int64_t rows, cols;
  int32_t dtype; /* frisk_dtype */
  double value;
  void* dst;
  int64_t ld;
} frisk_fill_desc;

int frisk_fill(const frisk_fill_desc* desc, void* stream);

/*
 * Rotary positions.  For pair i < rot_dim / 2 of a row at position p, with
 * phi = 2 pi p F_i / 2^64:
 *   (a, b) -> amplitude * (a cos phi - b sin phi, a sin phi + b cos phi)
 * where (a, b) are dims (2i, 2i + 1) when interleaved, else (i, i + rot_dim/2).
 * Dims rot_dim .. head_dim - 1 are copied.  backward = 1 applies the
 * transpose (phi negated): the gradient of x from that of out.  F_i
 * (frequencies, a device array of rot_dim / 2 words) is the pair's turns per
 * position in units of 2^-64, as frisk_rope_frequencies fills it: p F_i mod
 * 2^64 is the exact phase of that frequency at any 64-bit position.  The
 * rotation runs in f32 and is rounded once.
 *
 * One call rotates x and, if k is not NULL, k, by the same positions: two
 * tensors [batch, heads, seq, head_dim] of one dtype (f32, f16 or bf16), unit
 * innermost stride, other strides in elements.  out may be x itself (the same
 * pointer and strides); no other rows of the four tensors may overlap an
 * output.  Rows of tensors with the same strides (a dim of one row has any) are told
 * apart where they lie between each other, others by the ranges they reach.  The position of row (b, s) is
 * start[b] (0 if start is NULL) + positions[b * pos_stride_b + s *
 * pos_stride_s] (s if positions is NULL).
 * Positions of several axes (time, height and width of an image's or a video's
 * tokens): with pair_axis (device) a row has a position on each of `axes` (1 to
 * 4) axes, pos_stride_a apart in positions, and pair i turns by that of
 * axis pair_axis[i]; an axis outside 0 .. axes - 1 counts as 0.
 */
typedef struct frisk_rope_desc {
  int64_t batch, seq, heads, k_heads, head_dim, rot_dim;
  int32_t dtype; /* frisk_dtype: FRISK_F32, FRISK_F16 or FRISK_BF16 */
  int32_t interleaved, backward;
  float amplitude;
  const void* x;
  int64_t x_stride_b, x_stride_h, x_stride_s;
  void* out;
  int64_t out_stride_b, out_stride_h, out_stride_s;
  const void* k; /* optional second tensor */
  int64_t k_stride_b, k_stride_h, k_stride_s;
  void* k_out;
  int64_t k_out_stride_b, k_out_stride_h, k_out_stride_s;
  const void* positions; /* optional */
  int32_t position_bits; /* 32 or 64 (signed) */
  int64_t pos_stride_b, pos_stride_s;
  const int32_t* start; /* optional, [batch] */
  const uint64_t* frequencies;
  int64_t axes, pos_stride_a; /* with pair_axis */
  const uint8_t* pair_axis;   /* optional, [rot_dim / 2] */
} frisk_rope_desc;

int frisk_rope(const frisk_rope_desc* desc, void* stream);

/* How frisk_rope_frequencies slows frequencies down for long contexts, from
 * f_i = base^(-2 i / rot_dim) radians a position:
 *   NONE    f_i
 *   LINEAR  f_i / factor
 *   BASE    base * factor^(rot_dim / (rot_dim - 2)) in the place of base
 *   TURNS   w f_i + (1 - w) f_i / factor, w = clamp((t_i - slow) / (fast -
 *           slow), 0, 1), t_i = trained f_i / (2 pi): turns in the trained length
 *   INDEX   the same with w = 1 - clamp((i - lo) / (hi - lo), 0, 1), lo and hi
 *           the pair indices that turn fast and slow times in the trained length
 *           (lo rounded down, hi up, both held in 0 .. rot_dim - 1, hi at least lo +
 *           0.001) */
typedef enum frisk_rope_scaling {
  FRISK_ROPE_NONE = 0,
  FRISK_ROPE_LINEAR = 1,
  FRISK_ROPE_BASE = 2,
  FRISK_ROPE_TURNS = 3,
  FRISK_ROPE_INDEX = 4
} frisk_rope_scaling;

/* Fills frequencies[0 .. rot_dim / 2) (HOST memory; copy it to the device
 * once) for frisk_rope.  trained, fast and slow are read for TURNS and INDEX. */
int frisk_rope_frequencies(int64_t rot_dim, double base, int32_t scaling, double factor,
                           double trained, double fast, double slow, uint64_t* frequencies);

/*
 * A cache of keys and values.  k and v are [pages, kv_heads, page_size,
 * head_dim] with the strides below (elements, shared by k and v; head_dim
 * stride 1).  dtype bf16 or f16 holds them as they are; e4m3 or i8 holds
 * codes and an f32 scale for each row (page, head, slot) of k and of v: a
 * value is code * scale.  Scales are finite and above 0, or NaN (a value that is
 * NaN makes the o of tokens that see it NaN, not their lse).  Attention may take
 * the product of a weight and a value's scale as 0 below 2^-126, and sums in f32
 * values up to 256 times as large as they are: beyond 2^119 they may overflow.
 * With scale_block = 2^s above 1 (up to 256; with a table at most page_size) the
 * rows of 2^s slots share a scale: k_scale and v_scale are [pages, kv_heads,
 * ceil(page_size / scale_block)], and slot i's is entry i / scale_block.
 * Key n of sequence b is slot n % page_size of page block_table[b *
 * table_stride + n / page_size] (page_size a power of two), or without a
 * table slot n of page b; a sequence holds capacity = max_pages * page_size
 * (without a table page_size) keys.  A page number outside 0 .. pages - 1 is
 * no page: keys there are not written, not read and not seen.  Bases, and row
 * and stride bytes, are multiples of 16.  Rows do not overlap: each stride
 * holds what the smaller ones reach.
 */
typedef struct frisk_kv_cache {
  int64_t pages, kv_heads, page_size, head_dim;
  int32_t dtype; /* frisk_dtype: FRISK_BF16, FRISK_F16, FRISK_E4M3 or FRISK_I8 */
  void* k;
  void* v;
  int64_t stride_page, stride_head, stride_slot;
  float* k_scale; /* 8-bit types only */
  float* v_scale;
  int64_t scale_stride_page, scale_stride_head, scale_stride_slot;
  const int32_t* block_table; /* optional */
  int64_t table_stride, max_pages;
  int64_t scale_block; /* slots that share a scale; 0 or 1: each has its own */
} frisk_kv_cache;

/*
 * frisk_kv_append writes rows [batch, kv_heads, tokens, head_dim] of k and v
 * (bf16 or f16; bases and stride bytes are multiples of 16) into the cache:
 * token t < new_len[b] (all, if new_len is NULL) of sequence b becomes key
 * ctx_len[b] + t; keys behind the capacity or on a
 * page that is none are dropped.  frisk_kv_read is its inverse: those keys, as
 * code * scale rounded to dtype, into k and v, which must not overlap; rows from
 * new_len[b] on, and of keys the cache does not hold, are left as they were.
 * A sequence with ctx_len[b] < 0 takes no part.
 * A row x of an 8-bit cache, with top Q = 448 (e4m3) or 127 (i8): a = max |x|
 * held at least 2^-126 Q, scale = a / Q, code = x Q / a rounded to nearest
 * even.  A row that holds an infinity or a NaN has scale NaN and codes 0: it
 * reads back as NaN.  A 16-bit cache takes and gives its own dtype.
 * Slots that share a scale (scale_block): a block that takes new rows x has, from
 * the largest |x| of those, a and scale as above, or the scale s that it had if
 * that is larger and the block holds keys before ctx_len[b]; a code is x (1 /
 * scale), both f32, rounded to nearest even.  Where the scale grows the codes c of
 * those keys become c (s (1 / scale)), in f32, rounded likewise.  An infinity or
 * NaN makes the block's scale NaN, and all of its keys read back as NaN.
 * What the block holds behind the new rows has no meaning afterwards.
 * So drafts that are rejected leave their mark: the scale that they raised, the second rounding of the
 * codes before them, and NaN if they held a value that is not finite, stay with the block's decided
 * keys, and what is generated over such a cache may depend on the drafts.  Keys appended again from the
 * block's first slot on are as if the drafts had never been there.
 * Pages written by one call must be distinct between its sequences, and k, v
 * and the cache four tensors (six with the scales) that share no memory.
 */
typedef struct frisk_kv_desc {
  int64_t batch, tokens;
  int32_t dtype; /* frisk_dtype of k and v: FRISK_BF16 or FRISK_F16 */
  void* k;       /* read by append, written by read */
  int64_t k_stride_b, k_stride_h, k_stride_s;
  void* v;
  int64_t v_stride_b, v_stride_h, v_stride_s;
  const int32_t* ctx_len; /* [batch] */
  const int32_t* new_len; /* optional, [batch] */
  frisk_kv_cache cache;
} frisk_kv_desc;

int frisk_kv_append(const frisk_kv_desc* desc, void* stream);
int frisk_kv_read(const frisk_kv_desc* desc, void* stream);

/* Masks of drafted trees.  parents [batch, tokens]: the drafted token each one
 * continues (an earlier one), or -1: the context.  Token t sees itself and its
 * ancestors: bit j % 64 of word j / 64 of mask[b][t] ((tokens + 63) / 64 words
 * a token) is set for those, and depth[b][t] (optional) counts the ancestors.
 * A parent outside 0 .. t - 1 counts as -1.  Contiguous; tokens <= 4096. */
int frisk_tree_mask(int64_t batch, int64_t tokens, const int32_t* parents, uint64_t* mask,
                    int32_t* depth, void* stream);

/*
 * Attention of new tokens over a cache that holds them already (frisk_kv_append
 * first): token t < new_len[b] (all, if NULL) of sequence b sees keys 0 ..
 * ctx_len[b] - 1 and, of the new tokens' keys ctx_len[b] + j, those with j < new_len[b]
 * and bit j set in mask[b][t] (without a mask: j <= t):
 *   o[b,h,t,:] = softmax_n(sm_scale q[b,h,t,:] . K[b,h / group,n,:]) . V[b,h / group,n,:]
 * with group = heads / cache.kv_heads.  One token is a decode step, a mask
 * from frisk_tree_mask a step of drafted trees, no mask a prompt's chunk.
 * q is bf16 or f16 [batch, heads, tokens, head_dim]; o is that dtype or f32 (bases
 * multiples of 16 bytes, strides of 8 elements); lse, if
 * given, [batch, heads, tokens] contiguous f32 natural-log sums.  A 16-bit
 * cache has q's dtype.  A token that sees no key has o = 0 and lse = -inf.
 * What a hidden key or its value holds does not matter, NaN and infinities
 * included.  o may be q itself (its dtype and strides); other than that, o, lse and
 * workspace share no memory with each other or with what is read.  Tokens from new_len[b] on, and sequences with ctx_len[b] < 0,
 * are left as they were.  ctx_len and new_len are read on the device;
 * max_ctx (0: the cache's capacity) is a hint of the largest ctx_len that
 * only places the work.  head_dim is a multiple of 16 up to 256; 32, 64 and
 * 128 run on the matrix cores.
 * workspace: optional device scratch (16-byte aligned) of at least
 * frisk_tree_attn_workspace_size() bytes, with which the keys are split over
 * the whole GPU (f32 partial rows, added in split order).  Its contents
 * before a call do not matter; calls that share one must not overlap.
 */
typedef struct frisk_tree_attn_desc {
  int64_t batch, heads, tokens;
  int32_t dtype, o_dtype; /* frisk_dtype */
  float sm_scale;
  const void* q;
  int64_t q_stride_b, q_stride_h, q_stride_s;
  void* o;
  int64_t o_stride_b, o_stride_h, o_stride_s;
  float* lse;
  const int32_t* ctx_len;
  const int32_t* new_len;
  const uint64_t* mask;                 /* optional */
  int64_t mask_stride_b, mask_stride_t; /* words */
  int64_t max_ctx;
  frisk_kv_cache cache;
  void* workspace;
  int64_t workspace_bytes;
} frisk_tree_attn_desc;

int frisk_tree_attn(const frisk_tree_attn_desc* desc, void* stream);
int64_t frisk_tree_attn_workspace_size(const frisk_tree_attn_desc* desc);

/*
 * Pages of a cache.
 *
 * frisk_kv_compact moves the rows of an accepted branch (frisk_tree_verify's path
 * and count) behind the context they continue: for i = 0 .. count[b] - 1 in order,
 * key ctx_len[b] + i becomes the key that was ctx_len[b] + path[b][i].  path [batch,
 * tokens] (row stride path_stride) holds rising draft numbers; an entry
 * below its place i ends the path.  count[b] is held in 0 .. tokens; ctx_len[b] < 0:
 * the sequence takes no part.  A key that the cache does not hold is not moved,
 * nor moved to.  Rows keep their bits; a cache whose slots share scales (scale_block)
 * is FRISK_EUNSUP (append the rows again).
 */
typedef struct frisk_kv_compact_desc {
  int64_t batch, tokens;
  const int32_t* path;
  int64_t path_stride;
  const int32_t* ctx_len; /* [batch] */
  const int32_t* count;   /* [batch] */
  frisk_kv_cache cache;
} frisk_kv_compact_desc;

int frisk_kv_compact(const frisk_kv_compact_desc* desc, void* stream);

/* Copies pages src[i] to dst[i] (i < pairs): k, v and their scales, the first
 * rows[i] slots (all, if rows is NULL; with scale_block the scales of the blocks that
 * these lie in, so that the other slots of such a block no longer hold what they did); the other
 * slots are left as they were.  A pair with a page outside 0 .. pages
 * - 1 is left out.  Pages copied to must be distinct, and none is copied from. */
typedef struct frisk_kv_copy_pages_desc {
  int64_t pairs;
  const int32_t* src; /* [pairs] */
  const int32_t* dst;
  const int32_t* rows; /* optional, [pairs] */
  frisk_kv_cache cache;
} frisk_kv_copy_pages_desc;

int frisk_kv_copy_pages(const frisk_kv_copy_pages_desc* desc, void* stream);

/*
 * The block table of the next step: sequences fork, end, go back and grow.  Row b of
 * `out` continues row parent[b] (its own, if parent is NULL; one outside 0 .. batch - 1:
 * sequence b has ended, its row holds no page): it takes over the pages of that
 * row's first keep[b] keys (a length of the parent's row: entries of kept places that hold no page
 * get a new one, whose keys nobody has written) and has room for want[b] (keep[b], if less, or if want is
 * NULL); both are held in 0 .. max_pages * page_size (keep[b] < 0: the sequence has
 * ended).  Several rows may take over a page.  A last page that is not full,
 * where a row's next keys go, must be its own: where others take that page over in
 * full, or it is held, the row gets a copy, a new page; where several rows would
 * write it, all but the first do.  src[b], dst[b] and rows[b] are that copy's pages and its keys
 * (frisk_kv_copy_pages makes it, for every layer's cache), or -1, -1 and 0.  Every entry with
 * room that has no page gets a new one: in the order of rows and places, the lowest
 * numbers that no row takes over and that are not held (held, optional: [pages] bytes,
 * not 0: a page that is in use elsewhere).  If they do not suffice the last entries
 * are -1 and lacking[0] says how many.  Entries behind the room are -1.  A page
 * that no row has is free: there is no other state.
 * table and out are [batch, max_pages], row strides at least that, and share no memory; lengths
 * and outputs are device arrays.  page_size is a power of two.  FRISK_EUNSUP beyond the kernel's
 * memory: pages / 4 + 8 batch up to 155000 bytes.
 */
typedef struct frisk_kv_pages_desc {
  int64_t batch, max_pages, pages, page_size;
  const int32_t* table;
  int64_t table_stride;
  int32_t* out;
  int64_t out_stride;
  const int32_t* parent; /* optional, [batch] */
  const int32_t* keep;   /* [batch] */
  const int32_t* want;   /* optional, [batch] */
  const uint8_t* held;   /* optional, [pages] */
  int32_t* src;          /* optional, [batch], as the next two */
  int32_t* dst;
  int32_t* rows;
  int32_t* lacking; /* optional, [1] */
} frisk_kv_pages_desc;

int frisk_kv_pages(const frisk_kv_pages_desc* desc, void* stream);

/*
 * Verification of drafted tokens.  A tree's node 0 is a token that is decided (the
 * last one of the step before); node t > 0 is the draft drafts[b][t] that continues
 * node parents[b][t] < t (others are never reached).  logits[b][t] (f32, f16 or bf16
 * [batch, tokens, vocab], unit stride along the vocabulary) are the target's behind node t,
 * p = softmax(logits / temperature[b]) (1, if NULL; 0 or below: the first largest logit has p = 1).
 *
 * From node 0 on, a node's children are tried in order: with a = p, child t with
 * token x is accepted, and the walk goes on from it, if
 *   uniform[b][t] q(x) < a(x);
 * else a becomes max(a - q, 0) over its sum (and stays if that is 0).  q is draft_probs[b][node]
 * (f32 [batch, tokens, vocab], finite and at least 0), from which all of the node's children were
 * drawn independently (with replacement: of children drawn without it the tokens are not distributed
 * as the target's), or, if NULL, certain drafts: q(x) = 1 for the child's own token.  When no child is
 * left, token[b] is the first v at which a summed over 0 .. v passes final_uniform[b]
 * times its whole sum.  Random numbers are of [0, 1).  Probabilities are computed in 64 bits,
 * off by less than 2^-42 of themselves, what rejected drafts leave by 2^-42 of what there was before
 * them; one below 2^-1000 of its row's largest counts as 0.
 * With draft_probs each rejected child of a node but the last costs a pass over the row by one
 * workgroup, and a pass goes through the rejections before it: time grows with their square (64 over
 * a vocabulary of 50257: 7 ms; hundreds over a long one: seconds and more).
 *
 * path[b] ([tokens]) lists the nodes of the walk, node 0 first, then -1; count[b] is their
 * number.  probs[b][t] (optional) is p of a node's token given its parent, 0 for nodes without
 * one.  A row with a NaN, with +infinity or without a logit above -infinity gives no
 * probabilities (probs NaN): the walk ends there and token[b] is -1.  A draft outside the vocabulary
 * is never accepted.  Only the first new_len[b] nodes take part (all, if NULL; below 1: the tree's
 * outputs are left as they were).  temperature is finite.  drafts, parents, uniform, path and probs are contiguous [batch, tokens],
 * final_uniform, temperature, new_len, count and token [batch].  tokens <= 1024, vocab <= 2^24;
 * fewer than 2^22 trees, and fewer than 2^24 segments (of 1 KiB or more) of their rows.
 * workspace (16-byte aligned): at least frisk_tree_verify_workspace_size bytes, which the current
 * device decides (0, and NULL will do, for trees of one node with short rows or many of them); its contents before
 * a call do not matter, and calls that share one must not overlap in time.  No output overlaps another tensor
 * (the rows of logits and of draft_probs count with what lies between them).
 */
typedef struct frisk_tree_verify_desc {
  int64_t batch, tokens, vocab;
  int32_t dtype; /* frisk_dtype of the logits */
  const void* logits;
  int64_t stride_b, stride_t;
  const int32_t* drafts;
  const int32_t* parents;
  const float* uniform;
  const float* final_uniform;
  const float* draft_probs; /* optional */
  int64_t draft_stride_b, draft_stride_t;
  const float* temperature; /* optional */
  const int32_t* new_len;   /* optional */
  int32_t* path;
  int32_t* count;
  int32_t* token;
  float* probs; /* optional */
  void* workspace;
  int64_t workspace_bytes;
} frisk_tree_verify_desc;

int frisk_tree_verify(const frisk_tree_verify_desc* desc, void* stream);
int64_t frisk_tree_verify_workspace_size(const frisk_tree_verify_desc* desc);

/* Description of the last failure on the calling thread ("" if none). */
const char* frisk_last_error(void);

/* FRISK_ABI_VERSION of the loaded library. */
int frisk_abi_version(void);

/* MFMA fragment-layout probe.  No counterpart in the reference, whose SM90
 * fragment maps are pinned by golden rows (SM90MmaLayoutProofTest.cpp:10-82);
 * this one pins the CDNA4 maps the kernels use on the device itself.  Runs
 * one atom (0 = v_mfma_f32_32x32x16_bf16, 1 = v_mfma_f32_16x16x32_bf16,
 * 2 = v_mfma_i32_32x32x32_i8) for every k0 in [0, K) on operands with
 * A[i][k0] = i, A[i][k0+1] = S, B[k0][j] = 1, B[k0+1][j] = j (S = 64, or 32
 * for i8) and writes accumulator register r of lane L for k0 to
 * out[(k0 * 64 + L) * R + r] (R = 16, 4, 16), i.e. the value i + S j of the
 * element it holds.  `out` is a device buffer of at least K * 64 * R floats
 * (16384, 8192 and 32768). */
int frisk_probe_mfma_layout(int atom, float* out, int64_t out_floats, void* stream);

/* Transposing LDS read probe: LDS holds the identity pattern, every lane of
 * one wave addresses the 8 bytes at lane * 8 through ds_read_b64_tr_b16
 * (bits 16: out[lane * 4 + e] = the 16-bit element id returned as element
 * e, 256 values) or ds_read_b64_tr_b8 (bits 8: out[lane * 8 + e] = the byte
 * address returned as byte e, 512 values).  Pins the lane map the GEMM
 * kernels assume for M/N-major operands.  No counterpart in the reference
 * (SM90 has no such instruction). */
int frisk_probe_lds_transpose(int bits, uint16_t* out, int64_t out_elems, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FRISK_HIP_H */
