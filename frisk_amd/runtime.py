"""ctypes binding of libfrisk_hip.so (include/frisk_hip.h).

This is the Python side of the C-ABI: it fills the descriptors from torch
device tensors and calls frisk_gemm / frisk_attn_fwd / frisk_reduce /
frisk_copy / frisk_fill, and frisk_rope / frisk_kv_append / frisk_kv_read /
frisk_tree_mask / frisk_tree_attn / frisk_tree_verify / frisk_kv_compact /
frisk_kv_copy_pages / frisk_kv_pages, on the current HIP stream.  There is no fallback: if the library is missing or a call fails,
a RuntimeError (or ValueError for rejected requests, matching the
reference's ValueError on contract violations, ffi/ir.cpp:333-341) is raised.
"""
from __future__ import annotations

import ctypes
import os
import struct
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libfrisk_hip.so"

F32, F16, BF16, E4M3, I8, I32, F64 = 0, 1, 2, 3, 4, 5, 6
OK, EINVAL, EUNSUP, EHIP = 0, -1, -2, -3

DTYPE_NAMES = {F32: "f32", F16: "f16", BF16: "bf16", E4M3: "e4m3", I8: "i8", I32: "i32", F64: "f64"}

# Exported symbols declared by include/frisk_hip.h.
EXPORTS = ("frisk_gemm", "frisk_gemm_workspace_size", "frisk_gemm_plan", "frisk_gemm_noalloc",
           "frisk_attn_fwd", "frisk_attn_fwd_ws", "frisk_attn_workspace_size",
           "frisk_reduce", "frisk_reduce_workspace_size",
           "frisk_copy", "frisk_fill",
           "frisk_rope", "frisk_rope_frequencies", "frisk_kv_append", "frisk_kv_read",
           "frisk_tree_mask", "frisk_tree_attn", "frisk_tree_attn_workspace_size",
           "frisk_kv_compact", "frisk_kv_copy_pages", "frisk_kv_pages",
           "frisk_tree_verify", "frisk_tree_verify_workspace_size",
           "frisk_last_error", "frisk_abi_version", "frisk_probe_mfma_layout",
           "frisk_probe_lds_transpose")
ABI_VERSION = 9

REDUCE_SUM, REDUCE_MAX, REDUCE_MIN = 0, 1, 2
REDUCE_KINDS = {"sum": REDUCE_SUM, "add": REDUCE_SUM, "max": REDUCE_MAX, "min": REDUCE_MIN}


class GemmDesc(ctypes.Structure):
    _fields_ = [
        ("m", ctypes.c_int64), ("n", ctypes.c_int64), ("k", ctypes.c_int64),
        ("trans_a", ctypes.c_int32), ("trans_b", ctypes.c_int32),
        ("a_type", ctypes.c_int32), ("b_type", ctypes.c_int32), ("c_type", ctypes.c_int32),
        ("clear_accum", ctypes.c_int32),
        ("a", ctypes.c_void_p), ("lda", ctypes.c_int64),
        ("b", ctypes.c_void_p), ("ldb", ctypes.c_int64),
        ("c", ctypes.c_void_p), ("ldc", ctypes.c_int64),
        ("scale_a", ctypes.c_float), ("scale_b", ctypes.c_float),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64),
        ("tile", ctypes.c_int32), ("wave_m", ctypes.c_int32), ("wave_n", ctypes.c_int32),
        ("variant_flags", ctypes.c_int32), ("slices", ctypes.c_int32),
    ]


class AttnDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int64), ("heads", ctypes.c_int64), ("seq_q", ctypes.c_int64),
        ("seq_k", ctypes.c_int64), ("head_dim", ctypes.c_int64),
        ("dtype", ctypes.c_int32), ("causal", ctypes.c_int32), ("sm_scale", ctypes.c_float),
        ("q", ctypes.c_void_p), ("q_stride_b", ctypes.c_int64), ("q_stride_h", ctypes.c_int64),
        ("q_stride_s", ctypes.c_int64),
        ("k", ctypes.c_void_p), ("k_stride_b", ctypes.c_int64), ("k_stride_h", ctypes.c_int64),
        ("k_stride_s", ctypes.c_int64),
        ("v", ctypes.c_void_p), ("v_stride_b", ctypes.c_int64), ("v_stride_h", ctypes.c_int64),
        ("v_stride_s", ctypes.c_int64),
        ("o", ctypes.c_void_p), ("o_stride_b", ctypes.c_int64), ("o_stride_h", ctypes.c_int64),
        ("o_stride_s", ctypes.c_int64),
        ("lse", ctypes.c_void_p),
        ("o_dtype", ctypes.c_int32),
        ("k_transposed", ctypes.c_int32), ("waves", ctypes.c_int32),
    ]


class ReduceDesc(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
        ("dtype", ctypes.c_int32), ("kind", ctypes.c_int32), ("axis", ctypes.c_int32),
        ("clear", ctypes.c_int32),
        ("src", ctypes.c_void_p), ("ld_src", ctypes.c_int64),
        ("dst", ctypes.c_void_p), ("dst_stride", ctypes.c_int64),
        ("leaf_order_bits", ctypes.c_int32), ("leaf_order", ctypes.c_uint8 * 32),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64),
    ]


class CopyDesc(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
        ("src_type", ctypes.c_int32), ("dst_type", ctypes.c_int32),
        ("src", ctypes.c_void_p), ("ld_src", ctypes.c_int64),
        ("dst", ctypes.c_void_p), ("ld_dst", ctypes.c_int64),
    ]


class FillDesc(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
        ("dtype", ctypes.c_int32), ("value", ctypes.c_double),
        ("dst", ctypes.c_void_p), ("ld", ctypes.c_int64),
    ]


_i64, _i32, _ptr = ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p


def _strides(prefix, names):
    return [(f"{prefix}_stride_{n}", _i64) for n in names]


class RopeDesc(ctypes.Structure):
    _fields_ = [
        *((n, _i64) for n in ("batch", "seq", "heads", "k_heads", "head_dim", "rot_dim")),
        ("dtype", _i32), ("interleaved", _i32), ("backward", _i32), ("amplitude", ctypes.c_float),
        ("x", _ptr), *_strides("x", "bhs"), ("out", _ptr), *_strides("out", "bhs"),
        ("k", _ptr), *_strides("k", "bhs"), ("k_out", _ptr), *_strides("k_out", "bhs"),
        ("positions", _ptr), ("position_bits", _i32), *_strides("pos", "bs"),
        ("start", _ptr), ("frequencies", _ptr),
        ("axes", _i64), ("pos_stride_a", _i64), ("pair_axis", _ptr),
    ]


class KvCacheDesc(ctypes.Structure):
    _fields_ = [
        ("pages", _i64), ("kv_heads", _i64), ("page_size", _i64), ("head_dim", _i64),
        ("dtype", _i32), ("k", _ptr), ("v", _ptr),
        ("stride_page", _i64), ("stride_head", _i64), ("stride_slot", _i64),
        ("k_scale", _ptr), ("v_scale", _ptr),
        ("scale_stride_page", _i64), ("scale_stride_head", _i64), ("scale_stride_slot", _i64),
        ("block_table", _ptr), ("table_stride", _i64), ("max_pages", _i64), ("scale_block", _i64),
    ]


class KvDesc(ctypes.Structure):
    _fields_ = [
        ("batch", _i64), ("tokens", _i64), ("dtype", _i32),
        ("k", _ptr), *_strides("k", "bhs"), ("v", _ptr), *_strides("v", "bhs"),
        ("ctx_len", _ptr), ("new_len", _ptr), ("cache", KvCacheDesc),
    ]


class TreeAttnDesc(ctypes.Structure):
    _fields_ = [
        ("batch", _i64), ("heads", _i64), ("tokens", _i64), ("dtype", _i32), ("o_dtype", _i32),
        ("sm_scale", ctypes.c_float), ("q", _ptr), *_strides("q", "bhs"),
        ("o", _ptr), *_strides("o", "bhs"), ("lse", _ptr), ("ctx_len", _ptr), ("new_len", _ptr),
        ("mask", _ptr), *_strides("mask", "bt"), ("max_ctx", _i64), ("cache", KvCacheDesc),
        ("workspace", _ptr), ("workspace_bytes", _i64),
    ]


class KvCompactDesc(ctypes.Structure):
    _fields_ = [
        ("batch", _i64), ("tokens", _i64), ("path", _ptr), ("path_stride", _i64),
        ("ctx_len", _ptr), ("count", _ptr), ("cache", KvCacheDesc),
    ]


class KvCopyPagesDesc(ctypes.Structure):
    _fields_ = [("pairs", _i64), ("src", _ptr), ("dst", _ptr), ("rows", _ptr), ("cache", KvCacheDesc)]


class KvPagesDesc(ctypes.Structure):
    _fields_ = [
        ("batch", _i64), ("max_pages", _i64), ("pages", _i64), ("page_size", _i64),
        ("table", _ptr), ("table_stride", _i64), ("out", _ptr), ("out_stride", _i64),
        *((n, _ptr) for n in ("parent", "keep", "want", "held", "src", "dst", "rows", "lacking")),
    ]


class TreeVerifyDesc(ctypes.Structure):
    _fields_ = [
        ("batch", _i64), ("tokens", _i64), ("vocab", _i64), ("dtype", _i32),
        ("logits", _ptr), ("stride_b", _i64), ("stride_t", _i64),
        *((n, _ptr) for n in ("drafts", "parents", "uniform", "final_uniform", "draft_probs")),
        ("draft_stride_b", _i64), ("draft_stride_t", _i64),
        *((n, _ptr) for n in ("temperature", "new_len", "path", "count", "token", "probs")),
        ("workspace", _ptr), ("workspace_bytes", _i64),
    ]


_lib = None


def load() -> ctypes.CDLL:
    """Load libfrisk_hip.so once; raise if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -m frisk_amd.build` "
            "(there is no CPU fallback for the GEMM/attention path)")
    lib = ctypes.CDLL(str(LIB_PATH))
    lib.frisk_gemm.argtypes = [ctypes.POINTER(GemmDesc), ctypes.c_void_p]
    lib.frisk_gemm.restype = ctypes.c_int
    lib.frisk_gemm_workspace_size.argtypes = [ctypes.POINTER(GemmDesc)]
    lib.frisk_gemm_workspace_size.restype = ctypes.c_int64
    lib.frisk_gemm_plan.argtypes = [ctypes.POINTER(GemmDesc), ctypes.c_char_p, ctypes.c_int64]
    lib.frisk_gemm_plan.restype = ctypes.c_int
    lib.frisk_gemm_noalloc.argtypes = [ctypes.POINTER(GemmDesc), ctypes.c_void_p]
    lib.frisk_gemm_noalloc.restype = ctypes.c_int
    lib.frisk_attn_fwd.argtypes = [ctypes.POINTER(AttnDesc), ctypes.c_void_p]
    lib.frisk_attn_fwd.restype = ctypes.c_int
    lib.frisk_attn_fwd_ws.argtypes = [ctypes.POINTER(AttnDesc), ctypes.c_void_p, ctypes.c_int64,
                                      ctypes.c_void_p]
    lib.frisk_attn_fwd_ws.restype = ctypes.c_int
    lib.frisk_attn_workspace_size.argtypes = [ctypes.POINTER(AttnDesc)]
    lib.frisk_attn_workspace_size.restype = ctypes.c_int64
    lib.frisk_reduce.argtypes = [ctypes.POINTER(ReduceDesc), ctypes.c_void_p]
    lib.frisk_reduce.restype = ctypes.c_int
    lib.frisk_reduce_workspace_size.argtypes = [ctypes.POINTER(ReduceDesc)]
    lib.frisk_reduce_workspace_size.restype = ctypes.c_int64
    lib.frisk_copy.argtypes = [ctypes.POINTER(CopyDesc), ctypes.c_void_p]
    lib.frisk_copy.restype = ctypes.c_int
    lib.frisk_fill.argtypes = [ctypes.POINTER(FillDesc), ctypes.c_void_p]
    lib.frisk_fill.restype = ctypes.c_int
    lib.frisk_rope.argtypes = [ctypes.POINTER(RopeDesc), ctypes.c_void_p]
    lib.frisk_rope.restype = ctypes.c_int
    lib.frisk_rope_frequencies.argtypes = [_i64, ctypes.c_double, _i32, *[ctypes.c_double] * 4,
                                           ctypes.POINTER(ctypes.c_uint64)]
    lib.frisk_rope_frequencies.restype = ctypes.c_int
    for fn in (lib.frisk_kv_append, lib.frisk_kv_read):
        fn.argtypes = [ctypes.POINTER(KvDesc), ctypes.c_void_p]
        fn.restype = ctypes.c_int
    lib.frisk_tree_mask.argtypes = [_i64, _i64, _ptr, _ptr, _ptr, _ptr]
    lib.frisk_tree_mask.restype = ctypes.c_int
    lib.frisk_tree_attn.argtypes = [ctypes.POINTER(TreeAttnDesc), ctypes.c_void_p]
    lib.frisk_tree_attn.restype = ctypes.c_int
    lib.frisk_tree_attn_workspace_size.argtypes = [ctypes.POINTER(TreeAttnDesc)]
    lib.frisk_tree_attn_workspace_size.restype = ctypes.c_int64
    for fn, desc in ((lib.frisk_kv_compact, KvCompactDesc), (lib.frisk_kv_copy_pages, KvCopyPagesDesc),
                     (lib.frisk_kv_pages, KvPagesDesc), (lib.frisk_tree_verify, TreeVerifyDesc)):
        fn.argtypes = [ctypes.POINTER(desc), ctypes.c_void_p]
        fn.restype = ctypes.c_int
    lib.frisk_tree_verify_workspace_size.argtypes = [ctypes.POINTER(TreeVerifyDesc)]
    lib.frisk_tree_verify_workspace_size.restype = ctypes.c_int64
    lib.frisk_last_error.argtypes = []
    lib.frisk_last_error.restype = ctypes.c_char_p
    lib.frisk_abi_version.argtypes = []
    lib.frisk_abi_version.restype = ctypes.c_int
    lib.frisk_probe_mfma_layout.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_int64,
                                            ctypes.c_void_p]
    lib.frisk_probe_mfma_layout.restype = ctypes.c_int
    lib.frisk_probe_lds_transpose.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_int64,
                                              ctypes.c_void_p]
    lib.frisk_probe_lds_transpose.restype = ctypes.c_int
    if lib.frisk_abi_version() != ABI_VERSION:
        raise RuntimeError("libfrisk_hip.so ABI version mismatch; rebuild it")
    _lib = lib
    return lib


def _check(rc: int, what: str) -> None:
    if rc == OK:
        return
    msg = load().frisk_last_error().decode()
    if rc in (EINVAL, EUNSUP):
        raise ValueError(f"{what}: {msg}")
    raise RuntimeError(f"{what}: {msg}")


_dtype_codes: dict = {}


def torch_dtype_code(dt) -> int:
    if not _dtype_codes:
        import torch
        _dtype_codes.update({
            torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16,
            torch.float8_e4m3fn: E4M3, torch.int8: I8, torch.int32: I32, torch.float64: F64,
        })
    code = _dtype_codes.get(dt)
    if code is None:
        raise ValueError(f"unsupported tensor dtype {dt}")
    return code


def _stream_handle(stream) -> int:
    import torch
    if stream is None:
        # torch's raw accessor returns the current stream's handle without
        # building a Stream object (0.1 us against 3 us per launch); the
        # public path stays as the fallback.
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if raw is not None:
            return int(raw(torch.cuda.current_device()))
        stream = torch.cuda.current_stream()
    return int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)


def _empty(shape, dtype, device, stream, fill=None):
    """A new tensor, allocated (and filled) on the stream that the call's kernels run on:
    the allocator may have had its memory in use by, and may hand it out again to,
    work of that stream only."""
    import torch
    if stream is None:
        t = torch.empty(shape, dtype=dtype, device=device)
        return t if fill is None else t.fill_(fill)
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    with torch.cuda.stream(stream):
        return _empty(shape, dtype, device, None, fill)


def _scratch(nbytes: int, device, stream):
    """A call's scratch."""
    import torch
    return _empty(nbytes, torch.uint8, device, stream)


def _row_major(t, name: str) -> int:
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be a rank-2 tensor with unit column stride")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    return t.stride(0)


def gemm_desc(a, b, c, *, trans_a=False, trans_b=False, clear_accum=True,
              scale_a=1.0, scale_b=1.0, variant=None) -> GemmDesc:
    """Describe C (+)= op(A).op(B) for row-major device tensors (see frisk_hip.h).
    `variant` = (tile, wave_m, wave_n) or (tile, wave_m, wave_n, slices)
    requests a kernel variant (frisk_gemm_desc.tile ... slices)."""
    lda, ldb, ldc = _row_major(a, "A"), _row_major(b, "B"), _row_major(c, "C")
    m = a.shape[1] if trans_a else a.shape[0]
    k = a.shape[0] if trans_a else a.shape[1]
    kb = b.shape[1] if trans_b else b.shape[0]
    n = b.shape[0] if trans_b else b.shape[1]
    if kb != k or tuple(c.shape) != (m, n):
        raise ValueError(f"legacy-gemm-shape: effective shapes A{tuple(a.shape)} B{tuple(b.shape)} "
                         f"C{tuple(c.shape)} do not form an MxK . KxN -> MxN product")
    return GemmDesc(m, n, k, int(bool(trans_a)), int(bool(trans_b)),
                    torch_dtype_code(a.dtype), torch_dtype_code(b.dtype), torch_dtype_code(c.dtype),
                    int(bool(clear_accum)), a.data_ptr(), lda, b.data_ptr(), ldb,
                    c.data_ptr(), ldc, float(scale_a), float(scale_b), None, 0,
                    *(tuple(variant[:3]) if variant else (0, 0, 0)), 0,
                    int(variant[3]) if variant and len(variant) > 3 else 0)


def workspace_bytes_of(desc: GemmDesc) -> int:
    """frisk_gemm_workspace_size for a descriptor."""
    need = int(load().frisk_gemm_workspace_size(ctypes.byref(desc)))
    _check(need if need < 0 else OK, "frisk_gemm_workspace_size")
    return need


def gemm_workspace_bytes(a, b, c, *, trans_a=False, trans_b=False) -> int:
    """frisk_gemm_workspace_size for gemm(a, b, c, ...): 0 when no split-K applies."""
    return workspace_bytes_of(gemm_desc(a, b, c, trans_a=trans_a, trans_b=trans_b))


def plan_of(desc: GemmDesc) -> dict:
    """frisk_gemm_plan for a descriptor: the launch frisk_gemm would make."""
    import json
    buf = ctypes.create_string_buffer(1024)
    _check(load().frisk_gemm_plan(ctypes.byref(desc), buf, len(buf)), "frisk_gemm_plan")
    return json.loads(buf.value.decode())


def gemm_plan(a, b, c, *, trans_a=False, trans_b=False, workspace=True, variant=None) -> dict:
    """The launch gemm(a, b, c, ..., workspace=workspace, variant=variant) makes
    (frisk_gemm_plan): kernel, tiles, MFMA atom, wave grid, operand storage
    order and LDS reads, split-K, and the kernel's instruction contract."""
    d = gemm_desc(a, b, c, trans_a=trans_a, trans_b=trans_b, variant=variant)
    if workspace is not False:
        need = int(load().frisk_gemm_workspace_size(ctypes.byref(d)))
        _check(need if need < 0 else OK, "frisk_gemm_workspace_size")
        d.workspace_bytes = need if workspace is True else workspace.numel() * workspace.element_size()
    return plan_of(d)


def gemm(a, b, c, *, trans_a=False, trans_b=False, clear_accum=True,
         scale_a=1.0, scale_b=1.0, workspace=True, stream=None, variant=None):
    """C = op(A).op(B) (or C += ... with clear_accum=False) on the GPU.

    `workspace`: True allocates the scratch frisk_gemm_workspace_size asks
    for (torch's caching allocator), a device tensor supplies it, False runs
    the unsplit kernels.  `variant` = (tile, wave_m, wave_n[, slices]) runs
    that kernel variant: (256, 2, 2), or (128, gm, gn) with the wave grid
    2x2, 4x1, 1x4, 2x1 or 1x2, unsplit or (2x2 grid) in `slices` K slices."""
    d = gemm_desc(a, b, c, trans_a=trans_a, trans_b=trans_b, clear_accum=clear_accum,
                  scale_a=scale_a, scale_b=scale_b, variant=variant)
    ws = None
    if workspace is not False:
        need = load().frisk_gemm_workspace_size(ctypes.byref(d))
        _check(int(need) if need < 0 else OK, "frisk_gemm_workspace_size")
        if need > 0:
            ws = workspace if workspace is not True else _scratch(need, c.device, stream)
            d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
    _check(load().frisk_gemm(ctypes.byref(d), ctypes.c_void_p(_stream_handle(stream))),
           "frisk_gemm")
    return c


# FRISK_GEMM_NOALLOC_SCRATCH_BYTES of include/frisk_hip.h.
NOALLOC_SCRATCH_BYTES = 64 << 20


def gemm_noalloc(a, b, c, *, trans_a=False, trans_b=False, clear_accum=True,
                 scale_a=1.0, scale_b=1.0, stream=None):
    """frisk_gemm_noalloc: gemm() with the split-K partials in the library's
    own device scratch; nothing is allocated."""
    d = gemm_desc(a, b, c, trans_a=trans_a, trans_b=trans_b, clear_accum=clear_accum,
                  scale_a=scale_a, scale_b=scale_b)
    _check(load().frisk_gemm_noalloc(ctypes.byref(d), ctypes.c_void_p(_stream_handle(stream))),
           "frisk_gemm_noalloc")
    return c


# Atom codes of frisk_probe_mfma_layout: (mfma name, K, accumulators per lane, S).
PROBE_ATOMS = {0: ("v_mfma_f32_32x32x16_bf16", 16, 16, 64),
               1: ("v_mfma_f32_16x16x32_bf16", 32, 4, 64),
               2: ("v_mfma_i32_32x32x32_i8", 32, 16, 32)}


def probe_mfma_layout(atom: int, out, stream=None):
    """Run the MFMA layout probe into the f32 device tensor `out`."""
    if out.dtype.is_floating_point is False or out.element_size() != 4 or not out.is_contiguous() \
            or not out.is_cuda:
        raise ValueError("out must be a contiguous f32 device tensor")
    _check(load().frisk_probe_mfma_layout(int(atom), ctypes.c_void_p(out.data_ptr()), out.numel(),
                                          ctypes.c_void_p(_stream_handle(stream))),
           "frisk_probe_mfma_layout")
    return out


def probe_lds_transpose(bits: int, out, stream=None):
    """Run the transposing LDS read probe into the int16/uint16 device tensor `out`."""
    if out.element_size() != 2 or not out.is_contiguous() or not out.is_cuda:
        raise ValueError("out must be a contiguous 16-bit device tensor")
    _check(load().frisk_probe_lds_transpose(int(bits), ctypes.c_void_p(out.data_ptr()), out.numel(),
                                            ctypes.c_void_p(_stream_handle(stream))),
           "frisk_probe_lds_transpose")
    return out


def attn_desc(q, k, v, o, *, causal=False, sm_scale=None, lse=None,
              k_transposed=False, waves=0) -> AttnDesc:
    """Describe the attention forward of [batch, heads, seq, head_dim] device
    tensors; with k_transposed, K is [batch, heads, head_dim, seq_k] with unit
    key stride (read in place, not copied)."""
    shapes, strides = [], []
    for name, t in (("Q", q), ("K", k), ("V", v), ("O", o)):
        sh, st = t.shape, t.stride()
        if len(sh) != 4 or st[3] != 1 or not t.is_cuda:
            inner = "seq_k" if name == "K" and k_transposed else "head_dim"
            raise ValueError(f"{name} must be a rank-4 device tensor with unit {inner} stride")
        shapes.append(tuple(sh))
        strides.append(st)
    b, h, sq, d = shapes[0]
    sk = shapes[1][3] if k_transposed else shapes[1][2]
    k_shape = (b, h, d, sk) if k_transposed else (b, h, sk, d)
    if shapes[1] != k_shape or shapes[2] != (b, h, sk, d) or shapes[3] != (b, h, sq, d):
        raise ValueError("attention shapes disagree")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("Q/K/V must share one dtype")
    import torch
    if o.dtype not in (q.dtype, torch.float32):
        raise ValueError("O must have the Q/K/V dtype or float32")
    if lse is not None and (tuple(lse.shape) != (b, h, sq) or not lse.is_contiguous()
                            or lse.dtype.is_floating_point is False or lse.element_size() != 4):
        raise ValueError("lse must be a contiguous f32 [batch, heads, seq_q] tensor")
    if sm_scale is None:
        sm_scale = d ** -0.5
    qs, ks, vs, os_ = strides
    return AttnDesc(b, h, sq, sk, d, torch_dtype_code(q.dtype), int(bool(causal)),
                    float(sm_scale),
                    q.data_ptr(), qs[0], qs[1], qs[2],
                    k.data_ptr(), ks[0], ks[1], ks[2],
                    v.data_ptr(), vs[0], vs[1], vs[2],
                    o.data_ptr(), os_[0], os_[1], os_[2],
                    lse.data_ptr() if lse is not None else None, torch_dtype_code(o.dtype),
                    int(bool(k_transposed)), int(waves))


# frisk_attn_fwd_ws splits the keys only of calls with at most FEW_QUERIES
# queries and more than FEW_KEYS keys.
FEW_QUERIES, FEW_KEYS = 32, 768


def requested_waves(contract: dict) -> int:
    """AttnDesc.waves of an attention launch contract: the waves of the kernel
    that gives every wave its own queries; the few-query kernel takes none."""
    return contract["waves"] if contract["kernel"] == "attn_fwd" else 0


def attn_fwd(q, k, v, o, *, causal=False, sm_scale=None, lse=None, stream=None,
             k_transposed=False, waves=0):
    """O = softmax(sm_scale . Q K^T [causal mask]) V on the GPU.  K is
    [batch, heads, seq_k, head_dim], or [batch, heads, head_dim, seq_k] with
    k_transposed=True (read in place).  `waves` (4 or 8) requests the
    workgroup shape; 0 lets the library choose.  Few queries over many keys
    take scratch from torch's caching allocator, on the call's stream."""
    d = attn_desc(q, k, v, o, causal=causal, sm_scale=sm_scale, lse=lse, k_transposed=k_transposed,
                  waves=waves)
    lib, ws, need = load(), None, 0
    if d.seq_q <= FEW_QUERIES and d.seq_k > FEW_KEYS:
        need = lib.frisk_attn_workspace_size(ctypes.byref(d))
        _check(int(need) if need < 0 else OK, "frisk_attn_fwd")
    if need > 0:
        ws = _scratch(need, o.device, stream)
        rc = lib.frisk_attn_fwd_ws(ctypes.byref(d), ws.data_ptr(), need,
                                   ctypes.c_void_p(_stream_handle(stream)))
    else:
        rc = lib.frisk_attn_fwd(ctypes.byref(d), ctypes.c_void_p(_stream_handle(stream)))
    _check(rc, "frisk_attn_fwd")
    return o


def _matrix(t, name: str):
    """(rows, cols, row stride) of a rank-1 or rank-2 device tensor with unit
    innermost stride; a rank-1 tensor is one row."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dim() == 1:
        if t.stride(0) != 1 and t.numel() > 1:
            raise ValueError(f"{name} must have unit stride")
        return 1, t.shape[0], max(t.shape[0], 1)
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be a rank-1 or rank-2 tensor with unit column stride")
    return t.shape[0], t.shape[1], max(t.stride(0), t.shape[1])


def reduce_workspace_bytes(src, dst, kind="sum", *, axis=1) -> int:
    """frisk_reduce_workspace_size for reduce(src, dst, kind, axis=axis)."""
    rows, cols, ld = _matrix(src, "src")
    d = ReduceDesc(rows, cols, torch_dtype_code(src.dtype), REDUCE_KINDS[kind], axis, 1,
                   src.data_ptr(), ld, dst.data_ptr(), max(dst.stride(0), 1))
    need = int(load().frisk_reduce_workspace_size(ctypes.byref(d)))
    _check(need if need < 0 else OK, "frisk_reduce_workspace_size")
    return need


def reduce(src, dst, kind="sum", *, axis=1, clear=True, leaf_order=None, workspace=True,
           stream=None):
    """frisk.reduce: dst = reduce(src) along `axis` of the [rows, cols] tensor
    src (or dst = combine(dst, reduce(src)) with clear=False).  dst is a
    rank-1 tensor of the kept extent, any stride, same dtype.  `leaf_order`
    (a permutation of the reduced index bits, tree level j along bit
    leaf_order[j]) replaces the ascending leaf order.  `workspace`: True
    allocates the scratch frisk_reduce_workspace_size asks for (torch's
    caching allocator), a uint8 device tensor supplies it, False runs the
    single-pass kernels."""
    rows, cols, ld = _matrix(src, "src")
    if src.dim() != 2:
        raise ValueError("src must be rank 2")
    if kind not in REDUCE_KINDS:
        raise ValueError(f"unknown reduction kind {kind!r} (sum/add, max, min)")
    if axis not in (0, 1):
        raise ValueError("axis must be 0 or 1")
    n = rows if axis == 1 else cols
    if dst.dim() != 1 or dst.shape[0] != n or not dst.is_cuda:
        raise ValueError(f"dst must be a rank-1 device tensor of {n} elements")
    if dst.dtype != src.dtype:
        raise ValueError("src and dst must share one dtype")
    order = list(leaf_order or [])
    if len(order) > 32:
        raise ValueError("leaf_order has more than 32 bits")
    d = ReduceDesc(rows, cols, torch_dtype_code(src.dtype), REDUCE_KINDS[kind], axis,
                   int(bool(clear)), src.data_ptr(), ld, dst.data_ptr(), max(dst.stride(0), 1),
                   len(order), (ctypes.c_uint8 * 32)(*order), None, 0)
    ws = None
    if workspace is not False:
        need = load().frisk_reduce_workspace_size(ctypes.byref(d))
        _check(int(need) if need < 0 else OK, "frisk_reduce_workspace_size")
        if need > 0:
            ws = workspace if workspace is not True else _scratch(need, src.device, stream)
            d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
    _check(load().frisk_reduce(ctypes.byref(d), ctypes.c_void_p(_stream_handle(stream))),
           "frisk_reduce")
    return dst


def copy(src, dst, *, stream=None):
    """frisk.copy of a whole tile: dst = src converted to dst's dtype."""
    rows, cols, lds = _matrix(src, "src")
    drows, dcols, ldd = _matrix(dst, "dst")
    if (rows, cols) != (drows, dcols):
        raise ValueError(f"copy shapes differ: {tuple(src.shape)} -> {tuple(dst.shape)}")
    d = CopyDesc(rows, cols, torch_dtype_code(src.dtype), torch_dtype_code(dst.dtype),
                 src.data_ptr(), lds, dst.data_ptr(), ldd)
    _check(load().frisk_copy(ctypes.byref(d), ctypes.c_void_p(_stream_handle(stream))),
           "frisk_copy")
    return dst


def fill(dst, value, *, stream=None):
    """frisk.fill: every element of dst = value rounded to dst's dtype."""
    rows, cols, ld = _matrix(dst, "dst")
    d = FillDesc(rows, cols, torch_dtype_code(dst.dtype), float(value), dst.data_ptr(), ld)
    _check(load().frisk_fill(ctypes.byref(d), ctypes.c_void_p(_stream_handle(stream))),
           "frisk_fill")
    return dst


# ---- Rotary positions, the cache of keys and values, drafted trees -------------

ROPE_SCALINGS = {"none": 0, "linear": 1, "base": 2, "turns": 3, "index": 4}


def rope_table(rot_dim, base=10000.0, *, scaling="none", factor=1.0, trained=0.0, fast=32.0,
               slow=1.0, device="cuda"):
    """The int64 [rot_dim / 2] frequencies rope() takes, made once: turns per
    position in units of 2^-64.  `scaling` slows them down for contexts
    longer than the `trained` length (frisk_rope_scaling): "linear" by
    `factor`; "base" through the base; "turns" by `factor` where a pair turns
    at most `slow` times in the trained length, not where it turns `fast`
    times or more, evenly in turns between; "index" the same, evenly in the
    pair's index."""
    import torch
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r} ({', '.join(ROPE_SCALINGS)})")
    buf = (ctypes.c_uint64 * max(int(rot_dim) // 2, 1))()
    _check(load().frisk_rope_frequencies(int(rot_dim), float(base), ROPE_SCALINGS[scaling],
                                         float(factor), float(trained), float(fast), float(slow), buf),
           "frisk_rope_frequencies")
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in buf], dtype=torch.int64).to(device)


def rope_axes(sections, *, interleaved=False, device="cuda"):
    """The uint8 [rot_dim / 2] axes of pairs that rope() takes with positions of
    several axes: sections[a] pairs turn by axis a's position, axis after axis,
    or, if `interleaved`, in turn (an axis drops out when its pairs are dealt)."""
    import torch
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) < 1:
        raise ValueError(f"sections are the pairs of 1 to 4 axes (got {sections})")
    if interleaved:
        out = [a for i in range(max(sections)) for a, n in enumerate(sections) if i < n]
    else:
        out = [a for a, n in enumerate(sections) for _ in range(n)]
    return torch.tensor(out, dtype=torch.uint8).to(device)


# The calls below fill their descriptors with struct.pack, which takes a fifth
# of the time of a ctypes.Structure's fields (a decode step's launches are short).

def _packer(cls, until=None):
    """struct.Struct of a descriptor's fields, up to the field `until`, padded
    to its offset."""
    codes = {_i64: "q", _i32: "i", ctypes.c_float: "f", _ptr: "P"}
    fmt = "@"
    for name, kind in cls._fields_:
        if name == until:
            break
        fmt += codes[kind]
    end = getattr(cls, until).offset if until else ctypes.sizeof(cls)
    return struct.Struct(fmt + f"{end - struct.calcsize(fmt)}x")


_rope_pack = _packer(RopeDesc)
_kv_pack = _packer(KvDesc, "cache")
_tree_pack = _packer(TreeAttnDesc, "cache")
_compact_pack = _packer(KvCompactDesc, "cache")
_copy_pages_pack = _packer(KvCopyPagesDesc, "cache")
_pages_pack = _packer(KvPagesDesc)
_verify_pack = _packer(TreeVerifyDesc, "workspace")
_ws_pack = struct.Struct("@Pq")


_RANGE = (OverflowError, struct.error)


def _range_error(e) -> ValueError:
    return ValueError(f"argument out of range: {e}")


_raw: dict = {}


def _raw_fn(name: str):
    """The library's function `name` taking a packed descriptor."""
    fn = _raw.get(name)
    if fn is None:
        fn = load()[name]
        fn.restype = ctypes.c_int64 if name.endswith("_size") else ctypes.c_int
        fn.argtypes = [ctypes.c_char_p] + ([] if name.endswith("_size") else [ctypes.c_void_p])
        _raw[name] = fn
    return fn


def _heads(t, name: str):
    """Shape and strides of a [batch, heads, rows, head_dim] device tensor."""
    sh, st = t.shape, t.stride()
    if len(sh) != 4 or not t.is_cuda or (st[3] != 1 and sh[3] > 1):
        raise ValueError(f"{name} must be a rank-4 device tensor with unit head_dim stride")
    return sh, st


def _same_device(*ts) -> int:
    """The device index every tensor lies on, which the call runs on."""
    dev = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on different devices ({ts[0].device} and {t.device})")
    return dev


def _lengths(t, batch: int, name: str) -> int:
    """The pointer of an int32 [batch] device tensor, or 0."""
    if t is None:
        return 0
    import torch
    if t.dtype != torch.int32 or t.shape != (batch,) or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"{name} must be a contiguous int32 device tensor of {batch} elements")
    return t.data_ptr()


_accessors: list = []


def _current(dev: int, stream):
    """The handle of `stream` (None: the current one of device `dev`), or None
    if `dev` is not the current device."""
    if not _accessors:
        import torch
        # torch's raw accessors, without the Python layers of the public ones.
        _accessors[:] = [getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device),
                         getattr(torch._C, "_cuda_getCurrentRawStream", None)]
    device, raw = _accessors
    if dev != device():
        return None
    return raw(dev) if stream is None and raw is not None else _stream_handle(stream)


def _run(name: str, desc: bytes, dev: int, stream):
    """The library's `name` on a packed descriptor, with device `dev` current."""
    handle = _current(dev, stream)
    if handle is None:
        import torch
        with torch.cuda.device(dev):
            handle = _stream_handle(stream)
            rc = _raw_fn(name)(desc, handle)
    else:
        rc = _raw_fn(name)(desc, handle)
    if rc:
        _check(rc, name)


def rope(x, out, positions, table, *, k=None, k_out=None, start=None, pair_axis=None,
         interleaved=False, amplitude=1.0, backward=False, stream=None):
    """out = x [batch, heads, seq, head_dim] with its first 2 * len(table) dims
    rotated to their positions, and k_out = k (its own number of heads)
    likewise, in one launch.  out may be x.  `positions` (int32 or int64,
    [seq] or [batch, seq], or None: 0 .. seq - 1) are counted from `start`
    (int32 [batch], or None: 0).  With `pair_axis` (uint8 [len(table)],
    rope_axes) they have 1 to 4 axes, [axes, seq] or [axes, batch, seq], and
    pair i turns by that of axis pair_axis[i].  Pairs are dims (i, i +
    rot_dim / 2), or (2i, 2i + 1) if `interleaved`.  backward=True is the
    gradient: the transposed rotation."""
    import torch
    (b, h, s, d), xs = _heads(x, "x")
    osh, outs = _heads(out, "out")
    if osh != x.shape or out.dtype != x.dtype:
        raise ValueError("x and out must have one shape and dtype")
    if table.dtype != torch.int64 or table.dim() != 1 or not table.is_contiguous():
        raise ValueError("table must be a contiguous int64 device tensor (rope_table)")
    kh, second = 0, (0,) * 8
    if k is not None or k_out is not None:
        if k is None or k_out is None:
            raise ValueError("k and k_out go together")
        (kb, kh, ks_, kd), ks = _heads(k, "k")
        kosh, kos = _heads(k_out, "k_out")
        if (kb, ks_, kd) != (b, s, d) or kosh != k.shape or k.dtype != x.dtype or k_out.dtype != x.dtype:
            raise ValueError("k and k_out must have one shape, and x's dtype, batch, seq and head_dim")
        second = (k.data_ptr(), ks[0], ks[1], ks[2], k_out.data_ptr(), kos[0], kos[1], kos[2])
    at, axes = (0, 0, 0, 0), (0, 0, 0)
    if positions is not None:
        bits = 64 if positions.dtype == torch.int64 else 32
        shape, st = positions.shape, positions.stride()
        if pair_axis is not None:
            if pair_axis.dtype != torch.uint8 or pair_axis.shape != table.shape or \
                    not pair_axis.is_contiguous():
                raise ValueError(f"pair_axis must be a contiguous uint8 device tensor [{table.shape[0]}] (rope_axes)")
            if len(shape) not in (2, 3):
                raise ValueError("with pair_axis positions are [axes, seq] or [axes, batch, seq]")
            axes = (shape[0], st[0], pair_axis.data_ptr())
            shape, st = shape[1:], st[1:]
        if (bits == 32 and positions.dtype != torch.int32) or shape not in ((s,), (b, s)):
            raise ValueError("positions must be an int32 or int64 device tensor [seq] or [batch, seq]")
        at = (positions.data_ptr(), bits, *((0, st[0]) if len(st) == 1 else st))
    elif pair_axis is not None:
        raise ValueError("pair_axis needs positions")
    dev = _same_device(x, out, k, k_out, positions, table, start, pair_axis)
    start = _lengths(start, b, "start")
    try:
        desc = _rope_pack.pack(b, s, h, kh, d, 2 * table.shape[0], torch_dtype_code(x.dtype),
                               bool(interleaved), bool(backward), amplitude,
                               x.data_ptr(), xs[0], xs[1], xs[2], out.data_ptr(), outs[0], outs[1], outs[2],
                               *second, *at, start, table.data_ptr(), *axes)
    except _RANGE as e:
        raise _range_error(e) from None
    _run("frisk_rope", desc, dev, stream)
    return out if k is None else (out, k_out)


class KvCache:
    """A cache of keys and values (frisk_kv_cache) over tensors the caller
    owns: k and v [pages, kv_heads, page_size, head_dim] of one layout, in
    bf16 / f16, or in float8_e4m3fn / int8 with f32 k_scale and v_scale
    [pages, kv_heads, page_size].  With `scale_block` (a power of two, 2 to
    256) that many slots share a scale, and the scales are [pages, kv_heads,
    ceil(page_size / scale_block)].  `block_table` (int32 [batch, max_pages])
    names the pages of each sequence; without it page b is sequence b's."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "block_table", "scale_block", "desc", "_packed", "_device")

    def __init__(self, k, v, k_scale=None, v_scale=None, block_table=None, *, scale_block=1):
        import torch
        ksh, kst = _heads(k, "k")
        vsh, vst = _heads(v, "v")
        if tuple(ksh) != tuple(vsh) or tuple(kst) != tuple(vst) or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape, layout and dtype")
        if k.dtype not in (torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8):
            raise ValueError(f"a cache holds bf16, f16, float8_e4m3fn or int8 (got {k.dtype})")
        if (k_scale is None) != (k.element_size() == 2) or (v_scale is None) != (k_scale is None):
            raise ValueError("an 8-bit cache has k_scale and v_scale, a 16-bit one none")
        sst = (0, 0, 0)
        self._check_block(scale_block, k.element_size())
        if k_scale is not None:
            shape = (ksh[0], ksh[1], -(-ksh[2] // scale_block))
            for t in (k_scale, v_scale):
                if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_cuda:
                    raise ValueError(f"scales must be f32 device tensors {list(shape)}: [pages, kv_heads, "
                                     f"page_size], or one for scale_block slots")
            sst = k_scale.stride()
            if v_scale.stride() != sst:
                raise ValueError("k_scale and v_scale must have one layout")
        if block_table is not None and (block_table.dtype != torch.int32 or block_table.dim() != 2 or
                                        not block_table.is_cuda or
                                        (block_table.stride(1) != 1 and block_table.shape[1] > 1)):
            raise ValueError("block_table must be an int32 device tensor [batch, max_pages] with unit "
                             "stride along the pages")
        self._device = _same_device(k, v, k_scale, v_scale, block_table)
        self.k, self.v, self.k_scale, self.v_scale, self.block_table = k, v, k_scale, v_scale, block_table
        self.scale_block = scale_block
        self.desc = KvCacheDesc(
            *ksh, torch_dtype_code(k.dtype), k.data_ptr(), v.data_ptr(), *kst[:3],
            None if k_scale is None else k_scale.data_ptr(),
            None if v_scale is None else v_scale.data_ptr(), *sst,
            None if block_table is None else block_table.data_ptr(),
            0 if block_table is None else block_table.stride(0),
            0 if block_table is None else block_table.shape[1], scale_block)
        self._packed = bytes(self.desc)

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, dtype, *, block_table=None, scale_block=1,
              device="cuda"):
        """A cache over new tensors (their contents undefined until written)."""
        import torch
        cls._check_block(scale_block, dtype.itemsize)
        shape = (pages, kv_heads, page_size, head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        ks = vs = None
        if k.element_size() == 1:
            scales = (pages, kv_heads, -(-page_size // scale_block))
            ks, vs = (torch.empty(scales, dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs, block_table, scale_block=scale_block)

    @staticmethod
    def _check_block(scale_block, bytes_):
        if scale_block < 1 or (scale_block > 1 and bytes_ != 1):
            raise ValueError(f"scale_block must be 1 or more, and is for 8-bit caches (got {scale_block})")

    def __setattr__(self, name, value):
        # The calls take the descriptor that __init__ packed.
        if hasattr(self, "_packed"):
            raise AttributeError("a KvCache's tensors are fixed: write into them, or make another one")
        object.__setattr__(self, name, value)

    def _check(self, batch: int, *ts) -> int:
        """The device of the cache and `ts`, for a batch that fits the block table."""
        if self.block_table is not None and self.block_table.shape[0] != batch:
            raise ValueError(f"block_table has {self.block_table.shape[0]} rows for a batch of {batch}")
        return _same_device(self.k, *ts)


def _kv(name, k, v, cache, ctx_len, new_len, stream):
    (b, h, t, d), ks = _heads(k, "k")
    vsh, vs = _heads(v, "v")
    csh = cache.k.shape
    if vsh != k.shape or v.dtype != k.dtype or h != csh[1] or d != csh[3]:
        raise ValueError(f"k and v must be [batch, {csh[1]}, tokens, {csh[3]}] of one dtype "
                         f"(got {tuple(k.shape)} and {tuple(v.shape)})")
    dev = cache._check(b, k, v, ctx_len, new_len)
    ctx, new = _lengths(ctx_len, b, "ctx_len"), _lengths(new_len, b, "new_len")
    try:
        desc = _kv_pack.pack(b, t, torch_dtype_code(k.dtype), k.data_ptr(), ks[0], ks[1], ks[2],
                             v.data_ptr(), vs[0], vs[1], vs[2], ctx, new)
    except _RANGE as e:
        raise _range_error(e) from None
    _run(name, desc + cache._packed, dev, stream)


def kv_append(k, v, cache, ctx_len, *, new_len=None, stream=None):
    """Write k and v [batch, kv_heads, tokens, head_dim] (bf16 or f16) into the
    KvCache as keys ctx_len[b] .. of each sequence (int32 [batch] on the
    device; negative: the sequence takes no part), the first new_len[b]
    tokens of it.  An 8-bit cache quantises each row by its largest value, or
    a block's rows by theirs: a block's scale grows with its rows, and the codes
    before them follow (frisk_kv_append).  Both stay when the rows are drafts that
    are rejected, and so does NaN; a block appended from its first slot is made anew."""
    _kv("frisk_kv_append", k, v, cache, ctx_len, new_len, stream)
    return cache


def kv_read(cache, k, v, ctx_len, *, new_len=None, stream=None):
    """Read keys ctx_len[b] .. of each sequence back into k and v [batch,
    kv_heads, tokens, head_dim], the first new_len[b] rows of it; the other
    rows are left as they were."""
    _kv("frisk_kv_read", k, v, cache, ctx_len, new_len, stream)
    return k, v


def kv_compact(cache, path, ctx_len, count, *, stream=None):
    """Move the rows of an accepted branch behind its context: key ctx_len[b] + i
    becomes the one that was ctx_len[b] + path[b, i], for i < count[b] (path
    int32 [batch, tokens] and count int32 [batch] of tree_verify, on the device;
    ctx_len negative: the sequence takes no part).  Not for a cache with
    scale_block, whose rows are appended again instead."""
    import torch
    shape, st = path.shape, path.stride()
    if path.dtype != torch.int32 or len(shape) != 2 or not path.is_cuda or (st[1] != 1 and shape[1] > 1):
        raise ValueError("path must be an int32 device tensor [batch, tokens] with unit stride along the tokens")
    b, t = shape
    dev = cache._check(b, path, ctx_len, count)
    desc = _compact_pack.pack(b, t, path.data_ptr(), st[0] if b > 1 else t,
                              _lengths(ctx_len, b, "ctx_len"), _lengths(count, b, "count"))
    _run("frisk_kv_compact", desc + cache._packed, dev, stream)
    return cache


def kv_copy_pages(cache, src, dst, *, rows=None, stream=None):
    """Copy pages src[i] of the cache to pages dst[i] (int32 [pairs] on the device;
    a pair with a page outside the cache is left out), the first rows[i] slots
    of them (None: all).  No page is copied to twice, or copied to and from."""
    n = src.shape[0] if src.dim() == 1 else 0
    dev = _same_device(cache.k, src, dst, rows)
    desc = _copy_pages_pack.pack(n, _lengths(src, n, "src"), _lengths(dst, n, "dst"), _lengths(rows, n, "rows"))
    _run("frisk_kv_copy_pages", desc + cache._packed, dev, stream)
    return cache


def kv_pages(table, keep, want, page_size, pages, *, parent=None, held=None, out=None, src=None, dst=None,
             rows=None, lacking=None, stream=None):
    """(out, src, dst, rows, lacking): the block table of the next step, from `table`
    (int32 [batch, max_pages]) of a cache of `pages` pages.  Row b takes over the pages of the first
    keep[b] keys of row parent[b] (None: its own; outside the batch: sequence b has ended, and its
    pages are free) and has room for want[b] keys (None: keep[b]).  keep[b] is a length of the
    parent's row, not of b's own: a program that keeps all of it passes ctx_len[parent[b]], which
    is b's length from then on.  Sequences share whole pages; one that would write a shared page
    gets a copy of it: page dst[b] of src[b], the first rows[b] slots (-1, -1, 0: none), which
    kv_copy_pages makes in every layer's cache.  New pages are the lowest-numbered ones that no row has and that
    `held` (uint8 or bool [pages]) does not keep back; lacking[0] counts the entries
    that are -1 because there were too few.  keep, want, parent, src, dst, rows: int32
    [batch]; lacking: int32 [1].  `out` must be another tensor than `table`; a program with one table
    copies it back."""
    import torch
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_cuda or \
            (table.stride(1) != 1 and table.shape[1] > 1):
        raise ValueError("table must be an int32 device tensor [batch, max_pages] with unit stride along the pages")
    b, n = table.shape
    if out is None:
        out = _empty((b, n), torch.int32, table.device, stream)
    elif out.dtype != torch.int32 or out.shape != table.shape or (out.stride(1) != 1 and n > 1):
        raise ValueError(f"out must be an int32 tensor [{b}, {n}] with unit stride along the pages")
    if held is not None and (held.dtype not in (torch.uint8, torch.bool) or held.shape != (pages,) or
                             not held.is_contiguous()):
        raise ValueError(f"held must be a contiguous uint8 or bool device tensor [{pages}]")
    src, dst, rows = (_empty((b,), torch.int32, table.device, stream) if x is None else x
                      for x in (src, dst, rows))
    if lacking is None:
        lacking = _empty((1,), torch.int32, table.device, stream)
    dev = _same_device(table, out, keep, want, parent, held, src, dst, rows, lacking)
    try:
        desc = _pages_pack.pack(
            b, n, pages, page_size, table.data_ptr(), table.stride(0) if b > 1 else n, out.data_ptr(),
            out.stride(0) if b > 1 else n, _lengths(parent, b, "parent"), _lengths(keep, b, "keep"),
            _lengths(want, b, "want"), 0 if held is None else held.data_ptr(), _lengths(src, b, "src"),
            _lengths(dst, b, "dst"), _lengths(rows, b, "rows"), _lengths(lacking, 1, "lacking"))
    except _RANGE as e:
        raise _range_error(e) from None
    _run("frisk_kv_pages", desc, dev, stream)
    return out, src, dst, rows, lacking


def tree_mask(parents, mask=None, depth=None, *, stream=None):
    """(mask, depth) of drafted trees: parents int32 [batch, tokens] (the
    drafted token each one continues, -1: the context) to the int64 words
    [batch, tokens, ceil(tokens / 64)] that tree_attn takes, and the int32
    number of drafted tokens before each ([batch, tokens]; its position is
    ctx_len + depth).  Tensors it makes are of the call's stream."""
    import torch
    if parents.dtype != torch.int32 or parents.dim() != 2 or not parents.is_contiguous() or \
            not parents.is_cuda:
        raise ValueError("parents must be a contiguous int32 device tensor [batch, tokens]")
    b, t = parents.shape
    words = (t + 63) // 64
    if mask is None:
        mask = _empty((b, t, words), torch.int64, parents.device, stream)
    elif mask.dtype != torch.int64 or mask.shape != (b, t, words) or not mask.is_contiguous():
        raise ValueError(f"mask must be a contiguous int64 tensor [{b}, {t}, {words}]")
    if depth is None:
        depth = _empty((b, t), torch.int32, parents.device, stream)
    elif depth.dtype != torch.int32 or depth.shape != (b, t) or not depth.is_contiguous():
        raise ValueError(f"depth must be a contiguous int32 tensor [{b}, {t}]")
    dev = _same_device(parents, mask, depth)
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return tree_mask(parents, mask, depth, stream=stream)
    _check(load().frisk_tree_mask(b, t, parents.data_ptr(), mask.data_ptr(), depth.data_ptr(),
                                  _stream_handle(stream)), "frisk_tree_mask")
    return mask, depth


def _tree_values(q, cache, ctx_len, o, mask, new_len, sm_scale, lse, max_ctx):
    """Device and the fields of TreeAttnDesc before its cache."""
    import torch
    (b, h, t, d), qs = _heads(q, "q")
    osh, os_ = _heads(o, "o")
    if osh != q.shape or d != cache.k.shape[3]:
        raise ValueError(f"q and o must have one shape and the cache's head_dim {cache.k.shape[3]} "
                         f"(got {tuple(q.shape)} and {tuple(o.shape)})")
    if lse is not None and (lse.shape != (b, h, t) or not lse.is_contiguous()
                            or lse.dtype != torch.float32):
        raise ValueError("lse must be a contiguous f32 [batch, heads, tokens] tensor")
    words = (0, 0, 0)
    if mask is not None:
        n = (t + 63) // 64
        if mask.dtype != torch.int64 or mask.shape not in ((t, n), (b, t, n)) or \
                (mask.stride(-1) != 1 and n > 1):
            raise ValueError(f"mask must be int64 words [{t}, {n}] or [{b}, {t}, {n}] (tree_mask)")
        st = mask.stride()
        words = (mask.data_ptr(), *((0, st[0]) if len(st) == 2 else st[:2]))
    dev = cache._check(b, q, o, ctx_len, new_len, mask, lse)
    return dev, (b, h, t, torch_dtype_code(q.dtype), torch_dtype_code(o.dtype),
                 d ** -0.5 if sm_scale is None else sm_scale,
                 q.data_ptr(), qs[0], qs[1], qs[2], o.data_ptr(), os_[0], os_[1], os_[2],
                 0 if lse is None else lse.data_ptr(), _lengths(ctx_len, b, "ctx_len"),
                 _lengths(new_len, b, "new_len"), *words, max_ctx)


def tree_attn_desc(q, cache, ctx_len, o, *, mask=None, new_len=None, sm_scale=None, lse=None,
                   max_ctx=0) -> TreeAttnDesc:
    """Describe tree_attn's call (without a workspace)."""
    _, values = _tree_values(q, cache, ctx_len, o, mask, new_len, sm_scale, lse, max_ctx)
    return TreeAttnDesc(*values, cache.desc)


def tree_attn_workspace_bytes(desc: TreeAttnDesc) -> int:
    """frisk_tree_attn_workspace_size for a descriptor."""
    need = int(load().frisk_tree_attn_workspace_size(ctypes.byref(desc)))
    _check(need if need < 0 else OK, "frisk_tree_attn_workspace_size")
    return need


def tree_attn(q, cache, ctx_len, o, *, mask=None, new_len=None, sm_scale=None, lse=None, max_ctx=0,
              workspace=True, stream=None):
    """o = softmax(sm_scale . q K^T) V of new tokens q [batch, heads, tokens,
    head_dim] over a KvCache that holds them (kv_append) behind the ctx_len[b]
    keys every token sees.  Among themselves token t sees draft j where bit j
    of mask[b][t] is set (tree_mask; [tokens, words] for one tree of all
    sequences), without a mask where j <= t; tokens from new_len[b] on are
    left out.  `max_ctx` hints at the largest ctx_len (0: the capacity).
    `workspace`: True allocates the scratch of the key splits (torch's
    caching allocator, on the call's stream), a device tensor supplies it,
    False runs unsplit."""
    dev, values = _tree_values(q, cache, ctx_len, o, mask, new_len, sm_scale, lse, max_ctx)
    handle = _current(dev, stream)
    if handle is None:
        import torch
        with torch.cuda.device(dev):
            return tree_attn(q, cache, ctx_len, o, mask=mask, new_len=new_len, sm_scale=sm_scale,
                             lse=lse, max_ctx=max_ctx, workspace=workspace, stream=stream)
    try:
        head = _tree_pack.pack(*values) + cache._packed
    except _RANGE as e:
        raise _range_error(e) from None
    ws, tail = None, bytes(16)
    if workspace is not False:
        need = _raw_fn("frisk_tree_attn_workspace_size")(head + tail)
        if need < 0:
            _check(need, "frisk_tree_attn_workspace_size")
        if need > 0:
            ws = workspace if workspace is not True else _scratch(need, o.device, stream)
            if ws.get_device() != dev or not ws.is_contiguous():
                raise ValueError("workspace must be a contiguous tensor on q's device")
            tail = _ws_pack.pack(ws.data_ptr(), ws.numel() * ws.element_size())
    rc = _raw_fn("frisk_tree_attn")(head + tail, handle)
    if rc:
        _check(rc, "frisk_tree_attn")
    return o


def _words(t, shape, dtype, name: str) -> int:
    """The pointer of a contiguous tensor of that shape and dtype, or 0."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} device tensor {list(shape)}")
    return t.data_ptr()


def _vocab(t, shape, name: str):
    """Strides of a [batch, tokens, vocab] device tensor."""
    st = t.stride()
    if t.shape != shape or not t.is_cuda or (st[2] != 1 and shape[2] > 1):
        raise ValueError(f"{name} must be a device tensor {list(shape)} with unit stride along the vocabulary")
    return st


def tree_verify(logits, drafts, parents, uniform, final, *, draft_probs=None, temperature=None, new_len=None,
                path=None, count=None, token=None, probs=None, workspace=True, stream=None):
    """(path, count, token): which drafted tokens of each tree the target accepts, and
    the token after them.  Node 0 of a tree is the last token that is decided, node
    t the draft drafts[b, t] (int32 [batch, tokens]) that continues node parents[b, t] (int32,
    tree_mask's); logits [batch, tokens, vocab] (f32, f16 or bf16) are the target's behind
    each node, at `temperature` (f32 [batch], None: 1, 0: the largest logit).  uniform
    (f32 [batch, tokens]) decides about each draft, final (f32 [batch]) draws the last
    token; both are of [0, 1).  draft_probs (f32 [batch, tokens, vocab]): row n holds the
    probabilities that node n's children were drawn from, independently (with replacement:
    else tokens are not distributed as the target's); None: drafts are certain
    ones.  With one node a tree this samples from its logits.
    path (int32 [batch, tokens]) lists the accepted nodes from 0 on, then -1, count (int32 [batch])
    their number, token (int32 [batch]) is -1 where logits hold a NaN or +infinity; probs (f32 [batch, tokens],
    optional) takes the target's probability of each draft.  Trees have new_len[b]
    nodes (int32 [batch], None: all; 0: left as they were, -1, 0 and -1 in tensors that
    the call makes).  Frees no page and moves no row: kv_compact and kv_pages do.
    `workspace`: True allocates it (torch's caching allocator, on the call's
    stream), a device tensor of tree_verify_workspace_bytes supplies it, False or None
    is for calls that take none."""
    import torch
    if logits.dim() != 3:
        raise ValueError("logits must be a device tensor [batch, tokens, vocab]")
    b, t, v = shape = logits.shape
    ls = _vocab(logits, shape, "logits")
    qs = (0, 0)
    if draft_probs is not None:
        if draft_probs.dtype != torch.float32:
            raise ValueError("draft_probs must be f32")
        qs = _vocab(draft_probs, shape, "draft_probs")
    handle = _current(logits.get_device(), stream)
    if handle is None:
        with torch.cuda.device(logits.get_device()):
            return tree_verify(logits, drafts, parents, uniform, final, draft_probs=draft_probs,
                               temperature=temperature, new_len=new_len, path=path, count=count, token=token,
                               probs=probs, workspace=workspace, stream=stream)
    absent = new_len is not None  # trees of no nodes: nothing is written for them
    if path is None:
        path = _empty((b, t), torch.int32, logits.device, stream, -1 if absent else None)
    if count is None:
        count = _empty((b,), torch.int32, logits.device, stream, 0 if absent else None)
    if token is None:
        token = _empty((b,), torch.int32, logits.device, stream, -1 if absent else None)
    dev = _same_device(logits, drafts, parents, uniform, final, draft_probs, temperature, new_len, path, count,
                       token, probs)
    i32, f32, one, all_ = torch.int32, torch.float32, shape[:1], shape[:2]
    try:
        head = _verify_pack.pack(
            b, t, v, torch_dtype_code(logits.dtype), logits.data_ptr(), ls[0], ls[1],
            _words(drafts, all_, i32, "drafts"), _words(parents, all_, i32, "parents"),
            _words(uniform, all_, f32, "uniform"), _words(final, one, f32, "final"),
            0 if draft_probs is None else draft_probs.data_ptr(), qs[0], qs[1],
            _words(temperature, one, f32, "temperature"), _words(new_len, one, i32, "new_len"),
            _words(path, all_, i32, "path"), _words(count, one, i32, "count"),
            _words(token, one, i32, "token"), _words(probs, all_, f32, "probs"))
    except _RANGE as e:
        raise _range_error(e) from None
    tail = bytes(16)
    if workspace is True:
        need = _raw_fn("frisk_tree_verify_workspace_size")(head + bytes(16))
        if need < 0:
            _check(need, "frisk_tree_verify_workspace_size")
        if need:
            workspace = _scratch(need, logits.device, stream)
            tail = _ws_pack.pack(workspace.data_ptr(), need)
    elif workspace is False or workspace is None:
        pass
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor on the logits' device")
    else:
        tail = _ws_pack.pack(workspace.data_ptr(), workspace.numel() * workspace.element_size())
    rc = _raw_fn("frisk_tree_verify")(head + tail, handle)
    if rc:
        _check(rc, "frisk_tree_verify")
    return path, count, token


def tree_verify_workspace_bytes(batch: int, tokens: int, vocab: int, dtype) -> int:
    """Bytes of workspace that tree_verify takes for logits [batch, tokens, vocab] of a torch dtype."""
    d = TreeVerifyDesc(batch=batch, tokens=tokens, vocab=vocab, dtype=torch_dtype_code(dtype))
    need = int(load().frisk_tree_verify_workspace_size(ctypes.byref(d)))
    _check(need if need < 0 else OK, "frisk_tree_verify_workspace_size")
    return need
