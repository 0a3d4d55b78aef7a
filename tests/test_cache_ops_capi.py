"""Refusals of the rotary, cache and tree entries, before any device work (no
GPU needed), and the frequencies, which are made on the host."""
import ctypes
import math

import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import cache_ops as C


def cache_desc(**over):
    d = dict(pages=8, kv_heads=2, page_size=16, head_dim=64, dtype=rt.BF16, k=4096, v=8192,
             stride_page=2048, stride_head=1024, stride_slot=64, k_scale=None, v_scale=None,
             scale_stride_page=32, scale_stride_head=16, scale_stride_slot=1, block_table=64,
             table_stride=4, max_pages=4)
    d.update(over)
    return rt.KvCacheDesc(**d)


def kv_call(name, cache=None, **over):
    d = dict(batch=2, tokens=3, dtype=rt.BF16, k=16, k_stride_b=384, k_stride_h=192, k_stride_s=64,
             v=1 << 16, v_stride_b=384, v_stride_h=192, v_stride_s=64, ctx_len=64, new_len=None)
    d.update(over)
    desc = rt.KvDesc(**d, cache=cache_desc(**(cache or {})))
    lib = rt.load()
    rc = getattr(lib, name)(ctypes.byref(desc), None)
    return rc, lib.frisk_last_error().decode()


CACHE_REFUSALS = [
    (dict(pages=0), rt.EINVAL, "cache sizes"), (dict(dtype=rt.F32), rt.EINVAL, "cache dtype"),
    (dict(head_dim=72), rt.EUNSUP, "head_dim"), (dict(head_dim=272, stride_slot=272), rt.EUNSUP, "head_dim"),
    (dict(stride_slot=60), rt.EINVAL, "cache strides"), (dict(stride_slot=32), rt.EINVAL, "cache strides"),
    (dict(stride_page=-2048), rt.EINVAL, "cache strides"), (dict(stride_page=1 << 41), rt.EINVAL, "cache strides"),
    (dict(k=0), rt.EINVAL, "null cache"), (dict(v=8), rt.EINVAL, "the cache must be 16-byte"),
    (dict(k_scale=64), rt.EINVAL, "scales are for 8-bit"),
    (dict(page_size=24), rt.EUNSUP, "pages of a block table"),
    (dict(max_pages=0), rt.EINVAL, "block_table needs"), (dict(table_stride=3), rt.EINVAL, "block_table needs"),
    (dict(max_pages=1 << 28, table_stride=1 << 28), rt.EUNSUP, "a sequence of more"),
    (dict(block_table=0, pages=1), rt.EINVAL, "without a block table"),
    (dict(block_table=2), rt.EINVAL, "scales and block_table"),
    (dict(page_size=1 << 31), rt.EUNSUP, "cache sizes beyond"),
    (dict(dtype=rt.E4M3), rt.EINVAL, "an 8-bit cache needs"),
    (dict(dtype=rt.I8, k_scale=64, v_scale=64, scale_stride_slot=0), rt.EINVAL, "scale strides"),
]


@pytest.mark.parametrize("name", ["frisk_kv_append", "frisk_kv_read"])
@pytest.mark.parametrize("cache,code,msg", CACHE_REFUSALS)
def test_cache_refusals(name, cache, code, msg):
    rc, err = kv_call(name, cache)
    assert rc == code and err.startswith(f"{name}: {msg}"), err


@pytest.mark.parametrize("name", ["frisk_kv_append", "frisk_kv_read"])
@pytest.mark.parametrize("over,code,msg", [
    (dict(batch=0), rt.EINVAL, "sizes must"), (dict(tokens=-1), rt.EINVAL, "sizes must"),
    (dict(dtype=rt.F32), rt.EINVAL, "dtype must"), (dict(dtype=rt.F16), rt.EINVAL, "a bf16 cache"),
    (dict(k=0), rt.EINVAL, "null tensor"), (dict(ctx_len=None), rt.EINVAL, "null tensor"),
    (dict(v=8), rt.EINVAL, "k and v must be 16-byte"), (dict(k_stride_s=60), rt.EINVAL, "strides must"),
    (dict(new_len=2), rt.EINVAL, "ctx_len and new_len")])
def test_kv_refusals(name, over, code, msg):
    rc, err = kv_call(name, **over)
    assert rc == code and err.startswith(f"{name}: {msg}"), err


def test_read_refuses_rows_that_overlap():
    rc, err = kv_call("frisk_kv_read", k_stride_s=0)
    assert rc == rt.EINVAL and "overlap" in err
    for at in (16, 16 + 128, 16 + 2 * 383):  # v among k's rows
        rc, err = kv_call("frisk_kv_read", v=at & ~15)
        assert rc == rt.EINVAL and "k and v overlap" in err


def test_append_refuses_one_tensor_for_both():
    rc, err = kv_call("frisk_kv_append", cache=dict(v=4096))
    assert rc == rt.EINVAL and "must be two tensors" in err


def test_append_refuses_a_cache_that_meets_itself():
    # k and v a page apart in one buffer of 8, and two slots of one scale.
    rc, err = kv_call("frisk_kv_append", cache=dict(v=4096 + 2 * 2048))
    assert rc == rt.EINVAL and "the cache's k and v must be two tensors" in err
    codes = dict(dtype=rt.I8, v=1 << 20, k_scale=1 << 21)
    rc, err = kv_call("frisk_kv_append", cache=dict(codes, v_scale=(1 << 21) + 4))
    assert rc == rt.EINVAL and "k_scale and v_scale must be two tensors" in err
    for over in (dict(stride_head=64), dict(stride_page=1024 + 15 * 64), dict(dtype=rt.I8, scale_stride_head=15)):
        rc, err = kv_call("frisk_kv_append", cache=dict(codes, v_scale=1 << 22, **over) if "dtype" in over else over)
        assert rc == rt.EINVAL and "the cache's rows or scales overlap" in err, err


def test_a_cache_keeps_its_tensors():
    c = rt.KvCache.__new__(rt.KvCache)
    c.k = 1
    c._packed = b""
    with pytest.raises(AttributeError, match="fixed"):
        c.block_table = None


def tree_call(cache=None, fn="frisk_tree_attn", **over):
    d = dict(batch=2, heads=4, tokens=3, dtype=rt.BF16, o_dtype=rt.BF16, sm_scale=0.125,
             q=16, q_stride_b=768, q_stride_h=192, q_stride_s=64, o=16, o_stride_b=768,
             o_stride_h=192, o_stride_s=64, lse=None, ctx_len=64, new_len=None, mask=None)
    d.update(over)
    desc = rt.TreeAttnDesc(**d, cache=cache_desc(**(cache or {})))
    lib = rt.load()
    rc = getattr(lib, fn)(*([ctypes.byref(desc)] + ([None] if fn == "frisk_tree_attn" else [])))
    return rc, lib.frisk_last_error().decode()


@pytest.mark.parametrize("cache,code,msg", CACHE_REFUSALS)
def test_tree_cache_refusals(cache, code, msg):
    rc, err = tree_call(cache)
    assert rc == code and err.startswith(f"frisk_tree_attn: {msg}"), err


@pytest.mark.parametrize("over,code,msg", [
    (dict(tokens=0), rt.EINVAL, "sizes must"), (dict(heads=3), rt.EINVAL, "heads 3"),
    (dict(dtype=rt.F32), rt.EINVAL, "dtype must"), (dict(o_dtype=rt.F16), rt.EINVAL, "o_dtype"),
    (dict(dtype=rt.F16, o_dtype=rt.F16), rt.EINVAL, "a bf16 cache needs q"),
    (dict(tokens=1 << 23), rt.EUNSUP, "more than 2^24"), (dict(batch=1 << 30), rt.EUNSUP, "more than 2^24"),
    (dict(q=0), rt.EINVAL, "null tensor"), (dict(ctx_len=None), rt.EINVAL, "null tensor"),
    (dict(o=8), rt.EINVAL, "q and o must be 16-byte"), (dict(q_stride_h=4), rt.EINVAL, "strides must"),
    (dict(o_stride_s=0), rt.EINVAL, "the rows of o"), (dict(mask=4), rt.EINVAL, "lengths and lse"),
    (dict(mask=8, mask_stride_t=-1), rt.EINVAL, "mask strides"),
    (dict(sm_scale=0.0), rt.EINVAL, "sm_scale"), (dict(sm_scale=math.inf), rt.EINVAL, "sm_scale"),
    (dict(max_ctx=-1), rt.EINVAL, "negative max_ctx"), (dict(workspace_bytes=-1), rt.EINVAL, "negative workspace")])
def test_tree_refusals(over, code, msg):
    rc, err = tree_call(**over)
    assert rc == code and err.startswith(f"frisk_tree_attn: {msg}"), err


@pytest.mark.parametrize("over", [
    dict(o=16 + 128), dict(o=16 + 16), dict(o_stride_s=256, o_stride_h=64), dict(o_dtype=rt.F32),
    dict(o=16 + 2 * 1000, o_dtype=rt.F32), dict(o=16 + 2 * 1528)])
def test_tree_refuses_an_output_among_the_queries(over):
    rc, err = tree_call(**over)
    assert rc == rt.EINVAL and "q and o overlap" in err, err


def test_tree_output_rows_and_hints_of_any_size():
    rc, err = tree_call(o=1 << 20, o_stride_h=128)  # the heads of a token inside the next one's
    assert rc == rt.EINVAL and "the rows of o overlap" in err
    big = dict(block_table=64, max_pages=1 << 16, table_stride=1 << 16)
    size = "frisk_tree_attn_workspace_size"
    assert tree_call(big, size, max_ctx=(1 << 63) - 1)[0] == tree_call(big, size)[0] > 0


def test_tree_workspace():
    big = dict(block_table=64, max_pages=1 << 16, table_stride=1 << 16)
    need, _ = tree_call(big, "frisk_tree_attn_workspace_size", q=None, o=None, ctx_len=None)
    assert need > 0
    rc, err = tree_call(big, workspace=16, workspace_bytes=need - 1)
    assert rc == rt.EINVAL and "workspace of" in err
    rc, err = tree_call(big, workspace=24, workspace_bytes=need)
    assert rc == rt.EINVAL and "workspace must be 16-byte" in err
    assert tree_call(big, "frisk_tree_attn_workspace_size", max_ctx=1)[0] == 0


@pytest.mark.parametrize("args,code,msg", [
    ((0, 4, 64, 64), rt.EINVAL, "sizes"), ((1, 4097, 64, 64), rt.EUNSUP, "up to 4096"),
    ((1 << 24, 4, 64, 64), rt.EUNSUP, "up to 4096"), ((1, 4, None, 64), rt.EINVAL, "null"),
    ((1, 4, 64, 60), rt.EINVAL, "pointers")])
def test_tree_mask_refusals(args, code, msg):
    lib = rt.load()
    rc = lib.frisk_tree_mask(*args, None, None)
    assert rc == code and lib.frisk_last_error().decode().startswith(f"frisk_tree_mask: {msg}")


def rope_call(**over):
    d = dict(batch=2, seq=3, heads=4, k_heads=0, head_dim=64, rot_dim=64, dtype=rt.BF16, interleaved=0,
             backward=0, amplitude=1.0, x=1 << 20, x_stride_b=768, x_stride_h=64, x_stride_s=256,
             out=1 << 21, out_stride_b=768, out_stride_h=64, out_stride_s=256, positions=64,
             position_bits=32, pos_stride_b=0, pos_stride_s=1, start=None, frequencies=64)
    d.update(over)
    lib = rt.load()
    rc = lib.frisk_rope(ctypes.byref(rt.RopeDesc(**d)), None)
    return rc, lib.frisk_last_error().decode()


KT = dict(k_heads=2, k_stride_b=768, k_stride_h=64, k_stride_s=256, k_out_stride_b=768,
          k_out_stride_h=64, k_out_stride_s=256)


@pytest.mark.parametrize("over,code,msg", [
    (dict(seq=0), rt.EINVAL, "sizes must"), (dict(dtype=rt.I8), rt.EINVAL, "dtype must"),
    (dict(rot_dim=63), rt.EINVAL, "rot_dim"), (dict(rot_dim=66), rt.EINVAL, "rot_dim"),
    (dict(interleaved=2), rt.EINVAL, "interleaved"), (dict(amplitude=math.nan), rt.EINVAL, "amplitude"),
    (dict(frequencies=None), rt.EINVAL, "frequencies"), (dict(position_bits=16), rt.EINVAL, "position_bits"),
    (dict(positions=66), rt.EINVAL, "positions"), (dict(start=2), rt.EINVAL, "start"),
    (dict(pos_stride_s=-1), rt.EINVAL, "position strides"), (dict(x=0), rt.EINVAL, "null x"),
    (dict(x=(1 << 20) + 1), rt.EINVAL, "pointers"), (dict(x_stride_b=-1), rt.EINVAL, "strides"),
    (dict(out_stride_h=32), rt.EINVAL, "the rows of x's output"),
    (dict(head_dim=8192, x_stride_h=8192, out_stride_h=8192, out_stride_s=32768, out_stride_b=98304),
     rt.EUNSUP, "sizes beyond"),
    (dict(out=(1 << 20) + 2), rt.EINVAL, "x and its output overlap"),
    (dict(out=(1 << 20) + 128), rt.EINVAL, "x and its output overlap"),
    (dict(out=1 << 20, out_stride_s=512, out_stride_b=1536), rt.EINVAL, "x and its output overlap"),
    (dict(k=1 << 22, k_out=(1 << 22) + 128, **KT), rt.EINVAL, "k and its output overlap"),
    (dict(k=1 << 22, k_out=1 << 21, **KT), rt.EINVAL, "the output of x or k"),
    (dict(k=1 << 21, k_out=1 << 22, **KT), rt.EINVAL, "the output of x or k")])
def test_rope_refusals(over, code, msg):
    rc, err = rope_call(**over)
    assert rc == code and err.startswith(f"frisk_rope: {msg}"), err


def freqs(rot, base=10000.0, **kw):
    return [int(v) % 2 ** 64 * 2.0 ** -64 * 2 * math.pi for v in rt.rope_table(rot, base, device="cpu", **kw)]


def test_frequencies():
    plain = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert np.allclose(freqs(64), plain, rtol=1e-14)
    assert np.allclose(freqs(64, scaling="linear", factor=4.0), np.array(plain) / 4, rtol=1e-14)
    base = 10000.0 * 8.0 ** (64 / 62)
    assert np.allclose(freqs(64, scaling="base", factor=8.0), [base ** (-2 * i / 64) for i in range(32)], rtol=1e-14)
    got = freqs(64, scaling="turns", factor=8.0, trained=8192, fast=4.0, slow=1.0)
    for f, g in zip(plain, got):
        turns = 8192 * f / (2 * math.pi)
        assert g == pytest.approx(f if turns >= 4 else f / 8 if turns <= 1 else
                                  f * ((turns - 1) / 3 + (4 - turns) / 3 / 8), rel=1e-13)
    got = freqs(64, scaling="index", factor=8.0, trained=4096, fast=32.0, slow=1.0)
    at = [64 * math.log(4096 / (2 * math.pi * n)) / (2 * math.log(10000.0)) for n in (32, 1)]
    lo, hi = math.floor(at[0]), math.ceil(at[1])
    for i, (f, g) in enumerate(zip(plain, got)):
        w = min(1.0, max(0.0, 1 - (i - lo) / (hi - lo)))
        assert g == pytest.approx(w * f + (1 - w) * f / 8, rel=1e-13)


@pytest.mark.parametrize("kw,msg", [
    (dict(rot_dim=3), "rot_dim"), (dict(rot_dim=0), "rot_dim"), (dict(base=1.0), "base"), (dict(base=math.nan), "base"),
    (dict(scaling="linear", factor=0.5), "factor"), (dict(scaling="turns", factor=2.0), "trained"),
    (dict(scaling="index", factor=2.0, trained=100, fast=1.0, slow=1.0), "trained"),
    (dict(rot_dim=2, scaling="base", factor=2.0), "a scaled base"), (dict(scaling="other"), "unknown scaling")])
def test_frequency_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        rt.rope_table(**({"rot_dim": 64, "device": "cpu"} | kw))


def test_binding_refuses_host_tensors():
    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        rt.rope(x, x, None, torch.zeros(32, dtype=torch.int64))
    with pytest.raises(ValueError, match="device tensor"):
        rt.KvCache(x, x)
    with pytest.raises(ValueError, match="parents"):
        rt.tree_mask(torch.zeros(1, 4, dtype=torch.int32))


def test_oracle_rounds_codes_as_the_type():
    # torch's own f32 -> e4m3 conversion on rows whose quotient is exact (a = 448).
    x = np.concatenate([np.linspace(-448, 448, 9001), [0.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10]])
    x = torch.from_numpy(x).float().to(torch.bfloat16).double().numpy()
    codes, scale = C.quantise(x, "e4m3")
    assert scale == np.float32(1.0)
    assert np.array_equal(codes, torch.from_numpy(x).float().to(torch.float8_e4m3fn).double().numpy())
    assert np.array_equal(C.quantise(np.array([127.0, 0.5, 1.5, 2.5, -0.5]), "i8")[0], [127, 0, 2, 2, 0])


def test_oracle_words_and_ancestors():
    seen, depth = C.ancestors([-1, 0, 0, 2, 9])
    assert depth.tolist() == [0, 1, 1, 2, 0]
    assert C.words_of(seen)[:, 0].tolist() == [1, 3, 5, 13, 16]
    wide = np.zeros((1, 65), bool)
    wide[0, [0, 64]] = True
    assert C.words_of(wide).tolist() == [[1, 1]]
