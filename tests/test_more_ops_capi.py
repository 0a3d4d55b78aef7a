"""Refusals of the entries for draft verification, pages of a cache, positions of
several axes and shared scales, before any device work (no GPU needed), and their
descriptors' layouts."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from frisk_amd import runtime as rt
from tests.test_cache_ops_capi import CACHE_REFUSALS, cache_desc

HEADER = Path(__file__).resolve().parent.parent / "include" / "frisk_hip.h"


def call(name, desc):
    lib = rt.load()
    rc = getattr(lib, name)(ctypes.byref(desc), None)
    return rc, lib.frisk_last_error().decode()


def test_descriptor_layouts_match_the_header(tmp_path):
    structs = {"frisk_rope_desc": rt.RopeDesc, "frisk_kv_cache": rt.KvCacheDesc, "frisk_kv_desc": rt.KvDesc,
               "frisk_tree_attn_desc": rt.TreeAttnDesc, "frisk_kv_compact_desc": rt.KvCompactDesc,
               "frisk_kv_copy_pages_desc": rt.KvCopyPagesDesc, "frisk_kv_pages_desc": rt.KvPagesDesc,
               "frisk_tree_verify_desc": rt.TreeVerifyDesc}
    lines = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} . %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.strip().split("\n")}
    for cname, py in structs.items():
        assert got[cname, "."] == ctypes.sizeof(py), cname
        for field, _ in py._fields_:
            assert got[cname, field] == getattr(py, field).offset, (cname, field)


# ---- shared scales ------------------------------------------------------------------

CODES = dict(dtype=rt.E4M3, k_scale=1 << 20, v_scale=1 << 22)
BLOCK_REFUSALS = [
    (dict(scale_block=3), rt.EINVAL, "scale_block must"), (dict(scale_block=-1), rt.EINVAL, "scale_block must"),
    (dict(scale_block=512), rt.EINVAL, "scale_block must"), (dict(scale_block=16), rt.EINVAL, "scale_block is for 8-bit"),
    (dict(scale_block=32, **CODES), rt.EINVAL, "scale_block 32 is larger than a page"),
    (dict(scale_block=8, scale_stride_head=1, scale_stride_page=2, **CODES), rt.EINVAL,
     "the cache's rows or scales overlap"),
    (dict(scale_block=8, scale_stride_slot=0, **CODES), rt.EINVAL, "scale strides")]


@pytest.mark.parametrize("cache,code,msg", BLOCK_REFUSALS)
@pytest.mark.parametrize("name", ["frisk_kv_append", "frisk_kv_read", "frisk_tree_attn", "frisk_kv_compact",
                                  "frisk_kv_copy_pages"])
def test_block_scale_refusals(name, cache, code, msg):
    c = cache_desc(**cache)
    if name == "frisk_tree_attn":
        d = rt.TreeAttnDesc(batch=2, heads=4, tokens=3, dtype=rt.BF16, o_dtype=rt.BF16, sm_scale=0.125, q=16,
                            o=16, ctx_len=64, cache=c)
    elif name == "frisk_kv_compact":
        d = rt.KvCompactDesc(2, 3, 64, 3, 64, 64, c)
    elif name == "frisk_kv_copy_pages":
        d = rt.KvCopyPagesDesc(2, 64, 64, None, c)
    else:
        d = rt.KvDesc(batch=2, tokens=3, dtype=rt.BF16, k=16, v=1 << 16, ctx_len=64, cache=c)
    rc, err = call(name, d)
    assert rc == code and err.startswith(f"{name}: {msg}"), err


def test_scales_of_blocks_may_lie_next_to_each_other():
    # 8 pages, 2 heads, 2 scales a page: 128 bytes each, one behind the other.
    c = cache_desc(scale_block=8, scale_stride_slot=1, scale_stride_head=2, scale_stride_page=4, dtype=rt.E4M3,
                   k_scale=1 << 20, v_scale=(1 << 20) + 128, v=1 << 24, head_dim=72)
    # (head_dim 72 is refused behind the checks of the blocks' sizes.)
    d = rt.KvDesc(batch=2, tokens=3, dtype=rt.BF16, k=16, v=1 << 16, ctx_len=64, cache=c)
    assert "head_dim" in call("frisk_kv_append", d)[1]
    c.head_dim, d.k = 64, 0
    d.cache = c
    rc, err = call("frisk_kv_append", d)
    assert rc == rt.EINVAL and "null tensor" in err
    # One word less, and the page tables are the first thing wrong with it.
    c.v_scale = (1 << 20) + 124
    d.cache, d.k, d.k_stride_s, d.v_stride_s = c, 16, 64, 64
    d.k_stride_b = d.v_stride_b = 384
    d.k_stride_h = d.v_stride_h = 192
    rc, err = call("frisk_kv_append", d)
    assert rc == rt.EINVAL and "k_scale and v_scale must be two tensors" in err


# ---- pages --------------------------------------------------------------------------


# (Copies know no sequences, which these two refusals are about.)
PAGE_REFUSALS = [("frisk_kv_compact", *r) for r in CACHE_REFUSALS] + \
    [("frisk_kv_copy_pages", *r) for r in CACHE_REFUSALS if r[0].get("pages") != 1 and r[0].get("table_stride") != 3]


@pytest.mark.parametrize("name,cache,code,msg", PAGE_REFUSALS)
def test_page_cache_refusals(name, cache, code, msg):
    if name == "frisk_kv_compact":
        d = rt.KvCompactDesc(2, 3, 64, 3, 64, 64, cache_desc(**cache))
    else:
        d = rt.KvCopyPagesDesc(2, 64, 64, None, cache_desc(**cache))
    rc, err = call(name, d)
    assert rc == code and err.startswith(f"{name}: {msg}"), err


@pytest.mark.parametrize("over,cache,code,msg", [
    (dict(batch=0), {}, rt.EINVAL, "sizes must"), (dict(tokens=0), {}, rt.EINVAL, "sizes must"),
    (dict(path=None), {}, rt.EINVAL, "null tensor"), (dict(count=None), {}, rt.EINVAL, "null tensor"),
    (dict(ctx_len=None), {}, rt.EINVAL, "null tensor"), (dict(path=2), {}, rt.EINVAL, "path, ctx_len"),
    (dict(path_stride=-1), {}, rt.EINVAL, "path_stride"), (dict(batch=1 << 31), {}, rt.EUNSUP, "sizes beyond"),
    (dict(), dict(v=4096), rt.EINVAL, "k and v, and"),
    (dict(), dict(CODES, v_scale=1 << 20, v=1 << 24), rt.EINVAL, "k and v, and"),
    (dict(), dict(CODES, scale_block=8, v=1 << 24), rt.EUNSUP, "rows that share scales")])
def test_compact_refusals(over, cache, code, msg):
    d = dict(batch=2, tokens=3, path=64, path_stride=3, ctx_len=64, count=64) | over
    rc, err = call("frisk_kv_compact", rt.KvCompactDesc(**d, cache=cache_desc(**(dict(v=1 << 26) | cache))))
    assert rc == code and err.startswith(f"frisk_kv_compact: {msg}"), err


@pytest.mark.parametrize("over,cache,code,msg", [
    (dict(pairs=0), {}, rt.EINVAL, "sizes must"), (dict(src=None), {}, rt.EINVAL, "null tensor"),
    (dict(dst=None), {}, rt.EINVAL, "null tensor"), (dict(rows=2), {}, rt.EINVAL, "src, dst"),
    (dict(pairs=1 << 31), {}, rt.EUNSUP, "more pages"), (dict(), dict(v=4096), rt.EINVAL, "k and v, and")])
def test_copy_refusals(over, cache, code, msg):
    d = dict(pairs=2, src=64, dst=64, rows=None) | over
    rc, err = call("frisk_kv_copy_pages", rt.KvCopyPagesDesc(**d, cache=cache_desc(**(dict(v=1 << 26) | cache))))
    assert rc == code and err.startswith(f"frisk_kv_copy_pages: {msg}"), err


@pytest.mark.parametrize("over,code,msg", [
    (dict(batch=0), rt.EINVAL, "sizes must"), (dict(max_pages=0), rt.EINVAL, "sizes must"),
    (dict(pages=-1), rt.EINVAL, "sizes must"), (dict(page_size=24), rt.EINVAL, "page_size must"),
    (dict(pages=1 << 20), rt.EUNSUP, "more pages and"), (dict(batch=1 << 15, max_pages=1), rt.EUNSUP, "more pages and"),
    (dict(page_size=1 << 30), rt.EUNSUP, "a table of"), (dict(table_stride=3), rt.EINVAL, "rows of table"),
    (dict(out_stride=3), rt.EINVAL, "rows of table"), (dict(table=None), rt.EINVAL, "null tensor"),
    (dict(keep=None), rt.EINVAL, "null tensor"), (dict(out=None), rt.EINVAL, "null tensor"),
    (dict(src=2), rt.EINVAL, "pointers must"), (dict(out=64 + 28), rt.EINVAL, "an output overlaps"),
    (dict(src=4096, dst=4100), rt.EINVAL, "an output overlaps"), (dict(lacking=1024), rt.EINVAL, "an output overlaps"),
    (dict(held=4096, rows=4096 + 8), rt.EINVAL, "an output overlaps")])
def test_pages_refusals(over, code, msg):
    d = dict(batch=2, max_pages=4, pages=16, page_size=16, table=64, table_stride=4, out=512, out_stride=4,
             parent=None, keep=1024, want=None) | over
    rc, err = call("frisk_kv_pages", rt.KvPagesDesc(**d))
    assert rc == code and err.startswith(f"frisk_kv_pages: {msg}"), err


# ---- verification -------------------------------------------------------------------


def verify_desc(**over):
    d = dict(batch=2, tokens=3, vocab=100, dtype=rt.BF16, logits=1 << 20, stride_b=300, stride_t=100,
             drafts=1 << 12, parents=1 << 13, uniform=1 << 14, final_uniform=1 << 15, path=1 << 16, count=1 << 17,
             token=1 << 18, workspace=1 << 24, workspace_bytes=1 << 20) | over
    return rt.TreeVerifyDesc(**d)


@pytest.mark.parametrize("over,code,msg", [
    (dict(batch=0), rt.EINVAL, "sizes must"), (dict(tokens=0), rt.EINVAL, "sizes must"),
    (dict(vocab=0), rt.EINVAL, "sizes must"), (dict(dtype=rt.E4M3), rt.EINVAL, "dtype must"),
    (dict(tokens=1025), rt.EUNSUP, "up to 1024"), (dict(vocab=(1 << 24) + 1), rt.EUNSUP, "up to 1024"),
    (dict(batch=1 << 30), rt.EUNSUP, "more trees"), (dict(batch=1 << 24, vocab=1 << 20), rt.EUNSUP, "more rows"),
    (dict(stride_t=-1), rt.EINVAL, "strides must"), (dict(draft_probs=4, draft_stride_b=-1), rt.EINVAL, "strides must"),
    (dict(logits=None), rt.EINVAL, "null tensor"), (dict(final_uniform=None), rt.EINVAL, "null tensor"),
    (dict(token=None), rt.EINVAL, "null tensor"), (dict(logits=(1 << 20) + 1), rt.EINVAL, "pointers must"),
    (dict(probs=2), rt.EINVAL, "pointers must"), (dict(workspace=None), rt.EINVAL, "workspace of 0 bytes"),
    (dict(workspace_bytes=100), rt.EINVAL, "workspace of 100 bytes"),
    (dict(workspace=(1 << 24) + 8), rt.EINVAL, "workspace must be"),
    (dict(path=(1 << 12) + 20), rt.EINVAL, "an output overlaps"), (dict(count=1 << 18), rt.EINVAL, "an output overlaps"),
    (dict(token=(1 << 20) + 1196), rt.EINVAL, "an output overlaps"),
    (dict(probs=(1 << 24) + 16), rt.EINVAL, "an output overlaps")])
def test_verify_refusals(over, code, msg):
    rc, err = call("frisk_tree_verify", verify_desc(**over))
    assert rc == code and err.startswith(f"frisk_tree_verify: {msg}"), err


def test_null_descriptors_and_the_workspace_query():
    lib = rt.load()
    for name in ("frisk_kv_compact", "frisk_kv_copy_pages", "frisk_kv_pages", "frisk_tree_verify"):
        assert getattr(lib, name)(None, None) == rt.EINVAL
    assert lib.frisk_tree_verify_workspace_size(None) == rt.EINVAL
    assert lib.frisk_tree_verify_workspace_size(ctypes.byref(verify_desc(tokens=0))) == rt.EINVAL
    assert rt.tree_verify_workspace_bytes(1, 1, 1000, torch.float32) == 0
    small = rt.tree_verify_workspace_bytes(1, 2, 1, torch.float32)
    large = rt.tree_verify_workspace_bytes(64, 64, 131072, torch.bfloat16)
    assert 0 < small < 1024 and small < large < 64 << 20
    with pytest.raises(ValueError, match="up to 1024"):
        rt.tree_verify_workspace_bytes(1, 2000, 10, torch.float32)


# ---- positions of several axes ----------------------------------------------------------


@pytest.mark.parametrize("over,code,msg", [
    (dict(axes=0), rt.EUNSUP, "positions of 1 to 4 axes"), (dict(axes=5), rt.EUNSUP, "positions of 1 to 4 axes"),
    (dict(axes=3, positions=None), rt.EINVAL, "pair_axis needs"),
    (dict(axes=3, pos_stride_a=-1), rt.EINVAL, "position strides")])
def test_axes_refusals(over, code, msg):
    d = dict(batch=1, seq=2, heads=1, head_dim=64, rot_dim=64, dtype=rt.F32, amplitude=1.0, x=16, x_stride_b=128,
             x_stride_h=128, x_stride_s=64, out=16, out_stride_b=128, out_stride_h=128, out_stride_s=64, frequencies=8,
             positions=64, position_bits=32, pair_axis=1) | over
    rc, err = call("frisk_rope", rt.RopeDesc(**d))
    assert rc == code and err.startswith(f"frisk_rope: {msg}"), err


def test_axes_of_pairs():
    assert rt.rope_axes([2, 3, 1], device="cpu").tolist() == [0, 0, 1, 1, 1, 2]
    assert rt.rope_axes([2, 3, 1], interleaved=True, device="cpu").tolist() == [0, 1, 2, 0, 1, 1]
    assert rt.rope_axes([0, 2], device="cpu").tolist() == [1, 1]
    for bad in ([], [1, 2, 3, 4, 5], [-1, 2], [0, 0]):
        with pytest.raises(ValueError, match="sections"):
            rt.rope_axes(bad, device="cpu")


def test_binding_refuses_host_tensors():
    i32 = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="table must"):
        rt.kv_pages(i32, i32[:, 0], None, 16, 8)
    with pytest.raises(ValueError, match="logits must"):
        rt.tree_verify(torch.zeros(2, 4, 9), i32, i32, i32.float(), i32[:, 0].float())
    with pytest.raises(ValueError, match="logits must"):
        rt.tree_verify(torch.zeros(4, 9), i32, i32, i32.float(), i32[:, 0].float())
