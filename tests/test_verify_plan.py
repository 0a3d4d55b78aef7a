"""The rules by which draft verification is launched, as a host program runs them
(csrc/launch_plan.h), and the calls that one launch does not take."""
import ctypes

import pytest

from frisk_amd import runtime as rt
from tests.test_more_ops_capi import call, verify_desc


@pytest.mark.parametrize("tokens,vocab,dtype", [(1, 100, rt.BF16), (3, 100, rt.F32), (1, 8000, rt.F16)])
def test_more_trees_than_a_launch_takes(tokens, vocab, dtype):
    # A tree has a workgroup of 1024 threads, in the walk or by itself: 2^22 trees have 2^32.
    lib = rt.load()
    sizes = dict(tokens=tokens, vocab=vocab, dtype=dtype, logits=1 << 40)
    for batch in (1 << 22, (1 << 22) + 1, ((1 << 24) - 1) // (tokens * 16)):
        d = verify_desc(batch=batch, workspace_bytes=1 << 40, workspace=1 << 46, **sizes)
        fits = batch < 1 << 22
        assert (lib.frisk_tree_verify_workspace_size(ctypes.byref(d)) >= 0) == fits, batch
        if not fits:
            rc, err = call("frisk_tree_verify", d)
            assert rc == rt.EUNSUP and err.startswith("frisk_tree_verify: more "), err
