"""frisk_tree_attn over 8-bit caches whose scales differ widely or are NaN: the
weights, their sum and its logarithm depend on the scores only, and a result's dim
only on the keys whose values feed it.  Tolerances as in test_tree_attn_gpu.py
(per dim: A is the sum of weight * |v| of that dim)."""
import numpy as np
import pytest
import torch

from oracle import cache_ops as C
from tests.test_tree_attn_gpu import Setup

pytestmark = pytest.mark.gpu

KINDS8 = [("bf16", "e4m3"), ("f16", "e4m3"), ("bf16", "i8"), ("f16", "i8")]
# One query tile, drafted tokens, tiles of rows over shared keys (4, then 8), a
# head dim without a matrix-core kernel.
SIZES = [(1, 8, 2, 1, 128, 700), (2, 4, 4, 33, 64, 257), (1, 4, 1, 20, 32, 130), (1, 4, 2, 5, 80, 90),
         (4, 16, 4, 512, 64, 300), (4, 16, 4, 512, 128, 300), (8, 16, 4, 512, 128, 300)]
ROWS = (1, 31, 32, 200, 383)


def codes(s, which):
    return s.cache.k if which == "k" else s.cache.v


@pytest.mark.parametrize("dt,kind", KINDS8)
@pytest.mark.parametrize("batch,heads,kv,tokens,d,ctx", SIZES)
def test_dims_that_small_scales_feed(batch, heads, kv, tokens, d, ctx, dt, kind):
    # Every fourth value row is 2^k of the others and 0 in the first half of the
    # dims: what is there comes from the other rows alone.
    s = Setup(batch, heads, kv, tokens, d, dt, kind, 16, (ctx,) * batch, seed=d + tokens)
    for k in (14, 20, 40):
        v = s.cache.v.view(torch.uint8)
        v[:, :, ::4, :d // 2] = 0
        s.cache.v_scale.copy_(0.01 * torch.exp2(torch.randint(0, 3, s.cache.v_scale.shape).float()))
        s.cache.v_scale[:, :, ::4] *= 2.0 ** k
        o, lse = s.run(out=torch.float32)
        s.check(o, lse, rows=ROWS, heads=(0, heads - 1), seqs=(0, batch - 1))
