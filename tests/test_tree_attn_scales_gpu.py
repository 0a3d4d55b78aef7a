"""frisk_tree_attn over 8-bit caches whose scales differ widely or are NaN: the
weights, their sum and its logarithm depend on the scores only, and a result's dim
only on the keys whose values feed it.  Tolerances as in test_tree_attn_gpu.py
(per dim: A is the sum of weight * |v| of that dim)."""
import pytest
import torch

from tests.test_tree_attn_gpu import Setup

pytestmark = pytest.mark.gpu

KINDS8 = [("bf16", "e4m3"), ("f16", "e4m3"), ("bf16", "i8"), ("f16", "i8")]
# One query tile, drafted tokens, tiles of rows over shared keys (4, then 8), a
# head dim without a matrix-core kernel.
SIZES = [(1, 8, 2, 1, 128, 700), (2, 4, 4, 33, 64, 257), (1, 4, 1, 20, 32, 130), (1, 4, 2, 5, 80, 90),
         (4, 16, 4, 512, 64, 300), (4, 16, 4, 512, 128, 300), (8, 16, 4, 512, 128, 300)]
ROWS = (1, 31, 32, 200, 383)


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


@pytest.mark.parametrize("dt,kind", KINDS8)
@pytest.mark.parametrize("batch,heads,kv,tokens,d,ctx", SIZES)
def test_weights_do_not_depend_on_value_scales(batch, heads, kv, tokens, d, ctx, dt, kind):
    # Value scales of 2^-60 to 2^60, and zero rows with the least scale there is.
    s = Setup(batch, heads, kv, tokens, d, dt, kind, 16, (ctx,) * batch, seed=3 * d + tokens)
    s.cache.v_scale.fill_(1.0)
    _, want = s.run(out=torch.float32)
    gen = torch.Generator().manual_seed(tokens)
    s.cache.v_scale.copy_(torch.exp2(torch.randint(-60, 61, s.cache.v_scale.shape, generator=gen).float()))
    s.cache.v_scale[:, :, 5::6] = 2.0 ** -126
    s.cache.v.view(torch.uint8)[:, :, 5::6] = 0
    o, lse = s.run(out=torch.float32)
    assert torch.equal(lse, want)
    s.check(o, lse, rows=ROWS, heads=(0, heads - 1), seqs=(0, batch - 1))


@pytest.mark.parametrize("dt,kind", KINDS8)
@pytest.mark.parametrize("batch,heads,kv,tokens,d,ctx", SIZES)
def test_a_value_scale_that_is_nan(batch, heads, kv, tokens, d, ctx, dt, kind):
    # The scale of a row with an infinity: NaN results for the tokens that see it,
    # the same sums as without for all.
    s = Setup(batch, heads, kv, tokens, d, dt, kind, 16, (ctx,) * batch, seed=d + tokens)
    o0, l0 = s.run()
    assert torch.isfinite(l0).all()
    for key, first in ((11, 0), (ctx + tokens // 2, tokens // 2)):  # of the context, a draft
        p, r = int(s.table[0, key // 16]), key % 16
        keep = s.cache.v_scale[p, :, r].clone()
        s.cache.v_scale[p, :, r] = float("nan")
        o, lse = s.run()
        s.cache.v_scale[p, :, r] = keep
        assert torch.equal(lse, l0)
        assert torch.isnan(o[0, :, first:]).all()
        assert torch.equal(o[0, :, :first], o0[0, :, :first]) and torch.equal(o[1:], o0[1:])


@pytest.mark.parametrize("dt,kind", KINDS8 + [("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("batch,heads,kv,tokens,d,ctx", SIZES)
def test_a_first_row_that_is_nan(batch, heads, kv, tokens, d, ctx, dt, kind):
    # Keys that do not exist are loaded from the cache's first row and hidden:
    # NaN there, in a page that is no sequence's, changes no bit.
    s = Setup(batch, heads, kv, tokens, d, dt, kind, 16, (ctx,) * batch, seed=d + tokens)
    free = (set(range(s.cache.k.shape[0])) - set(s.table.flatten().tolist())).pop()
    s.cache.block_table[s.cache.block_table == 0] = free  # that page's sequence takes the free one
    o0, l0 = s.run()
    for t in (s.cache.k, s.cache.v):
        if t.element_size() == 2:
            t[0] = float("nan")
        elif kind == "e4m3":
            t.view(torch.uint8)[0] = 0x7F
    if s.cache.k_scale is not None:
        s.cache.k_scale[0] = s.cache.v_scale[0] = float("nan")
    o, lse = s.run()
    assert torch.isfinite(lse).all() and torch.equal(o, o0) and torch.equal(lse, l0)
