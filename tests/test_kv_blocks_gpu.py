"""A cache whose slots share scales: frisk_kv_append and frisk_kv_read to the bit
against the definition, frisk_tree_attn against the fp64 oracle (tolerances as
in test_tree_attn_gpu.py: codes times scales are exact there)."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import serving_ops as S
from tests.gpu_util import decode, randn
from tests.test_tree_attn_gpu import Setup, tree

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Blocks:
    """A cache of random codes and scales with a model of it in numpy."""

    def __init__(self, batch, kv, d, dt, kind, page, block, cap, slot_first=False, seed=1):
        self.kv, self.d, self.dt, self.kind, self.page, self.block, self.cap = kv, d, dt, kind, page, block, cap
        rng = np.random.default_rng(seed)
        table, pages, size = None, batch, cap
        if page:
            per = -(-cap // page)
            pages, size = batch * per + 1, page
            table = rng.permutation(pages)[:batch * per].reshape(batch, per)
        self.table = table
        shape = (pages, size, kv, d) if slot_first else (pages, kv, size, d)

        def codes(s):
            x = (randn(shape, s) * 40).clamp(-127, 127).to(DT[kind])
            return x.transpose(1, 2) if slot_first else x

        scales = [torch.exp(0.3 * randn((pages, kv, -(-size // block)), seed + i)) * 0.02 for i in (3, 4)]
        self.cache = rt.KvCache(codes(seed), codes(seed + 1), *scales,
                                None if table is None else ints(table.tolist()), scale_block=block)
        self.values = [decode(t.contiguous()).astype(np.float64) for t in (self.cache.k, self.cache.v)]
        self.scales = [s.cpu().numpy().copy() for s in (self.cache.k_scale, self.cache.v_scale)]

    def where(self, b, n):
        """(page, slot) of a key, or None."""
        if n >= (self.table.shape[1] * self.page if self.page else self.cap):
            return None
        if not self.page:
            return b, n
        page = int(self.table[b, n // self.page])
        return (page, n % self.page) if 0 <= page < len(self.values[0]) else None

    def append(self, k, v, ctx, new):
        for side, x in enumerate((k, v)):
            x = x.double().cpu().numpy()  # [batch, kv, tokens, d]
            for b, (c, n) in enumerate(zip(ctx, new)):
                if c < 0:
                    continue
                for first in range(c // self.block * self.block, c + n, self.block):
                    at = self.where(b, first)
                    lo, hi = max(first, c), min(first + self.block, c + n)
                    hi = min(hi, self.table.shape[1] * self.page if self.page else self.cap)
                    if at is None or lo >= hi:
                        continue
                    page, slot = at
                    for h in range(self.kv):
                        rows = slice(slot, slot + hi - first)
                        got, s = S.append_block(self.values[side][page, h, rows], self.scales[side][page, h, slot // self.block],
                                                lo - first, x[b, h, lo - c:hi - c], self.kind)
                        self.values[side][page, h, rows] = got
                        self.scales[side][page, h, slot // self.block] = s

    def check(self):
        """Every code and scale, the untouched ones too."""
        c = self.cache
        for t, values, s, scales in ((c.k, self.values[0], c.k_scale, self.scales[0]),
                                     (c.v, self.values[1], c.v_scale, self.scales[1])):
            np.testing.assert_array_equal(s.cpu().numpy(), scales)
            np.testing.assert_array_equal(decode(t.contiguous()), values)


def rows(batch, tokens, kv, d, dt, seed, spread=1.0):
    return [(spread * randn((batch, tokens, kv, d), seed + i) * torch.exp(0.5 * randn((d,), seed + 9))).to(DT[dt])
            .transpose(1, 2) for i in (0, 1)]


CASES = [
    # batch, tokens, kv heads, head_dim, dtype, kind, page (0: none), block, slot first
    (2, 5, 2, 128, "bf16", "e4m3", 16, 16, False), (1, 1, 1, 16, "f16", "i8", 0, 2, False),
    (3, 70, 3, 64, "f16", "e4m3", 32, 8, True), (2, 33, 5, 80, "bf16", "i8", 64, 32, False),
    (2, 300, 2, 256, "bf16", "i8", 256, 256, False), (2, 9, 1, 32, "f16", "e4m3", 64, 64, True),
    (1, 1000, 2, 128, "bf16", "e4m3", 0, 64, False), (2, 3, 2, 48, "bf16", "i8", 4, 4, False)]


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("b,t,kv,d,dt,kind,page,block,slot_first", CASES)
def test_append_and_read(b, t, kv, d, dt, kind, page, block, slot_first, ragged):
    ctx = [(5 * i + 3) % 11 for i in range(b)] if ragged else [block] * b
    new = [max(1, t - 2 * i) for i in range(b)] if ragged else [t] * b
    m = Blocks(b, kv, d, dt, kind, page, block, max(c + n for c, n in zip(ctx, new)) + 3, slot_first)
    # Twice: the second rows are larger, so that most blocks' scales grow, then smaller.
    for step, spread in enumerate((0.5, 3.0, 0.01)):
        k, v = rows(b, t, kv, d, dt, 10 * step + 1, spread)
        new_len = ints(new) if ragged else None
        rt.kv_append(k, v, m.cache, ints(ctx), new_len=new_len)
        m.append(k, v, ctx, new)
        m.check()
        ko, vo = (torch.full((b, kv, t, d), 5.0, dtype=DT[dt], device="cuda") for _ in range(2))
        rt.kv_read(m.cache, ko, vo, ints(ctx), new_len=new_len)
        for out, values, scales in ((ko, m.values[0], m.scales[0]), (vo, m.values[1], m.scales[1])):
            want = torch.full(out.shape, 5.0)
            for i in range(b):
                for n in range(new[i]):
                    at = m.where(i, ctx[i] + n)
                    if at:
                        # (f32: the product's one rounding before the output's)
                        want[i, :, n] = torch.from_numpy(values[at[0], :, at[1]].astype(np.float32) *
                                                         scales[at[0], :, at[1] // block][:, None])
            assert torch.equal(out.cpu(), want.to(DT[dt]))
        ctx = [c + max(0, n - 2) for c, n in zip(ctx, new)] if step == 0 else ctx
        ctx = [min(c, m.cap - n) for c, n in zip(ctx, new)]


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_token_by_token(kind):
    # A block filled by single tokens of rising size; then back into its middle.
    m = Blocks(2, 2, 64, "bf16", kind, 32, 32, 96)
    for n in list(range(40)) + [10, 11]:
        k, v = rows(2, 1, 2, 64, "bf16", n, 1.0 + n % 7)
        rt.kv_append(k, v, m.cache, ints([n, n + 20]))
        m.append(k, v, [n, n + 20], [1, 1])
        m.check()


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_values_that_are_not_finite(kind):
    m = Blocks(1, 2, 64, "bf16", kind, 16, 8, 64)
    for n, (value, at) in enumerate(((float("inf"), 3), (float("nan"), 9), (-float("inf"), 20))):
        k, v = rows(1, 6, 2, 64, "bf16", n)
        (k if n != 1 else v)[0, n % 2, 2, 5] = value
        rt.kv_append(k, v, m.cache, ints([at]))
        m.append(k, v, [at], [6])
        m.check()
    assert np.isnan(m.scales[0]).any() and np.isnan(m.scales[1]).any()
    # Keys behind in such a block stay NaN; from its start on it is another's.
    k, v = rows(1, 2, 2, 64, "bf16", 8)
    for at in (6, 0):
        rt.kv_append(k, v, m.cache, ints([at]))
        m.append(k, v, [at], [2])
        m.check()


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_zeros_and_extremes(dt, kind):
    m = Blocks(1, 1, 32, dt, kind, 8, 8, 40)
    top = torch.finfo(DT[dt]).max
    for at, value in ((0, 0.0), (2, torch.finfo(DT[dt]).tiny), (4, top), (8, top), (10, 0.0), (16, 2.0 ** -24)):
        k = torch.full((1, 1, 2, 32), value, dtype=DT[dt], device="cuda")
        v = -k
        rt.kv_append(k, v, m.cache, ints([at]))
        m.append(k, v, [at], [2])
        m.check()


def test_pages_that_are_none_and_lengths():
    m = Blocks(4, 2, 32, "bf16", "i8", 8, 4, 32)
    m.table[0, 1], m.table[1, 0], m.table[2, 2] = -1, len(m.values[0]), 2 ** 31 - 1
    m.cache.block_table.copy_(ints(m.table.tolist()))
    k, v = rows(4, 20, 2, 32, "bf16", 3)
    ctx, new = [3, 6, 14, -1], [20, 0, 20, 20]
    rt.kv_append(k, v, m.cache, ints(ctx), new_len=ints(new))
    m.append(k, v, ctx, new)
    m.check()
    rt.kv_append(k, v, m.cache, ints([30, 31, 32, 2 ** 31 - 1]), new_len=ints([20, 2 ** 31 - 1, 1, 1]))
    m.append(k, v, [30, 31, 32, 100], [20, 20, 1, 1])
    m.check()


# ---- attention -----------------------------------------------------------------------


class BlockSetup(Setup):
    """Setup's cache with a scale for `block` slots; `wide` has each row's own, equal ones."""

    def __init__(self, *args, block, **kw):
        super().__init__(*args, **kw)
        self.wide = self.cache
        c, n = self.cache, self.cache.k.shape[2]
        scales = [s[:, :, ::block].contiguous() for s in (c.k_scale, c.v_scale)]
        for s, w in zip(scales, (c.k_scale, c.v_scale)):
            w.copy_(s.repeat_interleave(block, 2)[:, :, :n])
        self.cache = rt.KvCache(c.k, c.v, *scales, c.block_table, scale_block=block)

    def rows(self, i):
        mine, self.cache = self.cache, self.wide
        try:
            return super().rows(i)
        finally:
            self.cache = mine


KINDS8 = [("bf16", "e4m3"), ("f16", "e4m3"), ("bf16", "i8"), ("f16", "i8")]
# batch, heads, kv, tokens, d, page, block, ctx: a query tile, drafts, tiles of rows over shared
# keys (4, then 8), a head dim without a matrix-core kernel; blocks below, of and above 64 keys.
SIZES = [(2, 8, 2, 1, 128, 64, 64, (700, 63)), (2, 8, 2, 1, 128, 16, 16, (129, 0)), (1, 4, 4, 33, 64, 0, 64, (257,)),
         (2, 4, 1, 20, 32, 128, 128, (130, 64)), (1, 4, 2, 5, 80, 32, 32, (90,)), (2, 4, 2, 40, 64, 256, 256, (333, 1)),
         (1, 4, 1, 3, 128, 64, 2, (65,)), (4, 16, 4, 512, 64, 64, 64, (300, 64, 1, 127)),
         (4, 16, 4, 512, 128, 16, 16, (300, 64, 1, 127)), (4, 16, 4, 512, 128, 64, 64, (300, 64, 1, 127)),
         (8, 16, 4, 512, 128, 64, 64, (300, 5, 64, 63, 190, 128, 1, 0))]
ROWS = (1, 31, 32, 200, 383)


@pytest.mark.parametrize("dt,kind", KINDS8)
@pytest.mark.parametrize("batch,heads,kv,tokens,d,page,block,ctx", SIZES)
def test_attention(batch, heads, kv, tokens, d, page, block, ctx, dt, kind):
    s = BlockSetup(batch, heads, kv, tokens, d, dt, kind, page, ctx, seed=d + tokens, block=block)
    for out in (None, torch.float32):
        o, lse = s.run(out=out)
        s.check(o, lse, rows=ROWS, heads=(0, heads - 1), seqs=(0, batch - 1))
    o, lse = s.run(workspace=False)
    s.check(o, lse, rows=ROWS, heads=(0, heads - 1), seqs=(0, batch - 1))


@pytest.mark.parametrize("dt,kind", KINDS8)
@pytest.mark.parametrize("block", [16, 64])
def test_trees_and_ragged_batches(dt, kind, block):
    for batch, heads, kv, tokens, d, ctx in ((3, 4, 2, 21, 128, (100, 64, -1)), (4, 16, 2, 130, 64, (500, 0, 63, 250))):
        new = [tokens - 3 * i for i in range(batch)]
        s = BlockSetup(batch, heads, kv, tokens, d, dt, kind, 64, ctx, new=new, seed=d + block, block=block)
        mask, seen = tree(batch, tokens, 5)
        o, lse = s.run(mask=mask)
        s.check(o, lse, seen=seen, heads=(0, heads - 1))


@pytest.mark.parametrize("dt,kind", KINDS8)
def test_value_scales_that_are_nan_or_far_apart(dt, kind):
    for tokens, d in ((1, 128), (33, 64), (5, 80), (512, 128)):
        batch, heads, kv, ctx = (4, 16, 4, 300) if tokens == 512 else (2, 4, 4, 300)
        s = BlockSetup(batch, heads, kv, tokens, d, dt, kind, 64, (ctx,) * batch, seed=tokens, block=64)
        gen = torch.Generator().manual_seed(tokens)
        s.cache.v_scale.copy_(torch.exp2(torch.randint(-60, 61, s.cache.v_scale.shape, generator=gen).float()))
        s.wide.v_scale.copy_(s.cache.v_scale.repeat_interleave(64, 2))
        o0, l0 = s.run(out=torch.float32)
        s.check(o0, l0, rows=ROWS, heads=(0, heads - 1), seqs=(0, batch - 1))
        # A block of the context: all of the sequence; the drafts' last: those that see into it.
        for key, first in ((130, 0), (ctx + tokens - 1, max(0, (ctx + tokens - 1) // 64 * 64 - ctx))):
            p = int(s.table[0, key // 64])
            keep = s.cache.v_scale[p].clone()
            s.cache.v_scale[p] = float("nan")
            o, lse = s.run(out=torch.float32)
            s.cache.v_scale[p] = keep
            assert torch.equal(lse, l0)
            assert torch.isnan(o[0, :, first:]).all()
            assert torch.equal(o[0, :, :first], o0[0, :, :first]) and torch.equal(o[1:], o0[1:])


@pytest.mark.parametrize("dt,kind", KINDS8)
def test_a_key_scale_that_is_nan(dt, kind):
    # What sees the block is NaN; pages behind a sequence and of others do not matter.
    for tokens, d in ((1, 64), (40, 128), (512, 128)):
        batch, heads, kv = (4, 16, 4) if tokens == 512 else (2, 4, 2)
        s = BlockSetup(batch, heads, kv, tokens, d, dt, kind, 64, (100,) * batch, seed=tokens, block=64, spare=200)
        o0, l0 = s.run()
        used = set()
        for i in range(batch):
            used |= {int(s.table[i, n // 64]) for n in range(100 + tokens)}
        for p in set(range(s.cache.k.shape[0])) - used:
            s.cache.k_scale[p] = s.cache.v_scale[p] = float("nan")
        o, lse = s.run()
        assert torch.equal(o, o0) and torch.equal(lse, l0)
        s.cache.k_scale[int(s.table[0, 0])] = float("nan")
        o, lse = s.run()
        assert torch.isnan(o[0]).all() and torch.equal(o[1:], o0[1:])


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_graph_replay_and_streams(kind):
    # A captured step of append, read and attention: tokens and lengths change between replays.
    m = Blocks(2, 2, 64, "bf16", kind, 32, 16, 96)
    k, v = (torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda").transpose(1, 2) for _ in range(2))
    q, ctx = randn((2, 4, 3, 64), 7).to(torch.bfloat16), ints([0, 0])
    ko, vo, o = (torch.zeros_like(x) for x in (k, v, q))

    def step(stream=None):
        rt.kv_append(k, v, m.cache, ctx, stream=stream)
        rt.kv_read(m.cache, ko, vo, ctx, stream=stream)
        rt.tree_attn(q, m.cache, ctx, o, stream=stream)

    def load(n):
        for x, new in zip((k, v), rows(2, 3, 2, 64, "bf16", n, 1.0 + n % 5)):
            x.copy_(new)
        ctx.copy_(ints([2 * n, 3 * n + 1]))
        torch.cuda.synchronize()
        m.append(k, v, [2 * n, 3 * n + 1], [3, 3])

    side = torch.cuda.Stream()
    load(0)
    step(side)
    side.synchronize()
    m.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in range(1, 6):
        load(n)
        graph.replay()
        torch.cuda.synchronize()
        m.check()
        got = [x.clone() for x in (ko, vo, o)]
        rt.kv_read(m.cache, ko, vo, ctx)
        rt.tree_attn(q, m.cache, ctx, o)
        assert all(torch.equal(x, y) for x, y in zip(got, (ko, vo, o)))
