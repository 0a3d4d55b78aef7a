"""frisk_tree_attn against the fp64 oracle.

Tolerance of an output: the weights enter the second product rounded to q's
type, each off by half a step h of it, so a result is off by at most h times
A = sum of weight * |v|; scores in f32 are off by at most (head_dim + 4) 2^-24
sum |q k| scale, under 2^-12 here, which moves every weight by that factor;
and the result is rounded to its type once: h |o| + (h + 2^-12) A.  lse: the
scores' 2^-12, and 2^-20 of its size."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import cache_ops as C
from tests.gpu_util import decode, randn

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8}


class Setup:
    """A cache filled with random rows (unused slots too), queries and lengths."""

    def __init__(self, batch, heads, kv, tokens, d, dt, kind, page, ctx, new=None, seed=1, spare=0,
                 garbage=False, slot_first=False):
        self.batch, self.heads, self.kv, self.tokens, self.d, self.dt = batch, heads, kv, tokens, d, dt
        self.ctx = list(ctx)
        self.new = [tokens] * batch if new is None else list(new)
        cap = max(max(self.ctx), 0) + tokens + spare
        rng = np.random.default_rng(seed)
        table, pages, size = None, batch, cap
        if page:
            per = -(-cap // page)
            pages, size = batch * per + 1, page
            table = torch.from_numpy(rng.permutation(pages)[:batch * per].reshape(batch, per).astype(np.int32))
        self.table, self.page = table, page
        shape = (pages, size, kv, d) if slot_first else (pages, kv, size, d)

        def rows(s):
            x = randn(shape, s) * torch.exp(0.5 * randn((d,), s + 50))
            return x.transpose(1, 2) if slot_first else x

        scales = (None, None)
        if kind in C.TOP:
            scales = tuple(0.01 * torch.exp(0.5 * randn((pages, kv, size), seed + i)) for i in (7, 8))
            k, v = ((rows(seed + i) * (30 if kind == "i8" else 60)).clamp(-127, 127).to(DT[kind]) for i in (2, 3))
        else:
            k, v = (rows(seed + i).to(DT[kind]) for i in (2, 3))
        self.cache = rt.KvCache(k, v, *scales, None if table is None else table.cuda())
        self.q = randn((batch, tokens, heads, d), seed + 4).to(DT[dt]).transpose(1, 2)
        self.ctx_len = torch.tensor(self.ctx, dtype=torch.int32, device="cuda")
        self.new_len = None if new is None else torch.tensor(self.new, dtype=torch.int32, device="cuda")

    def rows(self, i):
        """Sequence i's K and V in fp64, [kv, keys, d]."""
        n = self.ctx[i] + self.new[i]
        at = np.arange(n)
        if self.table is None:
            pages, row = np.full(n, i), at
        else:
            pages, row = self.table[i].numpy()[at // self.page], at % self.page
        pages, row = torch.from_numpy(pages).long().cuda(), torch.from_numpy(row).long().cuda()
        out = []
        for t, s in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            if t.element_size() == 1:
                x = decode(t.view(torch.uint8)[pages, :, row].contiguous().view(t.dtype)).astype(np.float64)
                x = x * s[pages, :, row].double().cpu().numpy()[..., None]
            else:
                x = t[pages, :, row].double().cpu().numpy()
            out.append(x.transpose(1, 0, 2))
        return out

    def run(self, mask=None, out=None, lse=True, **kw):
        o = torch.full((self.batch, self.tokens, self.heads, self.d), 5.0, dtype=DT[self.dt] if out is None else out,
                       device="cuda").transpose(1, 2)
        l = torch.full((self.batch, self.heads, self.tokens), 5.0, device="cuda") if lse else None
        rt.tree_attn(self.q, self.cache, self.ctx_len, o, mask=mask, new_len=self.new_len, lse=l, **kw)
        return o, l

    def check(self, o, lse, seen=None, scale=None, rows=None, heads=None, seqs=None):
        """`seen` bool [batch, tokens, tokens], or None: causal.  rows, heads,
        seqs: the ones looked at (None: all)."""
        h = torch.finfo(DT[self.dt]).eps / 2
        out_h = h if o.dtype == DT[self.dt] else 0.0
        scale = self.d ** -0.5 if scale is None else scale
        group = self.heads // self.kv
        qd, od = self.q.double().cpu().numpy(), o.double().cpu().numpy()
        ld = None if lse is None else lse.double().cpu().numpy()
        for i in seqs or range(self.batch):
            live = self.new[i] if self.ctx[i] >= 0 else 0
            assert (od[i, :, live:] == 5.0).all() and (ld is None or (ld[i, :, live:] == 5.0).all())
            if not live:
                continue
            k, v = self.rows(i)
            vis = np.ones((live, self.ctx[i] + live), bool)
            vis[:, self.ctx[i]:] = np.tril(np.ones((live, live), bool)) if seen is None else seen[i][:live, :live]
            for head in heads or range(self.heads):
                pick = range(live) if rows is None else sorted({0, live - 1, *(r % live for r in rows)})
                pick = list(pick)
                wo, wl, wa = C.attention(qd[i, head, pick], k[head // group], v[head // group], vis[pick], scale)
                err = np.abs(od[i, head, pick] - wo)
                tol = out_h * np.abs(wo) + (h + 2.0 ** -12) * wa
                assert (err <= tol).all(), (i, head, float((err - tol).max()))
                if ld is not None:
                    got = ld[i, head, pick]
                    assert np.array_equal(np.isinf(got), np.isinf(wl))
                    fin = np.isfinite(wl)
                    assert (np.abs(got[fin] - wl[fin]) <= 2.0 ** -12 + 2.0 ** -20 * np.abs(wl[fin])).all()


def tree(batch, tokens, seed):
    rng = np.random.default_rng(seed)
    parents = np.array([[rng.integers(max(-1, i // 4 - 1), i) if i else -1 for i in range(tokens)]
                        for _ in range(batch)])
    seen = np.stack([C.ancestors(p)[0] for p in parents])
    mask, _ = rt.tree_mask(torch.from_numpy(parents.astype(np.int32)).cuda())
    return mask, seen


KINDS = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3"), ("bf16", "i8"), ("f16", "i8")]


@pytest.mark.parametrize("dt,kind", KINDS)
@pytest.mark.parametrize("batch,heads,kv,d,page,ctx", [
    (2, 8, 2, 128, 16, (300, 65)), (1, 4, 4, 64, 0, (1000,)), (3, 10, 2, 32, 64, (0, 1, 130)),
    (2, 6, 2, 80, 8, (77, 0)), (1, 16, 1, 256, 0, (129,)), (1, 3, 1, 16, 1, (70,)),
    (2, 32, 1, 128, 128, (513, 64))])
def test_one_token(batch, heads, kv, d, page, ctx, dt, kind):
    s = Setup(batch, heads, kv, 1, d, dt, kind, page, ctx)
    s.check(*s.run())


@pytest.mark.parametrize("dt,kind", KINDS)
@pytest.mark.parametrize("batch,heads,kv,tokens,d,page,ctx", [
    (2, 8, 2, 7, 128, 16, (300, 63)), (1, 4, 4, 33, 64, 0, (257,)), (2, 4, 1, 65, 128, 32, (0, 190)),
    (1, 8, 2, 130, 32, 64, (100,)), (2, 2, 1, 20, 96, 16, (5, 40)), (1, 16, 2, 64, 64, 0, (64,)),
    (1, 8, 1, 40, 128, 0, (500,))])
def test_trees(batch, heads, kv, tokens, d, page, ctx, dt, kind):
    s = Setup(batch, heads, kv, tokens, d, dt, kind, page, ctx, seed=tokens)
    mask, seen = tree(batch, tokens, tokens)
    s.check(*s.run(mask), seen)


@pytest.mark.parametrize("dt,kind", KINDS)
@pytest.mark.parametrize("batch,heads,kv,tokens,d,page,ctx", [
    (1, 4, 2, 300, 128, 64, (200,)), (2, 2, 2, 129, 64, 16, (0, 1)), (1, 8, 1, 256, 32, 0, (333,))])
def test_chunks(batch, heads, kv, tokens, d, page, ctx, dt, kind):
    s = Setup(batch, heads, kv, tokens, d, dt, kind, page, ctx, seed=tokens)
    s.check(*s.run(), rows=(1, 31, 32, 63, 64, 127, 128, 200))


EDGES = (1, 30, 31, 32, 33, 127, 128, 255, 256, 300, 383, 500)


@pytest.mark.parametrize("dt,kind", KINDS)
@pytest.mark.parametrize("batch,d", [(4, 128), (8, 128), (4, 64), (4, 32)])
@pytest.mark.parametrize("masked", [False, True], ids=["causal", "tree"])
def test_many_rows(batch, d, masked, dt, kind):
    # Sizes at which the rule takes 4 and 8 tiles of rows over shared keys.
    ctx = [(300 if d > 32 else 100, 0, 37, 69)[i % 4] for i in range(batch)]
    new = [(512, 500, 257, 1)[i % 4] for i in range(batch)]
    s = Setup(batch, 16, 4, 512, d, dt, kind, 16, ctx, new=new, seed=batch + d)
    mask, seen = tree(batch, 512, 7) if masked else (None, None)
    o, lse = s.run(mask)
    s.check(o, lse, seen, rows=EDGES, heads=(0, 6, 15), seqs=(0, 1, 2, 3))
    assert torch.equal(o, s.run(mask)[0])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch,ctx", [(8, 4096), (2, 8192)])
def test_many_rows_and_splits(batch, ctx, kind):
    lens = [ctx - 700 * i for i in range(batch)]
    s = Setup(batch, 32, 8, 64, 128, "bf16", kind, 64, [max(0, c) for c in lens], seed=batch)
    mask, seen = tree(batch, 64, 2)
    s.check(*s.run(mask), seen, rows=(1, 7, 40), heads=(0, 31), seqs=(0, 1, batch - 1))


@pytest.mark.parametrize("dt,kind", KINDS)
@pytest.mark.parametrize("batch,d", [(4, 64), (4, 128), (8, 128)])
def test_many_rows_hidden_values(batch, d, dt, kind):
    # Not finite in drafts nobody sees, in one that some see, and behind the end.
    t = 512
    s = Setup(batch, 16, 4, t, d, dt, kind, 16, [300] * batch, new=[t - 5] * batch, spare=20, seed=3)
    rng = np.random.default_rng(2)
    one = rng.random((t, t)) < 0.3
    one[:, 200:203] = False
    one[:, 290] = np.arange(t) % 64 == 63
    one[0, 0] = True
    seen = np.stack([one] * batch)
    mask = torch.from_numpy(C.words_of(one).view(np.int64)).cuda()
    bad = [500, 501, 502] + list(range(300 + t - 5, 300 + t + 20))
    for i in range(batch):
        for n, at in enumerate(bad):
            p, r = int(s.table[i, at // 16]), at % 16
            v = (float("nan"), float("inf"), -float("inf"))[n % 3]
            if kind in C.TOP:
                s.cache.k_scale[p, :, r] = v
                s.cache.v_scale[p, :, r] = v
            else:
                s.cache.k[p, :, r] = v
                s.cache.v[p, :, r] = v
    o, lse = s.run(mask)
    s.check(o, lse, seen, rows=EDGES, heads=(0, 15), seqs=(0, batch - 1))
    p, r = int(s.table[0, 590 // 16]), 590 % 16
    if kind in C.TOP:
        s.cache.v_scale[p, :, r] = float("nan")
    else:
        s.cache.v[p, :, r] = float("nan")
    o2, _ = s.run(mask)
    sees = torch.from_numpy(one[:t - 5, 290]).cuda()
    assert torch.isnan(o2[0][:, :t - 5][:, sees]).all()
    assert torch.equal(o2[0][:, :t - 5][:, ~sees], o[0][:, :t - 5][:, ~sees])
    assert torch.equal(o2[1:], o[1:])


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
@pytest.mark.parametrize("tokens", [1, 20])
def test_value_scales_of_every_size(tokens, kind):
    # Value scales from 2^-60 to 2^15 in any order: f16 weights times a scale
    # stay in range.
    s = Setup(1, 8, 2, tokens, 128, "f16", kind, 16, (700,), seed=8)
    p = torch.randint(-60, 16, s.cache.v_scale.shape, generator=torch.Generator().manual_seed(4))
    s.cache.v_scale.copy_(torch.ldexp(torch.ones(()), p))
    s.cache.v_scale[int(s.table[0, 2]), :, 3] = 2.0 ** 15
    o, lse = s.run(out=torch.float32)
    s.check(o, lse)


def test_two_streams():
    # Calls at once on two streams, each with scratch of its own.
    a = Setup(1, 8, 2, 1, 128, "bf16", "bf16", 64, (20000,), seed=1)
    b = Setup(2, 8, 2, 3, 128, "bf16", "e4m3", 64, (15000, 300), seed=2)
    want = [s.run()[0] for s in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s, st in zip((a, b), streams):
            with torch.cuda.stream(st):
                got.append(s.run()[0])
    o = torch.empty_like(a.q)
    rt.tree_attn(a.q, a.cache, a.ctx_len, o, stream=streams[0])
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2])
    assert torch.equal(o, want[0])


def test_a_workspace_of_any_contents():
    s = Setup(1, 8, 2, 2, 128, "bf16", "bf16", 64, (9000,), seed=1)
    want, _ = s.run()
    need = rt.tree_attn_workspace_bytes(rt.tree_attn_desc(s.q, s.cache, s.ctx_len, torch.empty_like(s.q)))
    assert need > 0
    for byte in (0x00, 0xFF, 0x7F, 0x3C):
        ws = torch.full((need + 64,), byte, dtype=torch.uint8, device="cuda")
        for _ in range(3):
            assert torch.equal(s.run(workspace=ws)[0], want)
        assert (ws[need:] == byte).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("d", [128, 64, 80])
@pytest.mark.parametrize("tokens", [1, 6, 40, 150])
def test_ragged(tokens, d, kind):
    # Padded tokens, a sequence without new ones, one that takes no part.
    new = (tokens, 0, max(1, tokens // 2), tokens, 1)
    s = Setup(5, 4, 2, tokens, d, "bf16", kind, 32, (100, 50, 0, -1, 200), new=new, seed=tokens, spare=30)
    s.check(*s.run())
    mask, seen = tree(5, tokens, 3)
    s.check(*s.run(mask), seen)


@pytest.mark.parametrize("kind", ["bf16", "i8"])
@pytest.mark.parametrize("tokens", [1, 16, 140])
def test_rows_that_see_nothing(tokens, kind):
    # No context and an empty mask: o = 0, lse = -inf; one mask of all trees.
    s = Setup(2, 4, 2, tokens, 128, "bf16", kind, 16, (0, 0))
    seen = np.random.default_rng(1).random((tokens, tokens)) < 0.2
    seen[0] = False
    seen[tokens // 2] = False
    mask = torch.from_numpy(C.words_of(seen).view(np.int64)).cuda()
    o, lse = s.run(mask)
    s.check(o, lse, np.stack([seen] * 2))
    assert (o[:, :, 0] == 0).all() and torch.isinf(lse[:, :, 0]).all()


@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3", "i8"])
@pytest.mark.parametrize("heads,tokens,d", [(4, 1, 128), (4, 20, 128), (8, 70, 64), (2, 9, 80), (4, 150, 128)])
def test_hidden_rows_do_not_matter(heads, tokens, d, kind):
    # Infinities and NaN in hidden drafts, behind the last key, and their scales.
    dt = kind if kind in ("bf16", "f16") else "bf16"
    s = Setup(1, heads, 2, tokens, d, dt, kind, 16, (90,), new=(max(1, tokens - 3),), spare=70, seed=5)
    live = s.new[0]
    rng = np.random.default_rng(2)
    seen = rng.random((1, tokens, tokens)) < 0.5
    seen[0, :, ::3] = False  # every third draft is seen by nobody but (some) itself
    seen[0, 0, 0] = True
    mask = torch.from_numpy(C.words_of(seen).view(np.int64)).cuda()
    bad = [90 + j for j in range(live) if j % 3 == 0 and j > 0] + list(range(90 + live, 90 + tokens + 70))
    for n, at in enumerate(bad):
        p, r = int(s.table[0, at // 16]), at % 16
        v = (float("nan"), float("inf"), -float("inf"))[n % 3]
        if kind in C.TOP:
            s.cache.k_scale[p, :, r] = v
            s.cache.v_scale[p, :, r] = v
            if kind == "e4m3":
                s.cache.k.view(torch.uint8)[p, :, r] = 0x7F
                s.cache.v.view(torch.uint8)[p, :, r] = 0xFF
        else:
            s.cache.k[p, :, r] = v
            s.cache.v[p, :, r] = v
    s.check(*s.run(mask), seen)


@pytest.mark.parametrize("tokens", [3, 70, 150])
def test_hidden_to_some(tokens):
    # A NaN value that one drafted token sees and the others do not: that one
    # is NaN, the others are as without it.
    s = Setup(1, 4, 2, tokens, 128, "bf16", "bf16", 16, (90,), seed=5)
    mask, seen = tree(1, tokens, 4)
    who = tokens - 1
    p, r = int(s.table[0, (90 + who) // 16]), (90 + who) % 16
    s.cache.v[p, :, r] = float("nan")
    o, lse = s.run(mask)
    assert torch.isnan(o[:, :, who]).all() and not torch.isnan(lse).any()
    rest = o[:, :, :who].float()
    assert torch.isfinite(rest).all()
    s.cache.v[p, :, r] = 1.0
    o2, _ = s.run(mask)
    assert torch.equal(o2[:, :, :who], o[:, :, :who])


def test_splits_give_the_same_sums():
    # Unsplit and split, and a hint far off: within the tolerance of both.
    s = Setup(2, 4, 1, 3, 128, "bf16", "bf16", 64, (9000, 700), seed=9)
    outs = [s.run(workspace=False), s.run(), s.run(max_ctx=1), s.run(max_ctx=1 << 30)]
    for o, l in outs:
        s.check(o, l)
    assert torch.equal(outs[1][0], s.run()[0])  # the same bits again


@pytest.mark.parametrize("tokens", [1, 40])
def test_bad_pages_are_not_seen(tokens):
    # A page number that is none hides its keys; so does a length behind the capacity.
    s = Setup(1, 4, 2, tokens, 128, "bf16", "bf16", 16, (100,), seed=3)
    s.cache.block_table[0, 1] = -1
    s.cache.block_table[0, 3] = 1 << 20
    o, lse = s.run()
    k, v = s.rows(0)
    vis = np.ones((tokens, 100 + tokens), bool)
    vis[:, 100:] = np.tril(np.ones((tokens, tokens), bool))
    vis[:, 16:32] = vis[:, 48:64] = False
    wo, wl, wa = C.attention(s.q[0, 0].double().cpu().numpy(), k[0], v[0], vis, 128 ** -0.5)
    h = 2.0 ** -8
    assert (np.abs(o[0, 0].double().cpu().numpy() - wo) <= h * np.abs(wo) + (h + 2.0 ** -12) * wa).all()
    assert np.abs(lse[0, 0].double().cpu().numpy() - wl).max() <= 2.0 ** -11
    s.ctx_len.fill_(1 << 30)  # every key of the cache is context, no draft exists
    o, lse = s.run()
    assert torch.isfinite(o).all() and (o != 5.0).any()


@pytest.mark.parametrize("tokens", [1, 20, 150])
def test_f32_output_scale_and_layouts(tokens):
    s = Setup(2, 6, 3, tokens, 64, "f16", "e4m3", 32, (70, 3), seed=2, slot_first=True)
    o, lse = s.run(out=torch.float32, sm_scale=0.3)
    s.check(o, lse, scale=0.3)
    o2, none = s.run(out=torch.float32, sm_scale=0.3, lse=False)
    assert none is None and torch.equal(o, o2)


@pytest.mark.parametrize("batch,tokens,d,ctx,dt,kind", [
    (1, 1, 128, 4000, "bf16", "bf16"), (2, 33, 64, 1500, "f16", "i8"), (1, 150, 128, 3001, "bf16", "e4m3"),
    (4, 300, 128, 64, "bf16", "bf16"), (2, 3, 80, 700, "f16", "f16"), (2, 40, 32, 0, "bf16", "bf16")])
def test_output_in_place_of_the_queries(batch, tokens, d, ctx, dt, kind):
    s = Setup(batch, 8, 2, tokens, d, dt, kind, 16, [ctx] * batch, seed=6)
    want, lse = s.run()
    q = s.q.clone(memory_format=torch.preserve_format)
    assert q.stride() == s.q.stride()
    l = torch.empty_like(lse)
    rt.tree_attn(q, s.cache, s.ctx_len, q, lse=l)
    assert torch.equal(q, want) and torch.equal(l, lse)


def test_refuses_workspaces_it_cannot_write():
    s = Setup(1, 32, 8, 1, 128, "bf16", "bf16", 64, (30000,), seed=6)
    o = torch.empty_like(s.q)
    need = rt.tree_attn_workspace_bytes(rt.tree_attn_desc(s.q, s.cache, s.ctx_len, o))
    assert need > 0
    one = torch.empty(1, dtype=torch.uint8, device="cuda")
    for ws in (torch.empty(need, dtype=torch.uint8), one.expand(need)):
        with pytest.raises(ValueError, match="workspace must be a contiguous tensor"):
            rt.tree_attn(s.q, s.cache, s.ctx_len, o, workspace=ws)
    with pytest.raises(ValueError, match="workspace of"):
        rt.tree_attn(s.q, s.cache, s.ctx_len, o, workspace=one)


def test_long_cache_beyond_32_bits():
    # Keys of one sequence over 6 GB of cache.
    pages, size, d = 3, 1 << 20, 128
    k = torch.zeros((pages, 1, size, 1024), dtype=torch.bfloat16, device="cuda")[..., :d]
    v = torch.zeros((pages, 1, size, 1024), dtype=torch.bfloat16, device="cuda")[..., :d]
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    cache = rt.KvCache(k, v, block_table=table)
    q = torch.ones((1, 2, 1, d), dtype=torch.bfloat16, device="cuda")
    at = 2 * size + 5  # page 1, the last of the sequence
    k[1, 0, 5] = 8.0
    v[1, 0, 5] = 3.0
    k[2, 0, 77] = 8.0
    v[2, 0, 77] = 1.0
    o = torch.empty_like(q)
    rt.tree_attn(q, cache, torch.tensor([at], dtype=torch.int32, device="cuda"), o)
    # Two keys of score 8 * 128 / sqrt(128) = 90.5 and two million of 0.
    assert torch.allclose(o.float(), torch.full_like(o.float(), 2.0), atol=2.0 ** -7)


def test_graph_replay_two_graphs_and_streams():
    # A decode step captured: rope, append, attention, with lengths that grow
    # between replays; the workspaces of two graphs are their own.
    s = Setup(2, 8, 2, 1, 128, "bf16", "e4m3", 64, (3000, 200), spare=40, seed=6)
    table = rt.rope_table(128)
    k_new, v_new = randn((2, 2, 1, 128), 31).to(torch.bfloat16), randn((2, 2, 1, 128), 32).to(torch.bfloat16)

    def step(o):
        q2, k2 = torch.empty_like(s.q), torch.empty_like(k_new)
        rt.rope(s.q, q2, None, table, k=k_new, k_out=k2, start=s.ctx_len)
        rt.kv_append(k2, v_new, s.cache, s.ctx_len)
        rt.tree_attn(q2, s.cache, s.ctx_len, o)

    outs = [torch.empty_like(s.q) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(outs[0])
    torch.cuda.synchronize()
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(o)
        graphs.append(g)
    for n in range(4):
        s.ctx_len += 1
        want = torch.empty_like(s.q)
        step(want)
        for o in outs:
            o.fill_(5.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), n


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "i8"])
def test_a_drafting_step(kind):
    """The run of calls a serving program makes: masks of the drafted tree,
    rotation to ctx + depth, append, attention; then the accepted branch
    appended again in its final place and one plain token after it."""
    b, heads, kv, t, d = 2, 8, 2, 12, 64
    s = Setup(b, heads, kv, t, d, "bf16", kind, 16, (50, 9), spare=20, seed=4)
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 3, 3, 5, 6, 7, 8], [-1, -1, 0, 1, 2, 2, 3, 4, 4, 6, 7, 9]],
                           dtype=torch.int32, device="cuda")
    mask, depth = rt.tree_mask(parents)
    seen = np.stack([C.ancestors(p)[0] for p in parents.cpu().numpy()])
    table = rt.rope_table(d)
    q, k, v = s.q, *(randn((b, kv, t, d), i).to(torch.bfloat16) for i in (61, 62))
    qr, kr = torch.empty_like(q), torch.empty_like(k)
    rt.rope(q, qr, depth, table, k=k, k_out=kr, start=s.ctx_len)
    rt.kv_append(kr, v, s.cache, s.ctx_len)
    o = torch.full_like(q, 5.0)
    rt.tree_attn(qr, s.cache, s.ctx_len, o, mask=mask)
    s.q = qr
    s.check(o, None, seen)
    # Accept the branch 0 -> 1 -> 3 -> 6 and 1 -> 3 -> 6: the same rows again.
    path = torch.tensor([[0, 1, 3, 6], [1, 3, 6, 9]], device="cuda")
    take = path[:, None, :, None].expand(b, kv, 4, d)
    rt.kv_append(kr.gather(2, take), v.gather(2, take), s.cache, s.ctx_len)
    s.tokens, s.new = 4, [4, 4]
    s.q = qr.gather(2, path[:, None, :, None].expand(b, heads, 4, d))
    o2 = torch.full_like(s.q, 5.0)
    rt.tree_attn(s.q, s.cache, s.ctx_len, o2)
    s.check(o2, None)
    # What a token saw as a branch it sees as a chain: the same keys.
    both = o.gather(2, path[:, None, :, None].expand(b, heads, 4, d)).float()
    assert (both - o2.float()).abs().max() <= 2.0 ** -5 * both.abs().max()


@pytest.mark.parametrize("batch,heads,d", [((1 << 23) + 5, 1, 32), (1 << 18, 40, 16)])
def test_millions_of_sequences(batch, heads, d):
    # More query rows than a launch has workgroups of 512 threads: one key each,
    # whose value is the result.
    k = torch.ones((batch, heads, 1, d), dtype=torch.bfloat16, device="cuda")
    v = randn((batch, 1, 1, d), 4).to(torch.bfloat16).expand(batch, heads, 1, d).contiguous()
    o = torch.empty_like(k)
    rt.tree_attn(k, rt.KvCache(k, v), torch.zeros(batch, dtype=torch.int32, device="cuda"), o)
    assert torch.equal(o, v)
