"""frisk_kv_pages, frisk_kv_copy_pages and frisk_kv_compact against plain python
and indexing: every comparison is of bits."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import serving_ops as S
from tests.gpu_util import Guarded

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8}


def ints(x, dtype=torch.int32):
    return torch.tensor(np.asarray(x).tolist(), dtype=dtype, device="cuda")


# ---- tables ------------------------------------------------------------------------


def step(table, keep, want, page, pages, parent=None, held=None):
    """One call, its outputs between sentinels."""
    b, n = len(table), len(table[0])
    out, src, dst, rows = (Guarded(s, torch.int32) for s in ((b, n), (b,), (b,), (b,)))
    lacking = Guarded((1,), torch.int32)
    rt.kv_pages(ints(table), ints(keep), None if want is None else ints(want), page, pages,
                parent=None if parent is None else ints(parent), held=None if held is None else ints(held, torch.uint8),
                out=out.t, src=src.t, dst=dst.t, rows=rows.t, lacking=lacking.t)
    assert all(g.guards_intact() for g in (out, src, dst, rows, lacking))
    return [g.t.tolist() for g in (out, src, dst, rows)] + [int(lacking.t)]


def random_tables(rng, b, n, page, pages, wrong=0.0):
    order = rng.permutation(max(pages, b * n))[:b * n].reshape(b, n)
    table = np.where(order < pages, order, -1)
    table[rng.random((b, n)) < wrong] = rng.choice([-1, -7, pages, 2 ** 31 - 1, -2 ** 31])
    return table.astype(np.int64).tolist()


CASES = [(1, 1, 1, 1), (1, 5, 16, 3), (3, 4, 4, 40), (8, 17, 16, 33), (5, 70, 1, 400), (64, 130, 64, 9000),
         (200, 9, 16, 1801), (1500, 3, 2, 5000), (33, 64, 128, 4096)]


@pytest.mark.parametrize("b,n,page,pages", CASES)
def test_tables(b, n, page, pages):
    rng = np.random.default_rng(b + n)
    for trial in range(4):
        table = random_tables(rng, b, n, page, pages, 0.1 * (trial == 3))
        keep = rng.integers(0, n * page + 1, b).tolist()
        want = (np.array(keep) + rng.integers(-2, 3 * page, b)).tolist()
        parent = None if trial == 0 else rng.integers(-1, b + (trial == 2), b).tolist()
        held = rng.random(pages) < 0.2 if trial == 2 else None
        got = step(table, keep, want, page, pages, parent, held)
        assert got == list(S.next_table(table, keep, want, page, pages, parent, held)), trial


@pytest.mark.parametrize("n,page", [(1300, 4), (513, 1), (512, 16), (1024, 2), (515, 8)])
def test_long_tables(n, page):
    # More entries than four rows' lanes take at once, some of them no page.
    rng = np.random.default_rng(n)
    for wrong in (0.0, 0.01):
        table = random_tables(rng, 7, n, page, 8 * n, wrong)
        keep = [0, n * page, n * page - 1, 512 * page, min(513, n) * page, 1, int(rng.integers(0, n * page))]
        want = [n * page, n * page, 0, 600 * page, n * page, 3 * page, n * page]
        args = (table, keep, want, page, 8 * n, [1, 1, 2, 2, 5, 6, 0])
        assert step(*args) == list(S.next_table(*args))


def test_more_new_pages_than_are_listed():
    # 4000 entries of empty rows out of 6000 pages, then out of 3000.
    for pages in (6000, 3000):
        held = np.random.default_rng(5).random(pages) < 0.1
        args = ([[-1] * 100] * 40, [0] * 40, [800] * 40, 8, pages, None, held)
        assert step(*args) == list(S.next_table(*args))


def test_many_sequences_continue_one():
    # All of one parent within a page: the first writes it, the others copy.
    table = random_tables(np.random.default_rng(1), 300, 4, 8, 3000)
    for keep in (9, 16, 32, 0):
        args = (table, [keep] * 300, [32] * 300, 8, 3000, [7] * 300)
        got = step(*args)
        assert got == list(S.next_table(*args))
        assert sum(s >= 0 for s in got[1]) == (299 if keep == 9 else 0)


def test_a_table_that_shares_pages_already():
    # Rows that share their last page without being forks of one another; one keeps it whole.
    table = [[4, 9], [4, 9], [4, 9], [3, 9]]
    for keep in ([5, 5, 5, 5], [5, 8, 5, 5], [5, 5, 5, 8], [1, 2, 3, 4], [4, 4, 4, 4]):
        args = (table, keep, [8] * 4, 4, 12)
        assert step(*args) == list(S.next_table(*args))


def test_more_rows_than_threads_share_a_page():
    table = [[5, 1]] * 2100
    args = (table, [3] * 2100, [8] * 2100, 4, 3000)
    assert step(*args) == list(S.next_table(*args))


def test_lengths_out_of_range():
    table = random_tables(np.random.default_rng(2), 6, 3, 4, 30)
    args = (table, [-1, 2 ** 31 - 1, 13, 0, 5, 12], [9, 2 ** 31 - 1, -5, 0, 2 ** 31 - 1, 0], 4, 30)
    assert step(*args) == list(S.next_table(*args))
    args = (table, [4] * 6, None, 4, 30, [0, 6, -1, 2 ** 31 - 1, -2 ** 31, 5])
    assert step(*args) == list(S.next_table(*args))


def test_the_largest_tables():
    # LDS for 2^19 pages; entries far behind the first words.
    pages, b = 1 << 19, 64
    rng = np.random.default_rng(3)
    table = rng.integers(0, pages, (b, 40)).tolist()
    held = np.ones(pages, bool)
    held[[3, 70000, pages - 1, pages - 33]] = False
    args = (table, [40] * b, [44] * b, 1, pages, None, held)
    args = (table, [30] * b, [32] * b, 1, pages, None, held)
    got = step(*args)
    assert got == list(S.next_table(*args)) and got[4] > 0
    with pytest.raises(ValueError, match="more pages"):
        step(table, [1] * b, None, 1, 1 << 20)


def test_strided_tables_and_made_outputs():
    rng = np.random.default_rng(4)
    wide = ints(random_tables(rng, 5, 12, 4, 80))
    keep = ints([9, 3, 16, 0, 7])
    out, src, dst, rows, lacking = rt.kv_pages(wide[:, 3:9], keep, keep + 5, 4, 80, parent=ints([1, 1, 2, 3, 0]))
    want = S.next_table(wide[:, 3:9].tolist(), keep.tolist(), (keep + 5).tolist(), 4, 80, [1, 1, 2, 3, 0])
    assert [out.tolist(), src.tolist(), dst.tolist(), rows.tolist(), int(lacking)] == list(want)
    with pytest.raises(ValueError, match="an output overlaps"):
        rt.kv_pages(wide, keep, None, 4, 80, out=wide)
    with pytest.raises(ValueError, match="held"):
        rt.kv_pages(wide, keep, None, 4, 80, held=torch.zeros(79, dtype=torch.bool, device="cuda"))


def test_interleaved_tables():
    rng = np.random.default_rng(6)
    both = torch.full((5, 2, 6), -7, dtype=torch.int32, device="cuda")
    both[:, 0] = ints(random_tables(rng, 5, 6, 4, 80))
    table, out, keep = both[:, 0], both[:, 1], ints([9, 3, 16, 0, 7])
    before = table.tolist()
    rt.kv_pages(table, keep, keep + 5, 4, 80, out=out)
    assert out.tolist() == S.next_table(before, keep.tolist(), (keep + 5).tolist(), 4, 80)[0]
    assert table.tolist() == before
    with pytest.raises(ValueError, match="an output overlaps"):
        rt.kv_pages(both[:, 0], keep, None, 4, 80, out=both.view(5, 12)[:, 5:11])


# ---- rows and pages of a cache --------------------------------------------------------


def cache_of(pages, kv, size, d, kind, table=None, slot_first=False, block=1, seed=1):
    """A cache of random bytes (every bit pattern, NaN among them)."""
    gen = torch.Generator().manual_seed(seed)
    es = torch.empty((), dtype=DT[kind]).element_size()
    shape = (pages, size, kv, d * es) if slot_first else (pages, kv, size, d * es)

    def tensor():
        t = torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8).cuda().view(DT[kind])
        return t.transpose(1, 2) if slot_first else t

    scales = [None, None]
    if es == 1:
        scales = [torch.rand((pages, kv, -(-size // block)), generator=gen).cuda() for _ in range(2)]
    return rt.KvCache(tensor(), tensor(), *scales, table, scale_block=block)


def tensors(cache):
    return [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


def bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16 if t.element_size() == 2 else torch.int32)


def same(got, want):
    return all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))


KINDS = [("bf16", 128, False), ("f16", 80, True), ("e4m3", 64, False), ("i8", 16, True), ("bf16", 256, False),
         ("i8", 256, False), ("e4m3", 48, True)]


@pytest.mark.parametrize("kind,d,slot_first", KINDS)
@pytest.mark.parametrize("page", [0, 1, 8, 64])
def test_compact(kind, d, slot_first, page):
    b, kv, t = 5, 3, 150
    rng = np.random.default_rng(d + page)
    ctx = [0, 13, 7, -1, 40]
    cap = 40 + t
    if page:
        per = -(-cap // page)
        table = rng.permutation(b * per + 2)[:b * per].reshape(b, per)
        table[1, 20 // page] = -1  # a page that is none
        cache = cache_of(b * per + 2, kv, page, d, kind, ints(table), slot_first)
    else:
        table, cache = None, cache_of(b, kv, cap, d, kind, None, slot_first)
    path = np.full((b, t), -1)
    count = [t, 90, 9, 5, 3]
    path[0] = np.arange(t)                                     # nothing moves
    path[1, :90] = np.sort(rng.choice(t, 90, replace=False))   # overlapping moves, over several batches
    path[2, :9] = [0, 1, 5, 5, 4, 3, 200, 7, 149]              # ends at 3 (below its place); 200: behind the cache or not
    path[3, :5] = [1, 2, 3, 4, 5]                              # takes no part
    path[4, :3] = [2, 149, 2 ** 31 - 1]
    want = tensors(cache)

    def where(i, n):
        if n >= (len(table[i]) * page if page else cap):
            return None
        if not page:
            return i, n
        return (int(table[i][n // page]), n % page) if table[i][n // page] >= 0 else None

    before = [w.clone() for w in want]
    for i in range(b):
        if ctx[i] < 0:
            continue
        for j in range(min(count[i], t)):
            if path[i, j] < j:
                break
            a, z = where(i, ctx[i] + int(path[i, j])), where(i, ctx[i] + j)
            if a and z:
                for w, x in zip(want, before):
                    w[z[0], :, z[1]] = x[a[0], :, a[1]]  # (what lay there before the call)
    wide = torch.full((b, t + 9), -9, dtype=torch.int32, device="cuda")
    wide[:, 4:4 + t] = ints(path)
    rt.kv_compact(cache, wide[:, 4:4 + t], ints(ctx), ints(count))
    assert same(tensors(cache), want)
    rt.kv_compact(cache, ints(path), ints(ctx), ints([0, -3, 0, 7, -2 ** 31]))
    assert same(tensors(cache), want)


@pytest.mark.parametrize("kind,d,slot_first", KINDS)
@pytest.mark.parametrize("size,block", [(1, 1), (16, 1), (64, 16), (128, 128), (300, 32)])
def test_copy_pages(kind, d, slot_first, size, block):
    if kind in ("bf16", "f16"):
        block = 1
    pages, kv = 23, 3
    rng = np.random.default_rng(size + d)
    order = rng.permutation(pages)
    src, dst = order[:9].tolist(), order[9:18].tolist()
    src[2], dst[3] = -1, pages
    src[4], dst[5] = 2 ** 31 - 1, -2 ** 31
    src[6] = dst[6] = int(order[20])
    for rows in (None, [size, 1, size, size, 3, 2, 1, max(size - 1, 0), size + 5], [0, -4] + [size // 2] * 7):
        cache = cache_of(pages, kv, size, d, kind, None, slot_first, block, seed=size)
        want = tensors(cache)
        for i, (a, z) in enumerate(zip(src, dst)):
            n = size if rows is None else max(0, min(rows[i], size))
            if not (0 <= a < pages and 0 <= z < pages):
                continue
            for w in want:
                m = n if w.dim() == 4 else -(-n // block)
                w[z, :, :m] = w[a, :, :m].clone()
        rt.kv_copy_pages(cache, ints(src), ints(dst), rows=None if rows is None else ints(rows))
        assert same(tensors(cache), want)


def test_offsets_beyond_32_bits():
    # Two heads 2^31 + elements apart; the pages of a long cache.
    d, size = 128, 32
    k = torch.zeros((1 << 32) + (1 << 20), dtype=torch.uint8, device="cuda").view(torch.int8)
    v = torch.zeros_like(k)
    shape, st = (40, 2, size, d), (size * d, (1 << 32) - 4096, d, 1)
    scale = [torch.rand(40, 2, size, device="cuda") for _ in range(2)]
    cache = rt.KvCache(k.as_strided(shape, st), v.as_strided(shape, st), *scale)
    for x in (cache.k, cache.v):
        x[3] = torch.randint(-127, 128, (2, size, d), device="cuda", dtype=torch.int8)
    rt.kv_copy_pages(cache, ints([3]), ints([39]))
    for x in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        assert torch.equal(x[39], x[3])
    cache.k[0, 1, 9] = 5
    rt.kv_compact(cache, ints([[0, 9]] + [[0, 0]] * 39), ints([0] + [-1] * 39), ints([2] * 40))
    assert (cache.k[0, 1, 1] == 5).all() and (cache.k[0, 0, 1] == 0).all()


def test_graph_and_stream():
    cache = cache_of(12, 2, 16, 64, "bf16", ints([[0, 1], [2, 3]]))
    path, ctx, count = ints([[0, 3, 5], [2, 4, 6]]), ints([4, 10]), ints([3, 2])
    src, dst = ints([0, 2]), ints([7, 9])
    keep = ints([5, 20])
    out = torch.empty(2, 2, dtype=torch.int32, device="cuda")
    first = tensors(cache)

    def work(stream=None):
        rt.kv_compact(cache, path, ctx, count, stream=stream)
        rt.kv_copy_pages(cache, src, dst, rows=count, stream=stream)
        return rt.kv_pages(cache.block_table, keep, None, 16, 12, out=out, stream=stream)

    made = [x.tolist() for x in work()]
    want = tensors(cache)

    def reset():
        for t, x in zip((cache.k, cache.v), first):
            t.copy_(x)
        out.zero_()

    reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = work(side)
    side.synchronize()
    assert [x.tolist() for x in got] == made
    assert same(tensors(cache), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for _ in range(3):
        reset()
        graph.replay()
        assert [x.tolist() for x in got] == made and same(tensors(cache), want)


def test_refuses_wrong_arguments():
    cache = cache_of(4, 1, 16, 16, "i8", ints([[0], [1]]), block=16)
    with pytest.raises(ValueError, match="share scales"):
        rt.kv_compact(cache, ints([[0], [0]]), ints([1, 1]), ints([1, 1]))
    plain = cache_of(4, 1, 16, 16, "i8", ints([[0], [1]]))
    with pytest.raises(ValueError, match="rows for a batch"):
        rt.kv_compact(plain, ints([[0]]), ints([1]), ints([1]))
    with pytest.raises(ValueError, match="path"):
        rt.kv_compact(plain, ints([[0], [0]], torch.int64), ints([1, 1]), ints([1, 1]))
    with pytest.raises(ValueError, match="dst"):
        rt.kv_copy_pages(plain, ints([0, 1]), ints([2]))
    with pytest.raises(ValueError, match="scales must"):
        rt.KvCache(plain.k, plain.v, plain.k_scale, plain.v_scale, scale_block=16)
    with pytest.raises(ValueError, match="scale_block"):
        rt.KvCache.empty(1, 1, 16, 16, torch.bfloat16, scale_block=16)
