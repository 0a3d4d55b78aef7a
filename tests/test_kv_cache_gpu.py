"""frisk_kv_append, frisk_kv_read and frisk_tree_mask against numpy: codes and
scales are exact (include/frisk_hip.h defines them), so every comparison is of
bits."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import cache_ops as C
from tests.gpu_util import Guarded, decode, randn

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8}
FILL = 0x33


def make_cache(pages, kv, size, d, kind, table=None, slot_first=False):
    """A cache of FILL bytes; slot_first: [pages, page_size, kv_heads, d] in memory."""
    shape = (pages, size, kv, d) if slot_first else (pages, kv, size, d)
    es = torch.empty((), dtype=DT[kind]).element_size()

    def tensor():
        t = torch.full(shape[:3] + (shape[3] * es,), FILL, dtype=torch.uint8, device="cuda").view(DT[kind])
        return t.transpose(1, 2) if slot_first else t

    scale = [torch.full((pages, kv, size), 7.0, device="cuda") for _ in range(2)] if es == 1 else [None] * 2
    return rt.KvCache(tensor(), tensor(), *scale, table)


def expected(x, kind):
    """What a row reads back as, fp64 (before the output's rounding), scales."""
    if kind not in C.TOP:
        return x, None
    codes, scale = C.quantise(x, kind)
    # The kernel multiplies in f32, exact for the rounding that follows it.
    return (codes.astype(np.float32) * scale[..., None]).astype(np.float64), scale


def same(got, want):
    """Equal values, NaN equal to NaN."""
    np.testing.assert_array_equal(np.asarray(got.cpu().float() if torch.is_tensor(got) else got),
                                  np.asarray(want.float() if torch.is_tensor(want) else want))


def round_to(x, dt):
    return torch.from_numpy(x).float().to(DT[dt])


CASES = [
    # batch, tokens, kv heads, head_dim, dtype, kind, page (0: none), slot first
    (2, 5, 2, 128, "bf16", "e4m3", 16, False), (1, 1, 1, 16, "f16", "i8", 0, False),
    (3, 70, 3, 64, "f16", "e4m3", 32, True), (2, 33, 5, 80, "bf16", "i8", 1, False),
    (2, 9, 2, 256, "bf16", "i8", 64, False), (4, 17, 1, 32, "f16", "f16", 8, True),
    (2, 3, 2, 48, "bf16", "bf16", 0, False), (1, 1000, 4, 128, "bf16", "e4m3", 0, False)]


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("b,t,kv,d,dt,kind,page,slot_first", CASES)
def test_append_and_read(b, t, kv, d, dt, kind, page, slot_first, ragged):
    rng = np.random.default_rng(b * 1000 + t)
    ctx = rng.integers(0, 40, b)
    new = rng.integers(0, t + 1, b) if ragged else np.full(b, t)
    if ragged:
        ctx[-1] = -1 if b > 2 else ctx[-1]
        new[0] = t
    cap = 40 + t
    table, pages, size = None, b, cap
    if page:
        per = -(-cap // page)
        pages, size = b * per + 2, page
        order = rng.permutation(pages)[:b * per].reshape(b, per)
        table = torch.from_numpy(order.astype(np.int32)).cuda()
    cache = make_cache(pages, kv, size, d, kind, table, slot_first)
    # Rows of very different sizes, a zero row and one at the type's top.
    x = {n: randn((b, t, kv, d), 11 + i) * torch.exp(4 * randn((b, t, kv, 1), 21 + i))
         for i, n in enumerate("kv")}
    x["k"][0, 0] = 0
    x["v"][0, 0, 0, :4] = torch.tensor([65504.0, -65504.0, 32752.0, 146.0])
    x = {n: v.to(DT[dt]).transpose(1, 2) for n, v in x.items()}
    ctx_len = torch.from_numpy(ctx.astype(np.int32)).cuda()
    new_len = torch.from_numpy(new.astype(np.int32)).cuda() if ragged else None
    rt.kv_append(x["k"], x["v"], cache, ctx_len, new_len=new_len)
    back = {n: torch.full((b, kv, t, d), 5.0, dtype=DT[dt], device="cuda") for n in "kv"}
    rt.kv_read(cache, back["k"], back["v"], ctx_len, new_len=new_len)
    torch.cuda.synchronize()
    for n, tensor, scales in (("k", cache.k, cache.k_scale), ("v", cache.v, cache.v_scale)):
        raw = tensor.contiguous().view(torch.uint8).cpu().numpy().reshape(pages, kv, size, -1)
        touched = np.zeros((pages, size), bool)
        xd = x[n].double().cpu().numpy()
        got = back[n].cpu()
        for i in range(b):
            live = new[i] if ctx[i] >= 0 else 0
            assert (got[i, :, live:] == 5.0).all()
            if not live:
                continue
            want, scale = expected(xd[i, :, :live], kind)
            same(got[i, :, :live], round_to(want, dt))
            for j in range(live):
                at = int(ctx[i]) + j
                p, r = (int(table[i, at // page]), at % page) if page else (i, at)
                touched[p, r] = True
                if scale is not None:
                    same(scales[p, :, r], scale[:, j])
                    codes = decode(tensor[p, :, r].contiguous()).astype(np.float64)
                    same(codes, C.quantise(xd[i, :, j], kind)[0])
                else:
                    same(tensor[p, :, r], x[n][i, :, j].cpu())
        assert (raw.transpose(0, 2, 1, 3)[~touched] == FILL).all(), "a slot outside the call was written"
        if scales is not None:
            assert (scales.cpu().numpy().transpose(0, 2, 1)[~touched] == 7.0).all()


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_every_quotient(dt, kind):
    # Rows whose largest value takes every significand, against all others:
    # ties and near ties of the rounding among them.
    m = 256 if dt == "bf16" else 2048
    a = torch.arange(m // 2, m, dtype=torch.float32)
    x = torch.zeros(len(a), 64)
    gen = torch.Generator().manual_seed(3)
    x[:, 1:] = torch.randint(1, m, (len(a), 63), generator=gen) * 0.5 ** torch.randint(0, 9, (len(a), 63), generator=gen)
    x = torch.minimum(x, a[:, None])
    x[:, 0] = a
    x = x * torch.where(torch.rand(x.shape, generator=gen) < 0.5, -1.0, 1.0)
    x = (x / m).to(DT[dt])[None, None].cuda()
    n = x.shape[2]
    cache = make_cache(1, 1, n, 64, kind)
    rt.kv_append(x, x, cache, torch.zeros(1, dtype=torch.int32, device="cuda"))
    codes, scale = C.quantise(x[0].double().cpu().numpy(), kind)
    assert np.array_equal(decode(cache.k[0]).astype(np.float64), codes)
    assert np.array_equal(cache.v_scale[0].cpu().numpy(), scale)


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_extremes(kind):
    # The type's smallest and largest rows keep finite scales; rows with an
    # infinity or NaN read back as NaN and touch no other row.
    x = torch.zeros(1, 1, 6, 32, dtype=torch.bfloat16, device="cuda")
    x[0, 0, 0, 3] = 9.2e-41
    x[0, 0, 1] = 3.3895313892515355e38
    x[0, 0, 2, 5] = float("inf")
    x[0, 0, 3, 6] = float("nan")
    x[0, 0, 4] = 1.5
    cache = make_cache(1, 1, 6, 32, kind)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    rt.kv_append(x, x, cache, zero)
    k, v = torch.empty_like(x), torch.empty_like(x)
    rt.kv_read(cache, k, v, zero)
    assert torch.equal(k.view(torch.int16), v.view(torch.int16)) or torch.isnan(k[0, 0, 2:4]).all()
    assert torch.isnan(k[0, 0, 2:4]).all() and torch.isnan(cache.k_scale[0, 0, 2:4]).all()
    # Below 2^-126 top the step is the smallest scale times the code's.
    assert (k[0, 0, 0].float().abs() <= 9.2e-41 + 2.0 ** -127).all()
    assert torch.equal(k[0, 0, 1], x[0, 0, 1]) and torch.equal(k[0, 0, 4:], x[0, 0, 4:])


def test_bad_pages_and_capacity():
    # Pages that are none, and keys behind the capacity: not written, not read.
    table = torch.tensor([[3, -1, 99, 0]], dtype=torch.int32, device="cuda")
    cache = make_cache(5, 2, 4, 32, "e4m3", table)
    x = randn((1, 2, 19, 32), 1).to(torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    rt.kv_append(x, x, cache, zero)
    k, v = torch.full_like(x, 5.0), torch.full_like(x, 5.0)
    rt.kv_read(cache, k, v, zero)
    torch.cuda.synchronize()
    live = [0, 1, 2, 3, 12, 13, 14, 15]
    rest = [i for i in range(19) if i not in live]
    want, _ = expected(x.double().cpu().numpy(), "e4m3")
    assert torch.equal(k.cpu()[:, :, live], round_to(want, "bf16")[:, :, live])
    assert (k[:, :, rest] == 5.0).all() and (v[:, :, rest] == 5.0).all()
    raw = cache.k.view(torch.uint8)
    assert (raw[[1, 2, 4]] == FILL).all()


def test_keys_and_values_of_one_buffer():
    """k and v side by side in one tensor, and their scales: rows that never meet."""
    b, t, kv, d, page = 2, 37, 3, 64, 16
    x = torch.randn((2, b, kv, t, d), generator=torch.Generator().manual_seed(5)).cuda().bfloat16()
    table = torch.arange(2 * 3, dtype=torch.int32, device="cuda").flip(0).reshape(2, 3)
    start = torch.zeros(b, dtype=torch.int32, device="cuda")
    for dt in (torch.bfloat16, torch.int8):
        buf = torch.zeros((6, page, 2, kv, d), dtype=dt, device="cuda")
        scales = torch.zeros((6, page, 2, kv), device="cuda")
        k, v = (buf[:, :, i].transpose(1, 2) for i in (0, 1))
        ks, vs = (scales[:, :, i].transpose(1, 2) for i in (0, 1)) if dt == torch.int8 else (None, None)
        both = rt.KvCache(k, v, ks, vs, table)
        apart = rt.KvCache.empty(6, kv, page, d, dt, block_table=table)
        outs = []
        for cache in (both, apart):
            rt.kv_append(x[0], x[1], cache, start)
            out = torch.zeros_like(x)
            rt.kv_read(cache, out[0], out[1], start)
            outs.append(out)
        assert torch.equal(outs[0], outs[1])
        assert dt == torch.int8 or torch.equal(outs[0], x)


def test_offsets_beyond_32_bits():
    # A sequence's page 5 GB into the cache.
    pages, size = 1300, 4096
    k = torch.empty((pages, 1, size, 1024), dtype=torch.int8, device="cuda")[..., :64]
    v = torch.empty((pages, 1, size, 1024), dtype=torch.int8, device="cuda")[..., :64]
    ks, vs = (torch.empty((pages, 1, size), device="cuda") for _ in range(2))
    table = torch.tensor([[1299], [0]], dtype=torch.int32, device="cuda")
    cache = rt.KvCache(k, v, ks, vs, table)
    x = randn((2, 1, 10, 64), 2).to(torch.float16)
    ctx = torch.tensor([4080, 0], dtype=torch.int32, device="cuda")
    rt.kv_append(x, x, cache, ctx)
    a, b = torch.empty_like(x), torch.empty_like(x)
    rt.kv_read(cache, a, b, ctx)
    want, _ = expected(x.double().cpu().numpy(), "i8")
    assert torch.equal(a.cpu(), round_to(want, "f16")) and torch.equal(a, b)


@pytest.mark.parametrize("t", [1, 5, 64, 65, 200, 4096])
def test_tree_mask(t):
    rng = np.random.default_rng(t)
    parents = np.array([[rng.integers(-1, i) if i else -1 for i in range(t)] for _ in range(3)])
    parents[1] = np.arange(-1, t - 1)   # one chain
    parents[2, t // 2] = t              # not an earlier token: counts as -1
    mask = Guarded((3, t, (t + 63) // 64), torch.int64)
    words, depth = rt.tree_mask(torch.from_numpy(parents.astype(np.int32)).cuda(), mask.t)
    torch.cuda.synchronize()
    assert mask.guards_intact()
    for i in range(3):
        seen, deep = C.ancestors(parents[i])
        assert np.array_equal(words[i].cpu().numpy().view(np.uint64), C.words_of(seen))
        assert np.array_equal(depth[i].cpu().numpy(), deep)


@pytest.mark.parametrize("raw", [False, True])
def test_tree_mask_allocates_on_its_stream(raw):
    # Memory that the current stream's pool hands out may still be in use there.
    side = torch.cuda.Stream()
    parents = torch.arange(-1, 99, dtype=torch.int32, device="cuda").expand(2, 100).contiguous()
    torch.cuda.synchronize()
    mask, depth = rt.tree_mask(parents, stream=side.cuda_stream if raw else side)
    torch.cuda.synchronize()
    for t in (mask, depth):
        owner = [s["stream"] for s in torch.cuda.memory_snapshot()
                 if s["address"] <= t.data_ptr() < s["address"] + s["total_size"]]
        assert owner == [side.cuda_stream]
    assert torch.equal(depth[0].cpu(), torch.arange(100, dtype=torch.int32))


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_all_quotients_of_bf16(kind):
    # Every significand of the row's largest value against every smaller value's,
    # at each power of two that leaves a code: 128 rows of 9 * 128 values.
    m = torch.arange(128, 256, dtype=torch.float64)
    x = (m[None, :, None] * 2.0 ** -torch.arange(9.0, dtype=torch.float64)).reshape(1, -1).repeat(128, 1)
    x[x > m[:, None]] *= 0.5  # (at the largest power only those up to the largest value fit)
    x = x.reshape(128, -1, 64)  # 18 chunks of 64 values to a row of 80 with the largest value first
    rows = torch.zeros(128, x.shape[1], 80, dtype=torch.float64)
    rows[..., 0] = m[:, None]
    rows[..., 1:65] = x
    sign = torch.where(torch.rand(rows.shape, generator=torch.Generator().manual_seed(1)) < 0.5, -1.0, 1.0)
    rows = (rows * sign / 256).reshape(1, 1, -1, 80)
    half = rows.to(torch.bfloat16)
    assert torch.equal(half.double(), rows)
    n = rows.shape[2]
    cache = rt.KvCache.empty(1, 1, n, 80, DT[kind])
    rt.kv_append(half.cuda(), half.cuda(), cache, torch.zeros(1, dtype=torch.int32, device="cuda"))
    codes, scale = C.quantise(rows[0].numpy(), kind)
    assert (decode(cache.k[0]) == codes).all() and (decode(cache.v[0]) == codes).all()
    assert (cache.k_scale[0].cpu().numpy() == scale).all()
