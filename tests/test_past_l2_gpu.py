"""Rotations and cache rows beyond 32 MB, which are loaded and stored past the L2s:
the same bits as calls of parts below that, which test_rope_gpu.py and
test_kv_cache_gpu.py compare with the definitions."""
import pytest
import torch

from frisk_amd import runtime as rt
from tests.gpu_util import Guarded, randn

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn,
      "i8": torch.int8}
L2 = 32 << 20


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt,heads,kv,d,rot,seq", [
    ("f32", 8, 2, 128, 64, 7001), ("f32", 5, 5, 64, 64, 14003), ("bf16", 16, 4, 128, 128, 7001),
    ("f16", 9, 3, 256, 128, 6001)])
def test_rotation(dt, heads, kv, d, rot, seq, interleaved, backward):
    es = torch.empty((), dtype=DT[dt]).element_size()
    assert seq * (heads + kv) * d * es > L2
    q, k = (randn((1, seq, h, d), h).to(DT[dt]).transpose(1, 2) for h in (heads, kv + 20))
    k = k[:, :kv]
    table = rt.rope_table(rot)
    kw = dict(interleaved=interleaved, backward=backward, amplitude=1.25)
    qo, ko = Guarded((1, heads, seq, d), DT[dt]), Guarded((1, kv, seq, d), DT[dt])
    rt.rope(q, qo.t, None, table, k=k, k_out=ko.t, **kw)
    want_q, want_k = torch.empty_like(qo.t), torch.empty_like(ko.t)
    for part in torch.arange(seq, dtype=torch.int32, device="cuda").split(1500):
        a, b = int(part[0]), int(part[-1]) + 1
        assert (b - a) * (heads + kv) * d * es <= L2
        rt.rope(q[:, :, a:b], want_q[:, :, a:b], part, table, k=k[:, :, a:b], k_out=want_k[:, :, a:b], **kw)
    assert torch.equal(qo.t, want_q) and torch.equal(ko.t, want_k)
    assert qo.guards_intact() and ko.guards_intact()
    rt.rope(q, q, None, table, k=k, k_out=k, **kw)  # in place
    assert torch.equal(q, want_q) and torch.equal(k, want_k)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("dt,kind,batch,tokens,kv,d,page", [
    ("bf16", "e4m3", 3, 3001, 8, 128, 64), ("f16", "i8", 3, 3001, 8, 128, 0), ("bf16", "bf16", 2, 3501, 5, 256, 16),
    ("f16", "f16", 5, 7001, 4, 64, 0), ("f16", "e4m3", 3, 9001, 4, 80, 32), ("bf16", "i8", 5, 7001, 8, 32, 128)])
def test_append_and_read(dt, kind, batch, tokens, kv, d, page, ragged):
    assert batch * tokens * kv * d * 4 > L2
    gen = torch.Generator().manual_seed(tokens)
    ctx = torch.randint(0, 50, (batch,), generator=gen, dtype=torch.int32).cuda()
    new = torch.randint(tokens // 2, tokens + 1, (batch,), generator=gen, dtype=torch.int32)
    new[0] = tokens
    new = new.cuda() if ragged else torch.full_like(ctx, tokens)
    pages, size, table = batch, tokens + 50, None
    if page:
        per = -(-(tokens + 50) // page)
        pages, size = batch * per + 1, page
        table = torch.randperm(pages, generator=gen)[:batch * per].view(batch, per).int().cuda()
    x = [randn((batch, tokens, kv, d), i).to(DT[dt]).transpose(1, 2) for i in (1, 2)]
    whole, parts = (rt.KvCache.empty(pages, kv, size, d, DT[kind], block_table=table) for _ in range(2))
    for c in (whole, parts):
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            if t is not None:
                t.view(torch.uint8).fill_(0x33)
    rt.kv_append(x[0], x[1], whole, ctx, new_len=new if ragged else None)
    step = L2 // 4 // (batch * kv * d)
    for at in range(0, tokens, step):
        rows = slice(at, min(at + step, tokens))
        rt.kv_append(x[0][:, :, rows], x[1][:, :, rows], parts, ctx + at, new_len=(new - at).clamp(min=0))
    for t, u in ((whole.k, parts.k), (whole.v, parts.v), (whole.k_scale, parts.k_scale), (whole.v_scale, parts.v_scale)):
        assert t is None or torch.equal(t.view(torch.uint8), u.view(torch.uint8))
    out = [Guarded((batch, kv, tokens, d), DT[dt]) for _ in range(2)]
    want = [torch.full((batch, kv, tokens, d), 5.0, dtype=DT[dt], device="cuda") for _ in range(2)]
    for o in out:
        o.t.fill_(5.0)
    rt.kv_read(whole, out[0].t, out[1].t, ctx, new_len=new if ragged else None)
    for at in range(0, tokens, step):
        rows = slice(at, min(at + step, tokens))
        rt.kv_read(parts, want[0][:, :, rows], want[1][:, :, rows], ctx + at, new_len=(new - at).clamp(min=0))
    for o, w in zip(out, want):
        assert torch.equal(o.t, w) and o.guards_intact()
    live = torch.arange(tokens, device="cuda") < new[:, None]
    assert (want[0].transpose(1, 2)[~live] == 5.0).all()
    if kind == dt:  # a 16-bit cache gives back what it took
        assert torch.equal(out[0].t.transpose(1, 2)[live], x[0].transpose(1, 2)[live])
