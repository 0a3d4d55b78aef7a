"""frisk_rope against fp64 rotations whose phases are exact (integers), and its
refusals.

Tolerances: the phase is exact to 2^-32 turns and sine and cosine to 2^-24 of 1, so
with the two roundings of the fused products a result is within 4 * 2^-24 of
(|a| + |b|) amplitude, plus half a step of the output's type."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import cache_ops as C
from tests.gpu_util import Guarded, randn

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def table_ints(table):
    return [int(v) % 2 ** 64 for v in table.cpu().tolist()]


def check(got, x, pos, table, dt, **kw):
    xd = x.double().cpu().numpy()
    want = C.rope(xd, pos, table_ints(table), **kw)
    rot = 2 * table.shape[0]
    half = torch.finfo(DT[dt]).eps / 2
    size = np.zeros_like(xd)
    one = slice(0, rot, 2) if kw.get("interleaved") else slice(0, rot // 2)
    two = slice(1, rot, 2) if kw.get("interleaved") else slice(rot // 2, rot)
    size[..., one] = size[..., two] = (np.abs(xd[..., one]) + np.abs(xd[..., two]))
    tol = half * np.abs(want) * (dt != "f32") + 4 * 2.0 ** -24 * size * abs(kw.get("amplitude", 1.0))
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), float((err - tol).max())
    assert np.array_equal(got[..., rot:].cpu().float().numpy(), x[..., rot:].cpu().float().numpy())


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,h,s,d,rot", [
    (1, 1, 1, 128, 128), (2, 8, 33, 128, 128), (3, 5, 7, 80, 48), (1, 3, 19, 64, 6), (2, 2, 5, 34, 34),
    (1, 40, 300, 64, 64), (1, 1, 1, 2, 2), (2, 3, 4, 96, 20), (1, 7, 3, 4096, 4096)])
def test_rotation(b, h, s, d, rot, interleaved, dt):
    x = randn((b, s, h, d), 3).to(DT[dt]).transpose(1, 2)
    table = rt.rope_table(rot, 10000.0)
    pos = torch.randint(0, 1 << 20, (b, s), generator=torch.Generator().manual_seed(1))
    out = torch.empty_like(x)
    rt.rope(x, out, pos.cuda(), table, interleaved=interleaved, amplitude=1.25)
    check(out, x, pos.numpy()[:, None, :], table, dt, interleaved=interleaved, amplitude=1.25)


@pytest.mark.parametrize("far", [1 << 31, (1 << 40) + 12345, -77777])
def test_far_positions(far):
    # The product of position and frequency wraps exactly.
    x = randn((1, 2, 9, 64), 5)
    table = rt.rope_table(64, 500000.0, scaling="turns", factor=8.0, trained=8192, fast=4.0, slow=1.0)
    pos = torch.arange(far, far + 9)
    out = torch.empty_like(x)
    rt.rope(x, out, pos.cuda(), table)
    check(out, x, pos.numpy()[None, None], table, "f32")


def test_two_tensors_start_and_positions():
    q, k = randn((3, 6, 5, 64), 1), randn((3, 2, 5, 64), 2)
    table = rt.rope_table(64)
    start = torch.tensor([0, 100000, 7], dtype=torch.int32)
    off = torch.tensor([0, 1, 1, 2, 3], dtype=torch.int32)
    for positions, add in ((None, np.arange(5)), (off.cuda(), off.numpy())):
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        rt.rope(q, qo, positions, table, k=k, k_out=ko, start=start.cuda())
        pos = start.numpy()[:, None, None] + add
        check(qo, q, pos, table, "f32")
        check(ko, k, pos, table, "f32")


def test_in_place_inside_one_projection():
    # q and k as heads of one buffer, v between what moves left alone.
    qkv = randn((2, 9, 12, 64), 8).to(torch.bfloat16)
    before = qkv.clone()
    table = rt.rope_table(32)
    q, k = qkv[:, :, :8].transpose(1, 2), qkv[:, :, 8:10].transpose(1, 2)
    rt.rope(q, q, None, table, k=k, k_out=k)
    pos = np.arange(9)[None, None]
    check(qkv[:, :, :8].transpose(1, 2), before[:, :, :8].transpose(1, 2), pos, table, "bf16")
    check(qkv[:, :, 8:10].transpose(1, 2), before[:, :, 8:10].transpose(1, 2), pos, table, "bf16")
    assert torch.equal(qkv[:, :, 10:], before[:, :, 10:])
    # Out of place into other heads of the buffer.
    wide = randn((2, 9, 16, 64), 9)
    src = wide.clone()
    rt.rope(wide[:, :, :8].transpose(1, 2), wide[:, :, 8:].transpose(1, 2), None, table)
    check(wide[:, :, 8:].transpose(1, 2), src[:, :, :8].transpose(1, 2), pos, table, "f32")
    assert torch.equal(wide[:, :, :8], src[:, :, :8])


@pytest.mark.parametrize("offset", [0, 1, 3])
def test_alignment_and_guards(offset):
    buf = randn((2 * 3 * 5 * 24 + 8,), 4).to(torch.float16)
    x = buf[offset:offset + 720].view(2, 3, 5, 24)
    out = Guarded((2, 3, 5, 24), torch.float16)
    table = rt.rope_table(16)
    rt.rope(x, out.t, None, table, interleaved=True)
    torch.cuda.synchronize()
    check(out.t, x, np.arange(5)[None, None], table, "f16", interleaved=True)
    assert out.guards_intact()


@pytest.mark.parametrize("interleaved", [False, True])
def test_backward(interleaved):
    # Against the transposed rotation, and <g, R x> = <R^T g, x> as differences
    # of a linear map: sums of 960 products, each within the tolerance above.
    x, g = randn((2, 3, 5, 32), 1), randn((2, 3, 5, 32), 2)
    table = rt.rope_table(16)
    kw = dict(interleaved=interleaved, amplitude=0.75)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    rt.rope(x, y, None, table, **kw)
    rt.rope(g, dx, None, table, backward=True, **kw)
    check(dx, g, np.arange(5)[None, None], table, "f32", backward=True, **kw)
    one, two = (g.double() * y.double()).sum(), (dx.double() * x.double()).sum()
    bound = 4 * 2.0 ** -24 * 4 * float((g.abs().double() * x.abs().double().amax()).sum())
    assert abs(float(one - two)) <= bound
    # The gradient torch's own graph gives the same rotation.
    leaf = x.double().cpu().requires_grad_(True)
    ang = torch.arange(5, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(8, dtype=torch.float64) / 8)
    c, s = 0.75 * ang.cos(), 0.75 * ang.sin()
    a, b = (leaf[..., 0:16:2], leaf[..., 1:16:2]) if interleaved else (leaf[..., :8], leaf[..., 8:16])
    p, r = a * c - b * s, a * s + b * c
    pair = torch.stack((p, r), -1).flatten(-2) if interleaved else torch.cat((p, r), -1)
    torch.cat((pair, leaf[..., 16:]), -1).backward(g.double().cpu())
    tol = 8 * 2.0 ** -24 * 2 * float(g.abs().max())
    assert float((dx.double().cpu() - leaf.grad).abs().max()) <= tol


def test_graph_replay_and_streams():
    x = randn((2, 4, 16, 64), 1).to(torch.bfloat16)
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    table, out = rt.rope_table(64), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rt.rope(x, out, None, table, start=start)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.rope(x, out, None, table, start=start)
    for step in range(3):
        start.fill_(1000 * step)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(x)
        rt.rope(x, want, None, table, start=start)
        assert torch.equal(out, want)


@pytest.mark.parametrize("stride", [64, 384, 1])
def test_in_place_with_one_kv_head(stride):
    # A projection of 4 + 1 + 1 heads: k's dim of one head has a stride of its own.
    qkv = randn((2, 3, 6 * 64), 3).to(torch.bfloat16)
    before = qkv.clone()
    table = rt.rope_table(64)
    q = qkv[..., :256].view(2, 3, 4, 64).transpose(1, 2)
    k = torch.as_strided(qkv, (2, 1, 3, 64), (3 * 384, stride, 384, 1), 256)
    rt.rope(q, q, None, table, k=k, k_out=k)
    pos = np.arange(3)[None, None]
    check(q, before[..., :256].view(2, 3, 4, 64).transpose(1, 2), pos, table, "bf16")
    check(k, before[..., 256:320].view(2, 3, 1, 64).transpose(1, 2), pos, table, "bf16")
    assert torch.equal(qkv[..., 320:], before[..., 320:])
