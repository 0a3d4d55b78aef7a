"""frisk_rope with positions of several axes against fp64 rotations; tolerances as
in test_rope_gpu.py."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import cache_ops as C
from tests.gpu_util import Guarded, randn
from tests.test_rope_gpu import DT, table_ints

pytestmark = pytest.mark.gpu


def check(got, x, pos, axis, table, dt, interleaved=False, amplitude=1.0, backward=False):
    """pos [axes, batch, seq] whole numbers; axis of each pair."""
    xd = x.double().cpu().numpy()
    half, rot = torch.finfo(DT[dt]).eps / 2, 2 * len(axis)
    gd = got.double().cpu().numpy()
    turns = table_ints(table)
    for i, a in enumerate(axis):
        one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        pair = xd[..., [one, two]]
        p = pos[a if a < len(pos) else 0][:, None, :]
        want = C.rope(pair, np.broadcast_to(p, pair.shape[:-1]), [turns[i]], interleaved, amplitude, backward)
        size = np.abs(pair).sum(-1, keepdims=True)
        tol = half * np.abs(want) * (dt != "f32") + 4 * 2.0 ** -24 * size * abs(amplitude)
        # An f16 below its least normal number, 2^-14, is a multiple of 2^-24, whatever its
        # size: rounding to it is off by up to half of that.
        tol = tol + 2.0 ** -25 * (dt == "f16")
        err = np.abs(gd[..., [one, two]] - want)
        assert (err <= tol).all(), (i, float((err - tol).max()))
    assert np.array_equal(gd[..., rot:], xd[..., rot:])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved,backward", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("b,h,kv,s,d,sections", [
    (1, 1, 1, 1, 128, [16, 24, 24]), (2, 8, 2, 33, 128, [16, 24, 24]), (3, 5, 5, 7, 80, [8, 8, 4, 4]),
    (1, 3, 1, 19, 64, [1, 2]), (2, 2, 2, 5, 34, [17]), (1, 40, 8, 300, 64, [10, 11, 11]), (2, 3, 1, 4, 96, [0, 9, 1])])
def test_rotation(b, h, kv, s, d, sections, interleaved, backward, dt):
    x, k = (randn((b, s, n, d), 3 + n).to(DT[dt]).transpose(1, 2) for n in (h, kv))
    table = rt.rope_table(2 * sum(sections), 10000.0)
    axis = rt.rope_axes(sections, interleaved=interleaved)
    pos = torch.randint(-1000, 1 << 20, (len(sections), b, s), generator=torch.Generator().manual_seed(1))
    for kind in (torch.int64, torch.int32):
        out, k_out = torch.empty_like(x), torch.empty_like(k)
        rt.rope(x, out, pos.to(kind).cuda(), table, k=k, k_out=k_out, pair_axis=axis, interleaved=interleaved,
                backward=backward, amplitude=1.25)
        for got, t in ((out, x), (k_out, k)):
            check(got, t, pos.numpy(), axis.tolist(), table, dt, interleaved, 1.25, backward)


def test_positions_of_all_sequences_a_start_and_strides():
    x = randn((3, 2, 9, 64), 5)
    table, axis = rt.rope_table(64), rt.rope_axes([8, 12, 12])
    pos = torch.randint(0, 5000, (9, 5, 3), generator=torch.Generator().manual_seed(2)).cuda().permute(2, 1, 0)[:, 2]
    start = torch.tensor([7, 0, 100000], dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    rt.rope(x, out, pos, table, pair_axis=axis, start=start)
    whole = pos.cpu().numpy()[:, None] + start.cpu().numpy()[None, :, None]
    check(out, x, whole, axis.tolist(), table, "f32")
    # A view of the axes at an odd byte, in place, and axes that are none.
    odd = torch.zeros(40, dtype=torch.uint8, device="cuda")[3:35]
    odd.copy_(axis)
    odd[5], odd[20] = 3, 255
    y = x.clone()
    rt.rope(y, y, pos, table, pair_axis=odd, start=start)
    check(y, x, whole, odd.tolist(), table, "f32")


def test_one_axis_is_the_plain_rotation():
    x = randn((2, 4, 50, 128), 6).to(torch.bfloat16)
    table, pos = rt.rope_table(128), torch.randint(0, 10000, (2, 50)).cuda()
    a, b, c = (torch.empty_like(x) for _ in range(3))
    rt.rope(x, a, pos, table)
    rt.rope(x, b, pos[None], table, pair_axis=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    rt.rope(x, c, pos[None].expand(3, 2, 50), table, pair_axis=rt.rope_axes([16, 24, 24]))  # text: the same on all axes
    assert torch.equal(a, b) and torch.equal(a, c)


def test_the_gradient_is_the_transpose():
    # <dy, R x> = <R^T dy, x>, and a difference of the function along x.
    x, dy = randn((1, 2, 30, 64), 7), randn((1, 2, 30, 64), 8)
    table, axis = rt.rope_table(64), rt.rope_axes([8, 12, 12], interleaved=True)
    pos = torch.randint(0, 3000, (3, 30)).cuda()
    y, dx, moved = (torch.empty_like(x) for _ in range(3))
    rt.rope(x, y, pos, table, pair_axis=axis)
    rt.rope(dy, dx, pos, table, pair_axis=axis, backward=True)
    # n sums of products, each off by 5 * 2^-24 of |a| |b| at most: against their sum.
    size = float((dy.abs().double() * y.abs().double()).sum() + (dx.abs().double() * x.abs().double()).sum())
    assert abs(float((dy.double() * y.double()).sum() - (dx.double() * x.double()).sum())) <= 8 * 2.0 ** -24 * size
    step = randn(x.shape, 9)
    rt.rope(x + step, moved, pos, table, pair_axis=axis)
    size = float((dy.abs().double() * (moved.abs() + y.abs()).double()).sum() + (dx.abs() * step.abs()).double().sum())
    assert abs(float((dy.double() * (moved - y).double()).sum() - (dx.double() * step.double()).sum())) \
        <= 16 * 2.0 ** -24 * size


def test_past_l2_and_guards():
    # 40 MB of whole lines: stored past the caches.
    x = randn((1, 40, 2048, 128), 4).to(torch.float32)
    table, axis = rt.rope_table(128), rt.rope_axes([16, 24, 24])
    pos = torch.randint(0, 3000, (3, 1, 2048)).cuda()
    out = Guarded((1, 40, 2048, 128), torch.float32)
    rt.rope(x, out.t, pos, table, pair_axis=axis)
    assert out.guards_intact()
    check(out.t[:, 7:8], x[:, 7:8], pos.cpu().numpy(), axis.tolist(), table, "f32")
    some = torch.empty(1, 1, 2048, 128, device="cuda")
    for h in (0, 39):
        rt.rope(x[:, h:h + 1], some, pos, table, pair_axis=axis)
        assert torch.equal(some, out.t[:, h:h + 1])


def test_refuses_wrong_arguments():
    x = randn((1, 1, 4, 64), 1)
    table, axis = rt.rope_table(64), rt.rope_axes([8, 12, 12])
    pos = torch.zeros(3, 4, dtype=torch.int64, device="cuda")
    for kw, match in ((dict(pair_axis=axis[:5]), "pair_axis must"), (dict(pair_axis=axis.int()), "pair_axis must")):
        with pytest.raises(ValueError, match=match):
            rt.rope(x, x, pos, table, **kw)
    with pytest.raises(ValueError, match="positions"):
        rt.rope(x, x, None, table, pair_axis=axis)
    with pytest.raises(ValueError, match="positions"):
        rt.rope(x, x, pos[0], table, pair_axis=axis)
    with pytest.raises(ValueError, match="axes"):
        rt.rope(x, x, torch.zeros(5, 4, dtype=torch.int64, device="cuda"), table, pair_axis=axis)


def test_graph_replay_streams_and_in_place():
    x = randn((2, 5, 7, 64), 21)
    table, axis = rt.rope_table(48), rt.rope_axes([8, 12, 4])
    pos = torch.zeros(3, 2, 7, dtype=torch.int32, device="cuda")
    out, side = torch.empty_like(x), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    rt.rope(x, out, pos, table, pair_axis=axis, stream=side)
    side.synchronize()
    assert torch.equal(out, x)  # (no turn)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.rope(x, out, pos, table, pair_axis=axis)
    for step in range(3):
        pos.copy_(torch.randint(-50, 50, pos.shape, generator=torch.Generator().manual_seed(step)))
        graph.replay()
        torch.cuda.synchronize()
        check(out, x, pos.cpu().numpy(), axis.tolist(), table, "f32")
    # Heads of one buffer, more of them than a thread has in flight, turned in place.
    wide = randn((2, 7, 40, 64), 22)
    before = wide.clone()
    rt.rope(wide[:, :, :36].transpose(1, 2), wide[:, :, :36].transpose(1, 2), pos, table, pair_axis=axis)
    check(wide[:, :, :36].transpose(1, 2), before[:, :, :36].transpose(1, 2), pos.cpu().numpy(), axis.tolist(), table, "f32")
    assert torch.equal(wide[:, :, 36:], before[:, :, 36:])
