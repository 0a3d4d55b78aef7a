"""What drafts that are rejected leave behind in a cache whose slots share scales, as
frisk_kv_append defines it: a larger scale stays, codes before them stay rounded
again, a value that is not finite stays NaN; appending a block from its first slot
makes it anew."""
import pytest
import torch

from frisk_amd import runtime as rt
from tests.gpu_util import randn

pytestmark = pytest.mark.gpu

DT = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}
B, KV, D, BLOCK, CTX, TOKENS = 1, 2, 64, 16, 37, 5  # the last block has keys 32 .. 36


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rows(tokens, seed, scale=1.0):
    return [(scale * randn((B, KV, tokens, D), seed + i)).to(torch.bfloat16) for i in (0, 1)]


def state(cache, n):
    """Codes and scales of keys 0 .. n - 1."""
    at = torch.arange(n, device="cuda") // BLOCK
    return [t[:, :, :n].contiguous().view(torch.uint8) for t in (cache.k, cache.v)] + \
        [s[:, :, at].view(torch.int32) for s in (cache.k_scale, cache.v_scale)]


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_rejected_drafts_leave_their_mark(kind):
    cache = rt.KvCache.empty(B, KV, 64, D, DT[kind], scale_block=BLOCK)
    k, v = rows(CTX, 1)
    rt.kv_append(k, v, cache, ints([0]))
    plain = state(cache, CTX)
    # Small drafts change nothing before them; nor does what replaces them.
    rt.kv_append(*rows(TOKENS, 3, 0.01), cache, ints([CTX]))
    assert equal(state(cache, CTX), plain)
    # Larger ones grow the scale of their block, and of no other, for good.
    rt.kv_append(*rows(TOKENS, 5, 50.0), cache, ints([CTX]))
    grown = state(cache, CTX)
    assert all(torch.equal(x[:, :, :32], y[:, :, :32]) for x, y in zip(grown, plain))
    assert (cache.k_scale[:, :, 2] > 5 * k[:, :, 32:].abs().amax((2, 3)).float() / 448).all()
    assert not any(torch.equal(x[:, :, 32:], y[:, :, 32:]) for x, y in zip(grown, plain))
    rt.kv_append(*rows(TOKENS, 7, 0.01), cache, ints([CTX]))
    assert equal(state(cache, CTX), grown)
    # The decided keys of the block, appended from its first slot, are as they would have been.
    def anew():
        rt.kv_append(k[:, :, 32:], v[:, :, 32:], cache, ints([32]))
        assert equal(state(cache, CTX), plain)
    anew()
    # One value that is not finite makes the head's block NaN, after its draft is rejected too.
    kn, vn = rows(TOKENS, 9)
    vn[0, 1, 4, 3] = float("inf")
    rt.kv_append(kn, vn, cache, ints([CTX]))
    rt.kv_append(*rows(1, 11), cache, ints([CTX]))
    ko, vo = (torch.empty(B, KV, CTX + 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    rt.kv_read(cache, ko, vo, ints([0]))
    assert ko.isfinite().all() and vo[:, 0].isfinite().all() and vo[:, 1, :32].isfinite().all()
    assert vo[:, 1, 32:].isnan().all()
    anew()
