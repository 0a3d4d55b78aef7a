"""The guide's serving example as it stands there: sequences of different lengths
that verify drafts, then continue one another and end, over a cache with a scale a
row and one with a scale for 32 rows."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import serving_ops as S
from tests.gpu_util import randn
from tests.serving_example import FORK, REST, SETUP, STEP

pytestmark = pytest.mark.gpu

BATCH, TOKENS, MOST, VOCAB = 5, 9, 6, 300
BLOCKS = SETUP.replace("torch.float8_e4m3fn, block_table=block_table)",
                       "torch.int8, block_table=block_table, scale_block=32)")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def keys(cache, lengths):
    """Every key and value of each sequence."""
    b, most = len(lengths), max(max(lengths), 1)
    k, v = (torch.empty(b, 8, most, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    rt.kv_read(cache, k, v, ints([0 if n > 0 else -1 for n in lengths]))
    return [(k[i, :, :n].clone(), v[i, :, :n].clone()) for i, n in enumerate(lengths)]


@pytest.mark.parametrize("setup", [SETUP, BLOCKS], ids=["a scale a row", "a scale for 32"])
def test_the_example(setup):
    rng = np.random.default_rng(11)
    pages = BATCH * MOST + 7
    order = rng.permutation(pages)[:BATCH * MOST].reshape(BATCH, MOST)
    bf = torch.bfloat16
    env = dict(
        rt=rt, torch=torch, pages=pages, tokens=TOKENS, block_table=ints(order.tolist()),
        # Sequences of several lengths (0 and a full page among them), one that has ended.
        ctx=ints([70, 3, 128 - TOKENS, 0, -1]), new=ints([TOKENS, 4, TOKENS, 1, 0]), nodes=ints([9, 5, 9, 9, 0]),
        q=randn((BATCH, 16, TOKENS, 128), 1).to(bf), k=randn((BATCH, 8, TOKENS, 128), 2).to(bf),
        v=randn((BATCH, 8, TOKENS, 128), 3).to(bf), o=torch.zeros(BATCH, 16, TOKENS, 128, dtype=bf, device="cuda"),
        parents=ints([[-1] + [(t - 1) // 2 for t in range(1, TOKENS)]] * BATCH),
        drafts=ints(rng.integers(0, VOCAB, (BATCH, TOKENS)).tolist()), logits=randn((BATCH, TOKENS, VOCAB), 4),
        uniform=torch.full((BATCH, TOKENS), 0.002, device="cuda"), final=torch.full((BATCH,), 0.5, device="cuda"),
        temperature=torch.ones(BATCH, device="cuda"), parent=ints([2, 0, 2, -1, 1]),
        positions=torch.arange(3 * TOKENS, dtype=torch.int32, device="cuda").view(3, 1, TOKENS).expand(3, BATCH, TOKENS))
    exec(setup, env)
    # Keys that were there before.
    begin = env["ctx"].clone()
    old = [randn((BATCH, 8, 130, 128), s).to(bf) for s in (5, 6)]
    rt.kv_append(*old, env["cache"], torch.where(begin < 0, -1, 0).int(), new_len=begin.clamp(min=0))
    exec(STEP, env)
    count, path = env["count"].tolist(), env["path"].tolist()
    new = env["new"].tolist()
    ctx = [b if b < 0 else b + n + c for b, n, c in zip(begin.tolist(), new, count)]
    assert env["ctx"].tolist() == ctx and count[4] == 0 and max(count) > 1 and sum(count) > 4
    assert all(p[:c] == sorted(p[:c]) and p[c:] == [-1] * (TOKENS - c) for p, c in zip(path, count))
    before = keys(env["cache"], ctx)
    table = env["block_table"].tolist()

    exec(FORK, env)
    parent = env["parent"].tolist()
    keep = [-1 if p < 0 else ctx[p] for p in parent]
    assert env["ctx"].tolist() == keep and env["ctx"].dtype == env["nodes"].dtype == torch.int32
    assert env["nodes"].tolist() == [0 if p < 0 else [9, 5, 9, 9, 0][p] for p in parent]
    want = S.next_table(table, keep, [n + TOKENS for n in keep], 64, pages, parent)
    assert env["block_table"].tolist() == want[0] and int(env["lacking"]) == 0
    # Each one has its parent's keys, all of them.
    after = keys(env["cache"], keep)
    for b, p in enumerate(parent):
        if p >= 0:
            assert all(torch.equal(x, y) for x, y in zip(after[b], before[p])), b
            assert torch.isfinite(after[b][0]).all()
    # And pages of its own for what it writes next.
    write = [set(want[0][b][keep[b] // 64:-(-(keep[b] + TOKENS) // 64)]) for b in range(BATCH) if keep[b] >= 0]
    assert all(-1 not in w for w in write) and sum(len(w) for w in write) == len(set().union(*write))

    env["dy"], env["dx"] = randn((BATCH, 16, TOKENS, 128), 8), torch.empty(BATCH, 16, TOKENS, 128, device="cuda")
    env["k16"], env["v16"] = (torch.empty(BATCH, 8, 3, 128, dtype=bf, device="cuda") for _ in range(2))
    env["start"] = ints([0, 1, 2, -1, 0])
    exec(REST, env)
    torch.cuda.synchronize()
