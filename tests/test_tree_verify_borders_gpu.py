"""Decisions close to a border, against the fp64 oracle: what rejected drafts leave is a
difference, right to 2^-42 of what there was before them.  Here they take all but
2^-20, and random numbers lie 2^-21 beside the border or farther."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import serving_ops as S
from tests.test_tree_verify_gpu import DT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stages", [1, 2])
@pytest.mark.parametrize("dt,batch,tokens,vocab", [
    ("f32", 48, 4, 3000), ("f16", 48, 4, 8200), ("bf16", 48, 4, 50304),
    # Rows enough that their weights come from a table.
    ("bf16", 128, 64, 50304)])
def test_after_a_likely_draft_is_rejected(dt, batch, tokens, vocab, stages):
    rng = np.random.default_rng(vocab + stages)
    logits = np.empty((batch, 1, vocab))
    drafts, uniform = np.zeros((batch, tokens), np.int32), np.full((batch, tokens), 0.5, np.float32)
    parents = np.full((batch, tokens), -1, np.int32)
    parents[:, 1:stages + 2] = 0
    for b in range(batch):
        x = 20.0 - np.log(vocab) - 20.0 * np.log(2.0) + rng.normal(0, 0.5, vocab)
        likely = rng.permutation(vocab)[:stages + 1]
        # The first draft all but 2^-20, or each of two all but 2^-10 of what there is.
        x[likely[0]] = 20.0
        if stages == 2:
            x[likely[1]] = 20.0 - 10.0 * np.log(2.0)
        x[likely[-1]] += 6.0
        logits[b, 0] = torch.from_numpy(x).to(DT[dt]).double().numpy()
        a = S.probabilities(logits[b, 0])
        for i in range(stages):
            drafts[b, 1 + i], uniform[b, 1 + i] = likely[i], np.nextafter(np.float32(1), np.float32(0))
            assert a[likely[i]] < uniform[b, 1 + i]
            a[likely[i]] = 0.0
            a /= a.sum()
        last = likely[-1]
        drafts[b, 1 + stages] = last
        side = 1.0 + (1 if b % 2 else -1) * 2.0 ** -rng.uniform(12, 20)
        uniform[b, 1 + stages] = a[last] * side
        assert abs(float(uniform[b, 1 + stages]) / a[last] - 1.0) > 2.0 ** -21
    final = rng.random(batch, np.float32)
    path, count, token = rt.tree_verify(
        torch.from_numpy(logits).to(DT[dt]).cuda().expand(batch, tokens, vocab),
        *(torch.from_numpy(x).cuda() for x in (drafts, parents, uniform, final)))
    path, count, token = path.tolist(), count.tolist(), token.tolist()
    for b in range(batch):
        want, last, _ = S.verify(np.broadcast_to(logits[b], (tokens, vocab)), drafts[b], parents[b], uniform[b], final[b])
        assert len(want) == (1 if b % 2 else 2)
        assert (path[b][:count[b]], token[b]) == (want, last), b


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("batch", [1, 300])
def test_the_least_probability(dt, batch):
    # Weights below 2^-1000 of the largest are none: a random number of 0 picks the first that is
    # one, and accepts no draft without.  2^-1082, 2^-938 and 1, at T = 1/1024.
    x = torch.full((batch, 3, 40), -torch.inf)
    x[:, :, 3], x[:, :, 7], x[:, :, 30] = -750.0 / 1024, -650.0 / 1024, 0.0
    x = x.to(DT[dt]).cuda()
    cold = torch.full((batch,), 2.0 ** -10, device="cuda")
    zeros = torch.zeros(batch, 3, device="cuda")
    parents = torch.tensor([[-1, 0, 0]] * batch, dtype=torch.int32, device="cuda")
    for drafts, path, token in (((0, 3, 3), [0, -1, -1], 7), ((0, 3, 7), [0, 2, -1], 7)):
        got = rt.tree_verify(x, torch.tensor([drafts] * batch, dtype=torch.int32, device="cuda"), parents, zeros,
                             zeros[:, 0].contiguous(), temperature=cold)
        assert got[0].tolist() == [path] * batch and got[2].tolist() == [token] * batch
    # One node a tree.
    one = [t[:, :1].contiguous() for t in (torch.zeros(batch, 3, dtype=torch.int32, device="cuda"), parents, zeros)]
    assert rt.tree_verify(x[:, :1], *one, zeros[:, 0].contiguous(), temperature=cold)[2].tolist() == [7] * batch
