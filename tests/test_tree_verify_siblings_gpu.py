"""Many rejected children of one node, against the fp64 oracle: drafts that the oracle's
own rests reject one after the other, across the walk's 64 nodes at a time."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import serving_ops as S
from tests.test_tree_verify_gpu import DT

pytestmark = pytest.mark.gpu


def siblings(rng, vocab, kids, dense, accept, dt, empty=False):
    """One tree: the logits of its root, draft probabilities there (or None), drafts and
    random numbers; the last child is taken where `accept`.  `empty`: the first
    rejection leaves nothing (the draft probabilities are at least the target's)."""
    x = torch.from_numpy(rng.normal(0, 2, vocab)).to(DT[dt])
    p = S.probabilities(x.double().numpy())
    q = None
    if dense:
        y = np.exp(x.double().numpy() + rng.normal(0, 0.7, vocab))
        q = (y / y.sum()).astype(np.float32)
        if empty:
            q = np.maximum(q, np.nextafter(p.astype(np.float32), np.float32(2))).astype(np.float32)
    a, drafts, uniform = p.copy(), [0], [0.0]
    for i in range(kids):
        of = np.zeros(vocab) if q is None else q.astype(np.float64)
        u = np.float32(rng.uniform(0.5, 1.0))
        clear = 1e-6  # of a border
        ratio = np.full(vocab, u) if q is None else u * of
        if i == kids - 1 and accept:
            if q is None:
                u = np.float32(0.25 * a.max())
                token = int(np.argmax(a))
            else:
                token = int(rng.choice(np.nonzero(a > ratio * (1 + clear))[0]))
        else:
            token = int(rng.choice(np.nonzero(a < ratio * (1 - clear))[0]))
        drafts.append(token)
        uniform.append(u)
        if i == kids - 1 and accept:
            break
        if q is None:
            of = np.zeros(vocab)
            of[token] = 1.0
            rest = a * (1.0 - of)
        else:
            rest = np.maximum(a - of, 0.0)
        if rest.sum() > 0:
            a = rest / rest.sum()
    return x, q, drafts, uniform


def check(batch, vocab, kids, dense, dt, empty=False):
    rng = np.random.default_rng(kids * 1000 + vocab)
    trees = [siblings(rng, vocab, kids, dense, b % 2 == 0, dt, empty) for b in range(batch)]
    t = kids + 1
    logits = torch.stack([x for x, *_ in trees])[:, None].expand(batch, t, vocab).contiguous()
    q = None if not dense else np.stack([np.broadcast_to(q, (t, vocab)) for _, q, *_ in trees])
    drafts, uniform = (np.array([x[i] for x in trees], d) for i, d in ((2, np.int32), (3, np.float32)))
    parents = np.zeros((batch, t), np.int32)
    parents[:, 0] = -1
    final = rng.random(batch, np.float32)
    path, count, token = rt.tree_verify(
        logits.cuda(), *(torch.from_numpy(x).cuda() for x in (drafts, parents, uniform, final)),
        draft_probs=None if q is None else torch.from_numpy(q.copy()).cuda())
    path, count, token = path.cpu().numpy(), count.tolist(), token.tolist()
    for b in range(batch):
        want, last, _ = S.verify(logits[b].double().numpy(), drafts[b], parents[b], uniform[b], final[b],
                                 None if q is None else q[b].astype(np.float64))
        assert (count[b], token[b]) == (len(want), last), b
        assert path[b].tolist() == want + [-1] * (t - len(want)), b
        # Odd trees reject all of their children.
        assert len(want) == (2 if b % 2 == 0 else 1), b


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,kids", [(50, 65), (400, 63), (400, 64), (1000, 130), (9001, 65), (37, 200)])
def test_rests_of_many_rejections(vocab, kids, dt):
    check(4, vocab, kids, True, dt)


@pytest.mark.parametrize("vocab,kids", [(50, 3), (400, 70)])
def test_rests_without_mass(vocab, kids):
    # Nothing is left after the first rejection, nor after any other: the probabilities stay.
    rng = np.random.default_rng(5)
    x, q, *_ = siblings(rng, vocab, 1, True, False, "f32", True)
    assert (q >= S.probabilities(x.double().numpy())).all()
    check(4, vocab, kids, True, "f32", True)


@pytest.mark.parametrize("vocab,kids", [(400, 65), (1000, 130)])
def test_certain_drafts(vocab, kids):
    check(4, vocab, kids, False, "f32")
