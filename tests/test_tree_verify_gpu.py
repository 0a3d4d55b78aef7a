"""frisk_tree_verify against the fp64 oracle: paths, counts and tokens are equal,
probabilities off by their rounding to f32 (2^-24 of the value) and 2^-40 of it
for the 64-bit sums and exponentials of both sides."""
import numpy as np
import pytest
import torch

from frisk_amd import runtime as rt
from oracle import serving_ops as S
from tests.gpu_util import Guarded, randn

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class Trees:
    """Random trees over peaked logits; drafts that are likely under them."""

    def __init__(self, batch, tokens, vocab, dt="f32", branch=2, dense=False, seed=1, shift=0, temperature=None,
                 nodes=None):
        rng = np.random.default_rng(seed)
        self.batch, self.tokens, self.vocab, self.dense = batch, tokens, vocab, dense
        x = randn((batch, tokens, vocab), seed) * 2
        hot = torch.from_numpy(rng.integers(0, vocab, (batch, tokens, min(4, vocab)))).cuda()
        x.scatter_add_(2, hot, torch.full(hot.shape, 6.0, device="cuda"))
        # Rows `shift` elements off a 16-byte boundary, an odd distance apart.
        buf = torch.full((batch, tokens, vocab + 3 + shift), float("nan"), dtype=DT[dt], device="cuda")
        self.logits = buf[:, :, shift:shift + vocab]
        self.logits.copy_(x)
        self.parents = np.array([[-1] + [max(0, (t - 1) // branch - int(rng.integers(0, 2))) for t in range(1, tokens)]
                                 for _ in range(batch)], np.int32).reshape(batch, tokens)
        self.q = torch.softmax(x + 0.7 * randn(x.shape, seed + 1), -1) if dense else None
        self.drafts = rng.integers(0, vocab, (batch, tokens)).astype(np.int32)
        probs = (torch.softmax(x, -1) if self.q is None else self.q).double().cpu().numpy()
        for b in range(batch):
            for t in range(1, tokens):
                p = probs[b, self.parents[b, t]]
                self.drafts[b, t] = rng.choice(vocab, p=p / p.sum())
        self.uniform = rng.random((batch, tokens), np.float32)
        self.final = rng.random(batch, np.float32)
        self.temperature = None if temperature is None else np.array(temperature, np.float32)
        self.nodes = nodes

    def run(self, **kw):
        dev = lambda x: None if x is None else torch.as_tensor(x).cuda()  # noqa: E731
        probs = torch.full((self.batch, self.tokens), 5.0, device="cuda")
        out = [torch.full(s, 77, dtype=torch.int32, device="cuda")
               for s in ((self.batch, self.tokens), (self.batch,), (self.batch,))]
        new = None if self.nodes is None else torch.tensor(self.nodes, dtype=torch.int32, device="cuda")
        rt.tree_verify(self.logits, dev(self.drafts), dev(self.parents), dev(self.uniform), dev(self.final),
                       draft_probs=self.q, temperature=dev(self.temperature), new_len=new, path=out[0], count=out[1],
                       token=out[2], probs=probs, **kw)
        return (*(x.cpu().numpy() for x in out), probs.double().cpu().numpy())

    def check(self, got):
        path, count, token, probs = got
        x = self.logits.double().cpu().numpy()
        q = None if self.q is None else self.q.double().cpu().numpy()
        for b in range(self.batch):
            n = self.tokens if self.nodes is None else self.nodes[b]
            if n < 1:
                assert (path[b] == 77).all() and count[b] == 77 and token[b] == 77 and (probs[b] == 5.0).all()
                continue
            want, last, p = S.verify(x[b], self.drafts[b], self.parents[b], self.uniform[b], self.final[b],
                                     None if q is None else q[b],
                                     1.0 if self.temperature is None else self.temperature[b], n)
            assert path[b].tolist() == want + [-1] * (self.tokens - len(want)), b
            assert (count[b], token[b]) == (len(want), last), b
            assert np.array_equal(np.isnan(probs[b]), np.isnan(p))
            ok = ~np.isnan(p)
            # (Below 2^-126 an f32 has a step of 2^-149.)
            assert (np.abs(probs[b] - p)[ok] <= (2.0 ** -24 + 2.0 ** -40) * p[ok] + 2.0 ** -150).all()
        return self


SIZES = [(1, 1, 1), (3, 1, 2), (2, 2, 7), (2, 5, 8), (3, 3, 9), (2, 4, 63), (2, 9, 1000), (1, 3, 4097),
         (4, 66, 300), (1, 130, 129), (2, 2, 50257)]


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,tokens,vocab", SIZES)
def test_walks(batch, tokens, vocab, dt, dense):
    for seed in (1, 2):
        t = Trees(batch, tokens, vocab, dt, dense=dense, seed=seed + vocab, shift=seed - 1)
        t.check(t.run())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shift", range(8))
def test_rows_at_any_alignment(dt, shift):
    # Both chunk sizes (few rows, many), a vocabulary that ends inside a piece or with one.
    for batch, tokens, vocab in ((2, 3, 2999), (8, 16, 8192 + shift), (40, 16, 4096)):
        t = Trees(batch, tokens, vocab, dt, shift=shift, seed=shift + 5)
        t.check(t.run())


@pytest.mark.parametrize("kids", [2, 5])
def test_children_of_one_node(kids):
    # Every draft continues the root: rejection after rejection there, with the draft
    # probabilities' rests summed one after the other.
    for dense in (False, True):
        for vocab in (5, 400, 9000):
            t = Trees(6, kids + 1, vocab, dense=dense, seed=kids + vocab)
            t.parents[:, 1:] = 0
            t.uniform[:] = np.maximum(t.uniform, 0.7)
            t.check(t.run())


@pytest.mark.parametrize("shift", [0, 3])
@pytest.mark.parametrize("temperature", [None, (0.5, 3.0), (0.21, 0.2), (0.0, 1e-3)])
def test_many_rows_of_a_large_vocabulary(temperature, shift):
    # Enough rows of bf16 that their weights come from a table, but for numbers that it does not
    # hold: masked ones, zeros, the tiny and the large.
    t = Trees(2, 256, 50021, "bf16", branch=1, shift=shift, temperature=temperature, seed=13 + shift)
    t.check(t.run())
    t.logits[0, ::3, 48000:] = -torch.inf
    t.logits[0, 1::3, 3000:3010] = 0.0
    t.logits[1, ::3, 20000:20100] *= 2.0 ** -20
    t.logits[1, 1::3, 30000] = -300.0
    t.logits[1, 2::3, 40000] = 200.0
    t.check(t.run())
    t.logits[0, 5, 17] = float("nan")
    t.logits[1, 7, 45000] = float("inf")
    t.logits[1, 9, :] = -torch.inf
    t.check(t.run())


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("vocab", [4095, 4097, 8193, 20011, 70001])
def test_rows_from_short_to_long(vocab, dense, dt):
    # Rows around what a walk does by itself, and cut ones: greedy trees, masks, several
    # rejections at a node, trees that end early or take no part.
    for branch, seed in ((1, 41), (4, 42)):
        t = Trees(6, 9, vocab, dt, dense=dense, branch=branch, seed=seed, shift=seed % 3,
                  temperature=(0.0, 0.6, 1.0, 1.5, 0.0, 1.0), nodes=[9, 9, 5, 9, 1, 0])
        t.check(t.run())
        t.logits[1, :, vocab // 2:] = -torch.inf
        t.logits[2, 3, 7] = float("nan")
        t.uniform[3] = np.float32(1 - 2.0 ** -24)
        t.check(t.run())


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("batch,vocab,shift", [(2, 7, 0), (3, 8000, 1), (2, 20000, 3), (2, 32768, 0), (3, 32771, 2),
                                               (70, 50257, 1), (130, 131072, 0), (260, 65537, 5), (2, 140000, 1)])
def test_tokens_alone(batch, vocab, shift, dt):
    # One node a tree: rows that a workgroup has whole, and rows that are cut.
    t = Trees(batch, 1, vocab, dt, shift=shift, seed=vocab + shift, temperature=[0.3 + 0.2 * (i % 9) for i in range(batch)])
    t.temperature[::5] = 0.0
    t.logits[batch // 2, 0, vocab // 3:] = -torch.inf
    t.check(t.run())
    t.logits[0, 0, vocab - 1] = float("nan")
    t.logits[1, 0, :] = -torch.inf
    t.nodes = [1] * (batch - 1) + [0]
    t.check(t.run())


def test_many_rows_of_one_sign():
    t = Trees(2, 256, 50021, "bf16", branch=1, temperature=(0.7, 1.0), seed=31)
    t.logits.copy_(t.logits.float().abs() - 25.0)  # all negative, rest and peaks apart
    t.check(t.run())
    t.logits.copy_(t.logits.float() + 40.0)
    t.check(t.run())


def test_many_drafts_of_the_largest_tree():
    t = Trees(2, 1024, 50, branch=3, seed=9)
    t.uniform[0] *= 0.01
    t.check(t.run())
    t.parents[:, 1:] = 0  # 1023 children of the root, over 50 tokens
    t.uniform[:] = np.float32(1 - 2.0 ** -24)
    t.check(t.run())


def test_temperatures():
    for dense in (False, True):
        t = Trees(7, 12, 777, "bf16", dense=dense, temperature=[0.0, 1.0, 0.3, 5.0, 1e-30, 100.0, -1.0], seed=4)
        t.check(t.run())


def test_greedy_takes_the_first_largest():
    t = Trees(2, 4, 5000, "bf16", branch=1, temperature=[0.0, 0.0], seed=2)
    t.logits[0, 0, 1234] = t.logits[0, 0, 4321] = 60.0
    t.logits[1, :, 17] = t.logits[1, :, 4999] = 60.0
    t.drafts[0, 1], t.drafts[1, 1:] = 4321, 17
    t.check(t.run())
    t.parents[:] = np.arange(-1, 3)  # a chain
    path, count, token, _ = got = t.run()
    assert count.tolist() == [1, 4] and token.tolist() == [1234, 17]
    t.check(got)


def test_logits_that_are_masked():
    t = Trees(4, 9, 600, seed=6)
    low = torch.finfo(torch.float32).min
    t.logits[0, :, 100:] = -torch.inf
    t.logits[1, :, :590] = low
    t.logits[2, :, 1:] = -torch.inf  # one token has it all
    t.logits[3, :, ::2] = -torch.inf
    t.drafts[2] = 0
    path, count, token, probs = got = t.run()
    assert token[2] == 0 and count[2] > 1
    t.check(got)


def test_rows_that_give_no_probabilities():
    for bad in (float("nan"), float("inf")):
        t = Trees(4, 5, 3000, branch=1, seed=3)
        t.uniform[:] = 0
        t.logits[0, 0, 2999] = bad   # the root
        t.logits[1, 2, 0] = bad      # in the middle of the path
        t.logits[2, 4, 1500] = bad   # the last node
        t.check(t.run())
        t.parents[:] = np.arange(-1, 4)  # a chain
        path, count, token, probs = got = t.run()
        assert token[:3].tolist() == [-1] * 3 and count[:3].tolist() == [1, 3, 5] and token[3] >= 0
        t.check(got)
    t.logits[:] = -torch.inf
    path, count, token, _ = got = t.run()
    assert (token == -1).all() and (count == 1).all()
    # With temperature 0 too.
    t.temperature = np.zeros(4, np.float32)
    t.logits[:3] = float("nan")
    t.check(t.run())


def test_drafts_and_parents_that_are_none():
    t = Trees(3, 6, 50, seed=8)
    t.uniform[:] = 0
    t.drafts[0, 1:] = [50, -1, 2 ** 31 - 1, -2 ** 31, 51]
    t.parents[1] = [0, 5, -7, 3, 2 ** 31 - 1, -2 ** 31]
    t.parents[2] = [-1, 1, 2, 3, 4, 5]  # none before it: themselves
    path, count, token, probs = got = t.run()
    assert count.tolist() == [1, 1, 1] and (probs == 0).all() and (token >= 0).all()
    t.check(got)


def test_ragged_trees():
    t = Trees(6, 20, 500, nodes=[20, 1, 0, 7, -3, 13], seed=5)
    t.check(t.run())


def test_first_and_last_random_numbers():
    # 0: the first token with a weight; the largest below 1: one of the last.
    t = Trees(4, 3, 3000, seed=7)
    t.logits[:, :, :5] = -torch.inf
    t.uniform[:] = np.float32(1 - 2.0 ** -24)
    for u in (0.0, 1 - 2.0 ** -24):
        t.final[:] = np.float32(u)
        got = t.run()
        t.check(got)


def test_a_rest_without_mass():
    # The drafter's probabilities are above the target's everywhere: what was there stays.
    t = Trees(2, 3, 100, dense=True, seed=1)
    t.parents[:, 1:] = 0
    t.q[:] = 2.0
    t.uniform[:] = 0.999
    t.check(t.run())


def test_strides_and_shared_draft_rows():
    t = Trees(3, 5, 200, dense=True, branch=1, seed=2)
    wide = torch.zeros(5, 3, 231, device="cuda")
    wide[:, :, 7:207] = t.logits.transpose(0, 1)
    t.logits = wide[:, :, 7:207].transpose(0, 1)
    t.q = t.q[:1, :1].expand(3, 5, 200)  # one row for all
    t.check(t.run())


def test_writes_nothing_else_and_any_workspace():
    t = Trees(2, 7, 900, seed=3)
    dev = lambda x: torch.as_tensor(x).cuda()  # noqa: E731
    need = rt.tree_verify_workspace_bytes(2, 7, 900, torch.float32)
    results = []
    for fill in (0, 255, 0x7F):
        outs = [Guarded(s, d) for s, d in (((2, 7), torch.int32), ((2,), torch.int32), ((2,), torch.int32),
                                           ((2, 7), torch.float32))]
        ws = Guarded((need,), torch.uint8)
        ws.t.fill_(fill)
        rt.tree_verify(t.logits, dev(t.drafts), dev(t.parents), dev(t.uniform), dev(t.final), path=outs[0].t,
                       count=outs[1].t, token=outs[2].t, probs=outs[3].t, workspace=ws.t)
        assert all(x.guards_intact() for x in (*outs, ws))
        results.append([x.t.clone() for x in outs])
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], r))
    with pytest.raises(ValueError, match="workspace of"):
        rt.tree_verify(t.logits, dev(t.drafts), dev(t.parents), dev(t.uniform), dev(t.final), workspace=ws.t[:-16])


def test_refuses_wrong_arguments():
    t = Trees(2, 3, 10, seed=3)
    dev = lambda x: torch.as_tensor(x).cuda()  # noqa: E731
    good = dict(logits=t.logits, drafts=dev(t.drafts), parents=dev(t.parents), uniform=dev(t.uniform),
                final=dev(t.final))
    for name, bad in (("drafts", good["drafts"].long()), ("parents", good["parents"][:, :2]),
                      ("uniform", good["uniform"].double()), ("final", good["final"][:1]),
                      ("logits", t.logits.transpose(1, 2))):
        with pytest.raises(ValueError):
            rt.tree_verify(**(good | {name: bad}))
    with pytest.raises(ValueError, match="draft_probs"):
        rt.tree_verify(**good, draft_probs=t.logits.double())
    with pytest.raises(ValueError, match="different devices"):
        rt.tree_verify(**good, temperature=torch.ones(2))


def test_two_calls_at_once():
    # On two streams, from two threads, with workspaces of their own.
    import threading
    trees = [Trees(3, 40, 9000, "bf16", dense=d, seed=20 + d) for d in (False, True)]
    dev = lambda x: torch.as_tensor(x).cuda()  # noqa: E731
    args = [(t.logits, dev(t.drafts), dev(t.parents), dev(t.uniform), dev(t.final)) for t in trees]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        side = torch.cuda.Stream()
        for _ in range(20):
            got[i].append(rt.tree_verify(*args[i], draft_probs=trees[i].q, stream=side))
        side.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i, t in enumerate(trees):
        probs = t.run()[3]
        for out in got[i]:
            t.check((*(x.cpu().numpy() for x in out), probs)) if out is got[i][0] else None
            assert all(torch.equal(a, b) for a, b in zip(out, got[i][0]))


def test_another_stream_and_a_graph():
    t = Trees(4, 17, 5000, "bf16", dense=True, seed=11)
    dev = lambda x: torch.as_tensor(x).cuda()  # noqa: E731
    args = (t.logits, dev(t.drafts), dev(t.parents), dev(t.uniform), dev(t.final))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    path, count, token = rt.tree_verify(*args, draft_probs=t.q, stream=side)
    side.synchronize()
    t.check((*(x.cpu().numpy() for x in (path, count, token)), t.run()[3]))
    # Captured once, replayed on other logits and random numbers.
    ws = torch.empty(rt.tree_verify_workspace_bytes(4, 17, 5000, torch.bfloat16), dtype=torch.uint8, device="cuda")
    probs = torch.empty(4, 17, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.tree_verify(*args, draft_probs=t.q, path=path, count=count, token=token, probs=probs, workspace=ws)
    for seed in (12, 13, 14):
        n = Trees(4, 17, 5000, "bf16", dense=True, seed=seed)
        t.logits.copy_(n.logits)
        t.q.copy_(n.q)
        for x, y in zip(args[1:], (n.drafts, n.parents, n.uniform, n.final)):
            x.copy_(torch.as_tensor(y))
        graph.replay()
        n.check((*(x.cpu().numpy() for x in (path, count, token)), probs.double().cpu().numpy()))


@pytest.mark.parametrize("own_stream", [False, True])
def test_made_outputs_of_trees_without_nodes(own_stream):
    t = Trees(4, 5, 300, seed=61)
    junk = [torch.full((4096,), 9, dtype=torch.int32, device="cuda") for _ in range(8)]
    new, side = torch.tensor([5, 0, -3, 1], dtype=torch.int32, device="cuda"), torch.cuda.Stream()
    dev = lambda x: torch.as_tensor(x).cuda()  # noqa: E731
    args = (t.logits, dev(t.drafts), dev(t.parents), dev(t.uniform), dev(t.final))
    del junk
    torch.cuda.synchronize()
    path, count, token = rt.tree_verify(*args, new_len=new, stream=side if own_stream else None)
    torch.cuda.synchronize()
    assert (path[1:3] == -1).all() and path[3].tolist() == [0, -1, -1, -1, -1]
    assert count.tolist()[1:] == [0, 0, 1] and token.tolist()[1:3] == [-1, -1] and token[3] >= 0 and token[0] >= 0


@pytest.mark.parametrize("batch,tokens,vocab,dense", [(2, 17, 40000, False), (2, 9, 20011, True), (2, 1, 5000, False),
                                                      (2, 1, 140000, False), (4, 64, 131072, False)])
def test_graphs_of_every_way(batch, tokens, vocab, dense):
    # Long rows, one node a tree in one launch and in two, rows through a table; one workspace.
    first = Trees(batch, tokens, vocab, "bf16", dense=dense, seed=51)
    dev = lambda x: torch.as_tensor(x).cuda()  # noqa: E731
    args = (first.logits, dev(first.drafts), dev(first.parents), dev(first.uniform), dev(first.final))
    need = rt.tree_verify_workspace_bytes(batch, tokens, vocab, torch.bfloat16)
    ws = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    probs = torch.empty(batch, tokens, device="cuda")
    rt.tree_verify(*args, draft_probs=first.q, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        path, count, token = rt.tree_verify(*args, draft_probs=first.q, probs=probs, workspace=ws)
    for seed in (52, 53, 54):
        n = Trees(batch, tokens, vocab, "bf16", dense=dense, seed=seed)
        first.logits.copy_(n.logits)
        if dense:
            first.q.copy_(n.q)
        for x, y in zip(args[1:], (n.drafts, n.parents, n.uniform, n.final)):
            x.copy_(torch.as_tensor(y))
        ws.fill_(seed)  # (what it holds does not matter)
        for _ in range(2):
            graph.replay()
            n.check((*(x.cpu().numpy() for x in (path, count, token)), probs.double().cpu().numpy()))
