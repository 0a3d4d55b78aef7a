"""The oracles of the serving step: verified drafts keep the target's
distribution, tables keep every sequence's keys to itself, shared scales."""
import numpy as np
import pytest

from oracle import cache_ops as C
from oracle import serving_ops as S


def drawn(p, u):
    return int(np.nonzero(np.cumsum(p) > u * np.sum(p))[0][0])


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("kids", [1, 2, 3])
def test_the_next_token_has_the_targets_distribution(dense, kids):
    # 4 tokens, a root with 1 to 3 drafts: over a grid of the random numbers the token
    # behind the root (an accepted draft, or the last token) has its probabilities.
    # A midpoint grid of n points is off by less than 1 / n for each threshold that it
    # is cut at; here there are at most 4 in a row, and 12 in all for a draw.
    logits = np.log(np.array([[0.1, 0.2, 0.3, 0.4]] + [[0.25] * 4] * 3))
    q = np.array([0.4, 0.3, 0.2, 0.1])
    rng = np.random.default_rng(1)
    n, hits = 40000, np.zeros(4)
    parents = [-1] + [0] * kids
    for i in range(n):
        u = rng.random(kids + 2)
        if dense:
            drafts = [0] + [drawn(q, rng.random()) for _ in range(kids)]
        else:
            drafts = [0, 3, 1, 2][:kids + 1]
        path, token, _ = S.verify(logits[:kids + 1], drafts, parents, u[:kids + 1], u[-1],
                                  [q] * (kids + 1) if dense else None)
        hits[drafts[path[1]] if len(path) > 1 else token] += 1
    # 5 standard deviations of n draws.
    p = np.array([0.1, 0.2, 0.3, 0.4])
    assert (np.abs(hits / n - p) < 5 * np.sqrt(p * (1 - p) / n)).all()


def test_rows_without_probabilities_end_the_walk():
    logits = np.zeros((2, 3))
    assert S.verify(logits, [0, 1], [-1, 0], [0, 0.0], 0.5)[0] == [0, 1]
    for bad in ([np.nan, 0, 0], [np.inf, 0, 0], [-np.inf] * 3):
        logits[0] = bad
        path, token, probs = S.verify(logits, [0, 1], [-1, 0], [0, 0.0], 0.5)
        assert path == [0] and token == -1 and np.isnan(probs[1])


def test_a_table_that_forks_ends_and_grows():
    table = [[5, 2, -1, -1], [7, 1, 0, -1], [3, -1, -1, -1]]
    # Row 1 forks into rows 0 and 1 within its second page; row 2 ends.
    out, src, dst, rows, lacking = S.next_table(table, [6, 7, 0], [9, 8, 0], 4, 8, [1, 1, -1])
    assert out == [[7, 1, 0, -1], [7, 2, -1, -1], [-1, -1, -1, -1]]
    assert (src, dst, rows, lacking) == ([-1, 1, -1], [-1, 2, -1], [0, 3, 0], 0)
    # A row that keeps the page in full has it; the other copies.
    out, src, dst, rows, _ = S.next_table(table, [6, 8, 0], [6, 8, 0], 4, 8, [1, 1, -1])
    assert out[0][:2] == [7, 0] and out[1][:2] == [7, 1] and (src[0], dst[0], rows[0]) == (1, 0, 2)
    # Too few pages: the last entries stay empty.
    out, *_, lacking = S.next_table(table, [8, 12, 4], [16, 16, 16], 4, 8)
    assert lacking == 4 and out == [[5, 2, 4, 6], [7, 1, 0, -1], [3, -1, -1, -1]]
    # Pages that are held are not given, nor written.
    out, src, *_ = S.next_table(table, [5, 1, 1], None, 4, 8, held=[1, 0, 1, 0, 0, 0, 0, 0])
    assert out[0][:2] == [5, 1] and src[0] == 2


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_a_scale_that_grows_takes_its_codes_along(kind):
    rng = np.random.default_rng(3)
    values, scale = np.zeros((8, 16)), np.float32(7.0)
    first, second = rng.standard_normal((3, 16)), 5 * rng.standard_normal((2, 16))
    values, s1 = S.append_block(values, scale, 0, first, kind)
    kept, s1b = S.append_block(values, s1, 3, 0.1 * second, kind)
    assert s1b == s1 and (kept[:3] == values[:3]).all()
    moved, s2 = S.append_block(values, s1, 3, second, kind)
    assert s2 > s1 and np.abs(moved[3:5]).max() == C.TOP[kind]
    # Half a step of the largest codes, twice: once for each rounding.
    step = 1.0 if kind == "i8" else 32.0
    assert (np.abs(moved[:3] * s2 - first) <= 0.5 * step * (1 + 2 ** -20) * (s1 + s2)).all()
    bad, s3 = S.append_block(moved, s2, 5, [[np.inf] * 16], kind)
    assert np.isnan(s3) and (bad[:5] == moved[:5]).all() and (bad[5] == 0).all()
