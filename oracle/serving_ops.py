"""Oracles (numpy, fp64, and f32 where the definition says so) of what a serving
step with drafted tokens does around attention: verification of drafts, the
block table of the next step, rows that share scales.  Written from the
definitions in include/frisk_hip.h, one sequence and one step after the other."""
import math

import numpy as np

from oracle import cache_ops as C


# ---- verification of drafts -------------------------------------------------------

def probabilities(row, temperature=1.0):
    """softmax(row / temperature) in fp64, or None if the row gives none."""
    x = np.asarray(row, np.float64)
    if np.isnan(x).any() or not np.isfinite(x.max()):
        return None
    if not temperature > 0:
        p = np.zeros(len(x))
        p[int(np.argmax(x))] = 1.0
        return p
    w = np.exp((x - x.max()) / np.float64(np.float32(temperature)))
    return w / math.fsum(w)


def verify(logits, drafts, parents, uniform, final, draft_probs=None, temperature=1.0, nodes=None):
    """One tree: (path, token, probs of each node's token given its parent)."""
    t, v = logits.shape
    n = t if nodes is None else min(nodes, t)
    rows = {}

    def row(i):
        if i not in rows:
            rows[i] = probabilities(logits[i], temperature)
        return rows[i]

    probs = np.zeros(t)
    for i in range(1, n):
        up, x = int(parents[i]), int(drafts[i])
        if 0 <= up < i:
            p = row(up)
            probs[i] = np.nan if p is None else p[x] if 0 <= x < v else 0.0
    cur, path = 0, [0]
    while True:
        a = row(cur)
        if a is None:
            return path, -1, probs
        a = a.copy()
        for i in range(cur + 1, n):
            if int(parents[i]) != cur:
                continue
            x = int(drafts[i])
            known = 0 <= x < v
            if draft_probs is None:
                q = np.zeros(v)
                if known:
                    q[x] = 1.0
            else:
                q = np.asarray(draft_probs[cur], np.float64)
            if known and float(uniform[i]) * q[x] < a[x]:
                cur = i
                path.append(i)
                break
            rest = a * (1.0 - q) if draft_probs is None else np.maximum(a - q, 0.0)
            mass = math.fsum(rest)
            if mass > 0:
                a = rest / mass
        else:
            break
    total = np.cumsum(a)
    past = np.nonzero(total > float(final) * total[-1])[0]
    return path, int(past[0]), probs


# ---- the table of the next step ------------------------------------------------------

def next_table(table, keep, want, page, pages, parent=None, held=None):
    """(out, src, dst, rows, lacking) as lists."""
    batch, most = len(table), len(table[0])
    taken, room, part = [], [], []
    for b in range(batch):
        up = b if parent is None else parent[b]
        if not 0 <= up < batch or keep[b] < 0:
            taken.append([]), room.append(0), part.append(0)
            continue
        k = min(keep[b], most * page)
        w = k if want is None else max(min(want[b], most * page), k)
        row = [p if 0 <= p < pages else -1 for p in table[up][:-(-k // page)]]
        taken.append(row), room.append(-(-w // page)), part.append(k % page)
    whole = {i for i in range(pages) if held is not None and held[i]}
    for row, p in zip(taken, part):
        whole.update(row[:-1] if p else row)
    whole.discard(-1)
    writer, copies, used = {}, {}, set(whole)
    for b, (row, p) in enumerate(zip(taken, part)):
        if not p or row[-1] < 0:
            continue
        if row[-1] in whole or row[-1] in writer:
            copies[b] = row[-1]
        else:
            writer[row[-1]] = b
        used.add(row[-1])
    free = [i for i in range(pages) if i not in used]
    lacking, out, src, dst, rows = 0, [], [], [], []
    for b in range(batch):
        row = list(taken[b]) + [-1] * (most - len(taken[b]))
        if b in copies:
            row[len(taken[b]) - 1] = -1
        for i in range(room[b]):
            if row[i] < 0:
                if free:
                    row[i] = free.pop(0)
                else:
                    lacking += 1
        to = row[len(taken[b]) - 1] if b in copies else -1
        out.append(row), dst.append(to)
        src.append(copies[b] if to >= 0 else -1), rows.append(part[b] if to >= 0 else 0)
    return out, src, dst, rows, lacking


# ---- rows that share scales ---------------------------------------------------------

def _grid(kind):
    if kind == "i8":
        return np.arange(-127.0, 128.0), np.arange(-127, 128) % 2 == 0
    values = C.e4m3_values()
    keep = sorted((c for c in range(256) if not np.isnan(values[c]) and c != 128), key=lambda c: values[c])
    return values[keep], np.array([c % 2 == 0 for c in keep])


def nearest(y, kind):
    """Values of the type nearest to y (f32 or fp64, exactly), ties to the even code."""
    grid, even = _grid(kind)
    y = np.asarray(y, np.float64)
    hi = np.clip(np.searchsorted(grid, y), 1, len(grid) - 1)
    lo = hi - 1
    dl, dh = y - grid[lo], grid[hi] - y  # exact: 24 bits and 8
    return grid[np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(even[lo], lo, hi)))]


def append_block(values, scale, old, x, kind):
    """One block of one head: `values` [size, d] (of codes) with its `scale`, whose
    first `old` rows hold keys, takes rows x [n, d] behind them.  Returns
    (values, scale)."""
    f = np.float32
    values, x = np.array(values, np.float64), np.asarray(x, np.float64)
    if not np.isfinite(x).all() or (old and np.isnan(scale)):
        values[old:old + len(x)] = 0.0
        return values, f(np.nan)
    a = f(max(np.abs(x).max(), C.TOP[kind] * 2.0 ** -126))
    new = f(a / f(C.TOP[kind]))
    if old and not new > f(scale):
        new = f(scale)
    inv = f(f(1.0) / new)
    if old and new > f(scale):
        values[:old] = nearest(f(values[:old]) * f(f(scale) * inv), kind)
    values[old:old + len(x)] = nearest(f(x) * inv, kind)
    return values, new
