"""Oracles (numpy, fp64) of the operators around attention over a cache:
rotary positions, rows quantised to 8 bits, masks of drafted trees and the
attention of new tokens.  Written from the definitions in include/frisk_hip.h."""
from fractions import Fraction

import numpy as np

TOP = {"e4m3": 448.0, "i8": 127.0}


def rope(x, positions, table, interleaved=False, amplitude=1.0, backward=False):
    """x [..., head_dim] with positions [...] (whole numbers) and table (units
    of 2^-64 turns a position, python ints)."""
    x = np.asarray(x, np.float64)
    out = x.copy()
    rot = 2 * len(table)
    pos = np.asarray(positions)
    flat = np.broadcast_to(pos, x.shape[:-1]).reshape(-1)
    turn = np.empty((flat.size, len(table)))
    cache = {}
    for r, p in enumerate(flat.tolist()):
        if p not in cache:
            cache[p] = [float(Fraction((p * int(f)) % 2 ** 64, 2 ** 64)) for f in table]
        turn[r] = cache[p]
    turn = turn.reshape(x.shape[:-1] + (len(table),)) * (2 * np.pi)
    c, s = amplitude * np.cos(turn), amplitude * np.sin(turn)
    if backward:
        s = -s
    one = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    two = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    a, b = x[..., one], x[..., two]
    out[..., one], out[..., two] = a * c - b * s, a * s + b * c
    return out


def e4m3_values():
    """The 256 values of e4m3fn codes."""
    out = np.empty(256)
    for code in range(256):
        s, e, m = code >> 7, (code >> 3) & 15, code & 7
        v = np.nan if (e, m) == (15, 7) else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[code] = -v if s else v
    return out


def quantise(x, kind):
    """(code values, f32 scales) of the last dimension's rows (fp64).  Codes
    come from the exact quotient x top / a: the nearest of the type's values,
    ties to the even code.  A row that holds an infinity or NaN: codes 0, scale
    NaN."""
    x = np.asarray(x, np.float64)
    top = TOP[kind]
    finite = np.isfinite(x).all(-1)
    x = np.where(finite[..., None], x, 0.0)
    a = np.maximum(np.abs(x).max(-1, keepdims=True), top * 2.0 ** -126)
    scale = (a[..., 0].astype(np.float32) / np.float32(top))
    if kind == "i8":
        grid = np.arange(-127.0, 128.0)
        even = np.arange(-127, 128) % 2 == 0
    else:
        values = e4m3_values()
        keep = [c for c in range(256) if not np.isnan(values[c]) and c != 128]
        keep.sort(key=lambda c: values[c])
        grid = values[keep]
        even = np.array([c % 2 == 0 for c in keep])
    y = x * top  # exact: 11 + 7 bits
    hi = np.clip(np.searchsorted(grid, y / a), 1, len(grid) - 1)
    lo = hi - 1
    # |y - g a| for both neighbours; g a and the differences are exact in fp64.
    dl, dh = y - grid[lo] * a, grid[hi] * a - y
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(even[lo], lo, hi)))
    return grid[pick], np.where(finite, scale, np.float32(np.nan)).astype(np.float32)


def ancestors(parents):
    """bool [t, t] of one tree (itself and what it continues), depths."""
    t = len(parents)
    seen = np.zeros((t, t), bool)
    depth = np.zeros(t, np.int64)
    for i in range(t):
        p = int(parents[i])
        if 0 <= p < i:
            seen[i] = seen[p]
            depth[i] = depth[p] + 1
        seen[i, i] = True
    return seen, depth


def words_of(seen):
    """bool [..., t, n] to uint64 words [..., t, ceil(n / 64)]."""
    n = seen.shape[-1]
    pad = np.zeros(seen.shape[:-1] + (-n % 64,), bool)
    bits = np.concatenate([seen, pad], -1).reshape(seen.shape[:-1] + (-1, 64))
    return (bits.astype(np.uint64) << np.arange(64, dtype=np.uint64)).sum(-1, dtype=np.uint64)


def attention(q, k, v, visible, scale):
    """One head: q [t, d], k and v [n, d], visible [t, n] -> (o, lse, weight of
    |v|).  A row that sees nothing: 0, -inf, 0; hidden rows of k and v do not
    matter."""
    t, d = q.shape
    o, lse, w = np.zeros((t, d)), np.full(t, -np.inf), np.zeros((t, d))
    for i in range(t):
        at = np.nonzero(visible[i])[0]
        if at.size == 0:
            continue
        s = (k[at] @ q[i]) * scale
        m = s.max()
        p = np.exp(s - m)
        l = p.sum()
        o[i] = p @ v[at] / l
        w[i] = p @ np.abs(v[at]) / l
        lse[i] = m + np.log(l)
    return o, lse, w
