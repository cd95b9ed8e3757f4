"""Plain forms of the shared-prefix operators and of sampling, for their tests (numpy)."""
import math
from fractions import Fraction

import numpy as np

import tree_ref as R


def layout(prefix_cap, cap, prefix_len, used, prefix_of=None, length=None, rows=1, window=0):
    """What nd_prefix_plan lays out: (there, bad) [S] and the maps by name."""
    S, P = len(used), len(prefix_len)
    there, bad = np.zeros(S, int), np.zeros(S, bool)
    maps = {k: np.full((S, rows), -1, np.int64) for k in ("pos", "rot", "from", "lo")}
    groups = [[] for _ in range(P)]
    for i in range(S):
        p = (0 if P else -1) if prefix_of is None else int(prefix_of[i])
        m, u = rows if length is None else int(length[i]), int(used[i])
        L = int(prefix_len[p]) if 0 <= p < P else 0
        fits = 0 <= m <= rows
        there[i] = m if fits else rows
        bad[i] = not fits or p >= P or u < 0 or L < 0 or L + u + m - 1 > 2 ** 31 - 1
        if bad[i] or not m:
            continue
        want = []
        for n in range(m):
            rot = L + u + n
            start = max(0, rot + 1 - window) if window else 0
            want.append((u + n, rot, min(start, L), max(0, start - L)))
        bad[i] = u + m - want[0][3] > cap or L - want[0][2] > prefix_cap
        if bad[i]:
            continue
        for n, w in enumerate(want):
            for k, v in zip(("pos", "rot", "from", "lo"), w):
                maps[k][i, n] = v
            if p >= 0:
                groups[p].append(i * rows + n)
    order = [r for g in groups for r in g]
    maps["first"] = np.cumsum([0] + [len(g) for g in groups])
    maps["order"] = np.array(order + [-1] * (S * rows - len(order)))
    return there, bad, maps


def positions(unpacked, cap, pos):
    """Keys and values ([n][kvh][dim], fp64) at positions of a block's ring."""
    k, ks, v, vs = unpacked
    slot = np.asarray(pos, np.int64) % cap
    return (k[slot].astype(np.float64) * ks[slot].astype(np.float64)[..., None],
            v[slot].astype(np.float64) * vs[slot].astype(np.float64)[..., None])


def attend(H, own, cap, prefix, prefix_cap, L, maps, i, n, q, quant, scale):
    """Row (i, n): [H][v] in 64 bits.  own and prefix: unpacked blocks."""
    QK = len(q) // H
    qq = q.reshape(H, QK)
    if quant:
        c, s = R.stand_for(qq)
        qq = c * s.astype(np.float64)[:, None]
    k, v = positions(own, cap, np.arange(maps["lo"][i, n], maps["pos"][i, n] + 1))
    if L > maps["from"][i, n]:
        a, b = positions(prefix, prefix_cap, np.arange(maps["from"][i, n], L))
        k, v = np.concatenate([a, k]), np.concatenate([b, v])
    return R.attend(qq, k, v, np.ones(len(k), bool), scale)


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, chance, room): room is how far, in the sum's share, the rules'
    borders and the draw are from falling otherwise."""
    x = np.asarray(x, np.float32)
    ids = np.flatnonzero(x > -np.inf)
    if not len(ids):
        return -1, 0.0, 1.0
    top = x[ids].max()
    if not temperature > 0 or min_p > 1:
        return int(ids[np.argmax(x[ids])]), 1.0, 1.0
    if top == np.inf:
        ids, z = ids[x[ids] == np.inf], None
        z = np.zeros(len(ids))
    else:
        z = (x[ids].astype(np.float64) - float(top)) / float(np.float32(temperature))
    by = np.lexsort((ids, -x[ids].astype(np.float64)))
    ids, z = ids[by], z[by]
    w = np.array([math.exp(v) if v > -800 else 0.0 for v in z])
    room = 1.0
    if min_p > 0:
        mp = float(np.float32(min_p))
        keep = w >= mp
        room = min(room, np.abs(w - mp).min()) if mp < 1 else room
        ids, w = ids[keep], w[keep]
    if top_k > 0:
        ids, w = ids[:top_k], w[:top_k]
    if top_p < 1:
        sums, p = np.cumsum(w), max(float(np.float32(top_p)), 0.0)
        end = int(np.searchsorted(sums, p * sums[-1], side="left")) + 1
        room = min(room, np.abs(sums / sums[-1] - p).min()) if p > 0 else room
        ids, w = ids[:end], w[:end]
    sums = np.cumsum(w)
    uu = min(max(float(np.float32(u)), 0.0), 1.0) if u == u else 0.0
    j = min(int(np.searchsorted(sums, uu * sums[-1], side="right")), int(np.flatnonzero(w > 0)[-1]))
    room = min(room, np.abs(sums / sums[-1] - uu).min()) if 0 < uu < 1 else room
    return int(ids[j]), w[j] / sums[-1], room


def draw_in_whole_numbers(weights, u, top_p=1.0):
    """The place drawn from whole weights in order, by exact fractions."""
    if top_p < 1:
        need, got, end = Fraction(float(np.float32(top_p))) * sum(weights), 0, 0
        while end == 0 or got < need:
            got += weights[end]
            end += 1
        weights = weights[:end]
    target, got = Fraction(float(np.float32(u))) * sum(weights), 0
    for j, w in enumerate(weights):
        got += w
        if got > target:
            return j
    return len(weights) - 1
