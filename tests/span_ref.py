"""Plain implementations in 64 bits of the operators for several new tokens a sequence over paged caches
(paged_ref.py's Cache), and the error bounds their tests hold the kernels to."""

import numpy as np

from paged_ref import U

NONE = 0xffffffff


def lines(parent, fresh):
    """Per sequence: [F][F] whether node j is node i or one that it comes from; [F] depths."""
    out, at = [], 0
    for f in fresh:
        up, depth = np.zeros((f, f), bool), np.zeros(f, np.int64)
        for i in range(f):
            p = int(parent[at + i])
            if p >= 0:
                up[i], depth[i] = up[p], depth[p] + 1
            up[i, i] = True
        out.append((up, depth))
        at += f
    return out


def random_tree(rng, fresh, roots=False):
    """Parents of the rows: mostly near the first node; some more roots if wanted."""
    out = []
    for f in fresh:
        for i in range(f):
            p = int(rng.random() ** 1.5 * i) if i else -1
            out.append(-1 if roots and rng.random() < 0.1 else p)
    return np.array(out, np.int64)


def attend(c, fresh, q, scale, reach=None, gap=0, born=False, parent=None):
    """y [rows][H][dh] and its bound (without fp16 mode's rounding)."""
    rows, H, dh = q.shape
    G, at = H // c.KH, 0
    reach = 1 << 62 if reach is None else reach
    born = born and (gap or reach < 1 << 32)
    tree = None if parent is None else lines(parent, fresh)
    y, bound = np.zeros((rows, H, dh)), np.zeros((rows, H, 1))
    for b, f in enumerate(fresh):
        pg, sl = c.where(b)
        n = len(pg)
        old = n - f
        step = np.arange(f) if tree is None else tree[b][1]
        line = np.tril(np.ones((f, f), bool)) if tree is None else tree[b][0]
        for h in range(H if f else 0):
            kh = h // G
            pos = c.born[pg, kh, sl].astype(np.int64)[:old] if born else np.arange(old)
            end = int(c.seen[b]) - f if born else old
            pos = np.concatenate([pos, end + step])
            back = (end + step)[:, None] - pos[None]
            sees = (back >= gap) & (back < reach)
            sees[:, old:] &= line
            k, v = c.k[pg, kh, sl].astype(np.float64), c.v[pg, kh, sl].astype(np.float64)
            qq = q[at:at + f, h].astype(np.float64)
            for i in range(f):
                on = sees[i]
                m = int(on.sum())
                if not m:
                    continue
                with np.errstate(all="ignore"):
                    s = k[on] @ qq[i] * scale
                    e = np.exp(s - s.max())
                    w = e / e.sum()
                    y[at + i, h] = w @ v[on]
                # A score: a chain of at most dh + 8 roundings of at most sum |q k|, the query's to 23 bits (2 U
                # of an element), three roundings of the score itself (scale, log2 e, its product); the
                # maximum's error cancels. A weight's relative error is the score's, twice (its own and the
                # sum's), the exponential's and division's (8), its two parts' (8, and 2^-37 of the largest
                # for each), and the sums': chains of at most all its slots, rescaled at most once every
                # 16, trees of at most 32 steps.
                a = (np.abs(k[on]) @ np.abs(qq[i]) * abs(scale)).max()
                d = U * ((dh + 10) * a + 3 * np.abs(s).max())
                r = 2 * d + U * (16 + m * 2.0 ** -13 + m + m / 16 + 32)
                bound[at + i, h] = r * np.abs(v[on]).max()
        at += f
    return y, bound


def pick(x):
    """The first maximum: b = 0, b = i whenever x[i] > x[b]."""
    if np.isnan(x[0]):
        return 0
    return int(np.argmax(np.where(np.isnan(x), -np.inf, x)))


def verify(fresh, parent, ids, x):
    """count, path [rows], next."""
    count, path, after, at = [], [], [], 0
    for f in fresh:
        if not f:
            count.append(0)
            after.append(NONE)
            continue
        on = [0]
        while True:
            said = pick(x[at + on[-1]])
            then = [j for j in range(f) if parent[at + j] == on[-1] and ids[at + j] == said]
            if not then:
                break
            on.append(then[0])
        count.append(len(on))
        after.append(said)
        path += on + [NONE] * (f - len(on))
        at += f
    return np.array(count, np.uint32), np.array(path, np.uint32), np.array(after, np.uint32)


def keep(c, fresh, count, path):
    """In place: slot i of the new ones gets what slot path[i] holds, while the path rises among them."""
    at = 0
    for b, f in enumerate(fresh):
        pg, sl = c.where(b)
        pg, sl = pg[len(pg) - f:], sl[len(sl) - f:]
        p = path[at:at + min(int(count[b]), f)].astype(np.int64)
        for i, x in enumerate(p):
            if x < i or x >= f or (i and p[i - 1] >= x):
                p = p[:i]
                break
        for a in (c.k, c.v, c.mass):
            a[pg[:len(p)], :, sl[:len(p)]] = a[pg[p], :, sl[p]]
        at += f
