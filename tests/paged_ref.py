"""Plain implementations in 64 bits of the operators over paged caches and rows of logits, and the
error bounds their tests hold the kernels to."""

import numpy as np

U = 2.0 ** -24   # half a step of fp32, relative
U16 = 2.0 ** -11  # of fp16


class Cache:
    """A paged cache on the host: k, v [pages][KH][page][dh] float32 (of fp16 values with half), mass
    and born [pages][KH][page]; a batch of sequences over it."""

    def __init__(self, rng, lens, KH, dh, page, half=False, seen=None, spare=3, scale=0.8):
        self.KH, self.dh, self.page, self.half = KH, dh, page, half
        self.lens = np.asarray(lens, np.uint32)
        self.seen = self.lens.copy() if seen is None else np.asarray(seen, np.uint32)
        used = -(-self.lens.astype(int) // page)
        self.pages = int(used.sum()) + spare
        ids = rng.permutation(self.pages).astype(np.uint32)
        self.width = int(max(used.max(), 1)) + 1
        self.table = np.full((len(lens), self.width), 0xfffffff0, np.uint32)  # (not looked at behind a sequence)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = ids[at:at + u]
            at += u
        shape = (self.pages, KH, page)
        self.k = self.values(rng.standard_normal((*shape, dh)) * scale)
        self.v = self.values(rng.standard_normal((*shape, dh)) * scale)
        self.mass = rng.random(shape).astype(np.float32) * 3
        self.born = np.zeros(shape, np.uint32)
        for b in range(len(lens)):
            for h in range(KH):
                pg, sl = self.where(b)
                self.born[pg, h, sl] = np.arange(len(pg))

    def values(self, a):
        a = np.asarray(a, np.float32)
        return a.astype(np.float16).astype(np.float32) if self.half else a

    def where(self, b, n=None):
        """Pages and slots of the sequence's first n tokens."""
        t = np.arange(int(self.lens[b]) if n is None else n)
        return self.table[b, t // self.page].astype(int), t % self.page

    def used(self):
        """[pages][KH][page]: the slots that hold tokens."""
        u = np.zeros((self.pages, self.KH, self.page), bool)
        for b in range(len(self.lens)):
            pg, sl = self.where(b)
            u[pg, :, sl] = True
        return u

    # -- the operators --
    def store(self, fresh, k, v):
        row = 0
        for b, f in enumerate(fresh):
            pg, sl = self.where(b)
            for i in range(f):
                at = len(pg) - f + i
                self.k[pg[at], :, sl[at]] = self.values(k[row])
                self.v[pg[at], :, sl[at]] = self.values(v[row])
                self.mass[pg[at], :, sl[at]] = 0
                self.born[pg[at], :, sl[at]] = int(self.seen[b]) - f + i
                row += 1

    def attend(self, q, scale, gap=0, born=True):
        """y [n][H][dh], mass + weights [pages][KH][page], and the bounds of both (without fp16
        mode's rounding)."""
        n, H, dh = q.shape
        G = H // self.KH
        y, bound = np.zeros((n, H, dh)), np.zeros((n, H, 1))
        mass, mbound = self.mass.astype(np.float64), U * (np.abs(self.mass.astype(np.float64)) + 2 * G)
        for b in range(n):
            pg, sl = self.where(b)
            if not len(pg):
                continue
            for h in range(H):
                kh = h // G
                pos = self.born[pg, kh, sl].astype(np.int64) if born else np.arange(len(pg))
                sees = pos + gap < int(self.seen[b] if born else self.lens[b])
                if not sees.any():
                    continue
                k = self.k[pg, kh, sl].astype(np.float64)[sees]
                v = self.v[pg, kh, sl].astype(np.float64)[sees]
                qq = q[b, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = k @ qq * scale
                    e = np.exp(s - s.max())
                    w = e / e.sum()
                    y[b, h] = w @ v
                mass[pg[sees], kh, sl[sees]] += w
                # A score: dh products in chains of at most dh + 8 roundings of at most sum |q k|,
                # three roundings of the score itself (scale, log2 e, its product); the maximum's
                # error cancels. A weight's relative error is the score's, twice (its own and the
                # sum's), the exponential's and division's (8), and the sums': a chain of at most
                # 256 in a superblock, one of all superblocks, trees of at most 32 steps.
                a = (np.abs(k) @ np.abs(qq) * abs(scale)).max()
                d = U * ((dh + 8) * a + 3 * np.abs(s).max())
                r = 2 * d + U * (8 + 256 + len(pg) // 256 + 32)
                bound[b, h] = r * np.abs(v).max()
                with np.errstate(all="ignore"):
                    mbound[pg[sees], kh, sl[sees]] += r * w
        return y, mass, bound, mbound

    def evict(self, keep, recent):
        """In place; rank by (newest, weight, lower slot). NaN below all, -0 as 0."""
        for b in range(len(self.lens)):
            pg, sl = self.where(b)
            if len(pg) <= keep:
                continue
            for h in range(self.KH):
                w = self.mass[pg, h, sl].astype(np.float64) + 0.0
                w = np.where(np.isnan(w), -np.inf, w)
                nan = np.isnan(self.mass[pg, h, sl])
                newest = self.born[pg, h, sl].astype(np.int64) + recent >= int(self.seen[b])
                order = np.lexsort((np.arange(len(pg)), nan & ~newest, np.where(newest, -np.inf, -w), ~newest))
                kept = np.zeros(len(pg), bool)
                kept[order[:keep]] = True
                to, frm = np.flatnonzero(~kept[:keep]), keep + np.flatnonzero(kept[keep:])
                for a in (self.k, self.v, self.mass, self.born):
                    a[pg[to], h, sl[to]] = a[pg[frm], h, sl[frm]]

    # -- on the device --
    def upload(self, hip, pkg, mass=True, born=True):
        up = {}
        for name in ("k", "v"):
            up[name] = hip.alloc_pages(self.pages, self.KH, self.page, self.dh, half=self.half)
            hip.write(up[name], getattr(self, name))
        if mass:
            up["mass"] = hip.upload(self.mass)
        if born:
            up["born"] = upload_bits(hip, self.born)
        g = pkg.Pages(pages=self.pages, page=self.page, key_heads=self.KH, dh=self.dh,
                      **{k: b.ptr for k, b in up.items()})
        return g, up

    def batch(self, hip, max_pages=None):
        return hip.seqs(self.page, len(self.lens), max_pages or self.width)


def upload_bits(hip, a):
    """32-bit whole numbers into a device buffer, bit for bit (outside fp16 mode)."""
    return hip.upload(np.ascontiguousarray(a, np.uint32).view(np.float32))


def read_bits(buf):
    return buf.read().view(np.uint32)


def logprobs(x, ids, top):
    """lp, entropy, top ids, top lp in 64 bits, and an absolute bound for lp and entropy."""
    m, n = x.shape
    lp, ent, ti, tl = np.zeros(m), np.zeros(m), np.zeros((m, top), np.int64), np.zeros((m, top))
    bl, be = np.zeros(m), np.zeros(m)
    with np.errstate(all="ignore"):
        for i in range(m):
            r = x[i].astype(np.float64)
            key = np.where(np.isnan(r), -np.inf, r + 0.0)
            ti[i] = np.lexsort((np.arange(n), np.isnan(r), -key))[:top]
            if np.all(r == -np.inf):
                lp[i], ent[i], tl[i] = -np.inf, 0.0, -np.inf
                continue
            M = key.max()
            # (the maximum goes first: next to a logit of 1e38 the sum's logarithm would be lost)
            lse = np.log(np.exp(r - M).sum()) if np.isfinite(M) else 0.0
            if np.isnan(r).any():
                lse = np.nan
            l = (r - M) - lse
            lp[i], tl[i] = l[ids[i]], l[ti[i]]
            p = np.exp(l)
            ent[i] = -np.where(p > 0, p * np.where(p > 0, l, 0), 0).sum() if np.isfinite(M + lse) else np.nan
            # e^d of a rounded d = x - M (and its product with log2 e): relative error at most
            # (2 |d| + 2) U, of |d| e^d at most that times |d|; sums in chains of at most n / 1024
            # and trees of at most 32 steps; the logarithm (4) and two last roundings of x - M - log L
            d = np.minimum(M - key[np.isfinite(key)], 100.0) if np.isfinite(M) else np.zeros(1)
            pe = np.exp(-d) / np.exp(-d).sum()
            chain = n / 1024 + 32
            rel = (pe * (2 * d + 2)).sum() + chain
            bl[i] = U * (rel + 4 + 2 * np.log(n)) 
            be[i] = U * (rel + 4 + 2 * np.log(n) + (pe * d * (2 * d + 4)).sum() + 2 * (pe * d).sum() * (chain + rel))
    return lp, ent, ti, tl, bl, be
