"""The operators for several new tokens a sequence as a server uses them: prompts that come in together, drafted trees
stored, attended, verified and kept, call by call and in recorded steps that are kept as graphs."""

import numpy as np
import pytest

import span_ref as R
from paged_ref import Cache, read_bits, upload_bits
from test_gpu_paged import check, hip, rng_of  # noqa: F401
from test_gpu_spans import queries

pytestmark = pytest.mark.gpu

DH, H, KH, VOCAB = 32, 4, 2, 61


class Server:
    """Sequences over one layer's pages, that hands out pages as they grow."""

    def __init__(self, hip, pkg, n, half, room=40, page=16):
        self.hip, self.rng, self.n, self.page = hip, rng_of(1, n), n, page
        self.c = Cache(self.rng, [0] * n, KH, DH, page, half, spare=n * room)
        self.c.table = np.full((n, room), 0xfffffff0, np.uint32)
        self.c.width = room
        self.free = list(self.rng.permutation(self.c.pages))
        self.g, self.up = self.c.upload(hip, pkg)
        self.s = self.c.batch(hip)
        self.bufs = {}
        self.inv, self.cs, self.sn = hip.upload(np.ones(2, np.float32)), hip.alloc(2), hip.alloc(2)

    def buf(self, name, a):
        """The same device buffer for every step's data of a name (kept steps name it)."""
        if name not in self.bufs:
            self.bufs[name] = self.hip.alloc(1 << 16)
        if a is not None and a.size:
            self.hip.write(self.bufs[name], a)
        return self.bufs[name]

    def set(self, lens, fresh):
        c = self.c
        for b, n in enumerate(lens):
            for i in range(-(-int(n) // self.page)):
                if c.table[b, i] >= c.pages:
                    c.table[b, i] = self.free.pop()
        c.lens = c.seen = np.asarray(lens, np.uint32)
        self.s.set(c.lens, c.table, fresh=fresh)

    def step(self, fresh, tree, recorded, number, reach=None, gap=0):
        """One step of new tokens: y, and for a tree the tokens that were kept."""
        hip, rng, c, rows = self.hip, self.rng, self.c, int(np.sum(fresh))
        self.set(c.lens.astype(int) + fresh, fresh)
        q, k, v = (rng.standard_normal((rows, x, DH)).astype(np.float32) for x in (H, KH, KH))
        parent = R.random_tree(rng, fresh) if tree else None
        ids = rng.integers(0, VOCAB, rows)
        x = rng.standard_normal((rows, VOCAB)).astype(np.float32)
        if tree:
            first = np.repeat(np.cumsum(fresh) - fresh, fresh)
            on = (parent >= 0) & (rng.random(rows) < 0.7)
            x[(first + parent)[on], ids[on]] = 9.0
            self.s.tree(parent, ids)
        dq, dk, dv, dx = (self.buf(*a) for a in (("q", q), ("k", k), ("v", v), ("x", x)))
        y, count, path, after = (self.buf(a, None) for a in ("y", "count", "path", "next"))
        if recorded:
            hip.rope_table(self.cs.ptr, self.sn.ptr, self.inv.ptr, number, 1, 2)
        hip.paged_store(self.s, self.g, dk.ptr, dv.ptr)
        call = hip.paged_tree if tree else hip.paged_prompt
        call(self.s, self.g, y.ptr, dq.ptr, heads=H, scale=DH ** -0.5, reach=reach, gap=gap)
        if tree:
            hip.verify(self.s, count.ptr, path.ptr, after.ptr, dx.ptr, VOCAB)
            hip.paged_keep(self.s, self.g, count.ptr, path.ptr)
        if recorded:
            hip.flush()
        c.store(fresh, k, v)
        want, bound = R.attend(c, fresh, q, DH ** -0.5, reach, gap, born=True, parent=parent)
        got = y.read(q.size).reshape(q.shape)
        check(got, want, bound, (number, fresh))
        out = [got]
        if tree:
            wc, wp, wa = R.verify(fresh, parent, ids, x)
            gc, gp, ga = (read_bits(b)[:k] for b, k in ((count, self.n), (path, rows), (after, self.n)))
            assert np.array_equal(gc, wc) and np.array_equal(gp, wp) and np.array_equal(ga, wa)
            R.keep(c, fresh, wc, wp)
            out += [gc, gp]
            c.lens = (c.lens - np.asarray(fresh) + wc).astype(np.uint32)
        for name in ("k", "v"):
            assert np.array_equal(self.up[name].read(), getattr(c, name).ravel()), (name, number)
        assert np.array_equal(read_bits(self.up["born"]), c.born.ravel())
        return out


FRESH = [([40, 3, 0, 90], False), ([1, 1, 25, 2], False), ([7, 9, 3, 1], True), ([7, 9, 3, 1], True), ([7, 9, 3, 1], True),
         ([0, 60, 2, 2], False), ([7, 9, 3, 1], True), ([7, 9, 3, 1], True), ([7, 9, 3, 1], True), ([1, 1, 1, 1], False)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("reach,gap", [(None, 0), (50, 0), (None, 20)])
def test_served_together(hip, pkg, half, reach, gap):
    """Call by call and as recorded steps: the plain results, and the same bits."""
    runs = []
    for recorded in (False, True):
        t = Server(hip, pkg, 4, half)
        runs.append([t.step(f, tree, recorded, i, reach, gap) for i, (f, tree) in enumerate(FRESH)])
    for a, b in zip(*runs):
        for x, y in zip(a, b):
            assert np.array_equal(x, y)


def test_kept_steps_follow_the_batch(pkg):
    """Recorded steps of one shape, kept as graphs, between prompts and direct calls that need more of the workspace;
    another session's in turn."""
    hip = pkg.Hip(0)
    a, b = Server(hip, pkg, 4, False, room=60), Server(hip, pkg, 3, True, room=60)
    before = hip.graph_stats()["captured"]
    a.step([400, 3, 9, 90], False, False, 0), b.step([30, 300, 1], False, False, 0)
    for i in range(10):
        a.step([7, 9, 3, 1], True, True, i)
        b.step([16, 1, 5], True, True, i)
        if i == 5:
            a.step([100, 200, 1, 1], False, False, i)
    assert hip.graph_stats()["captured"] >= before + 2
    hip.close()


def test_more_kinds_of_attention_than_are_kept(hip, pkg):
    """One recorded step with a dozen windows, and the same handle for caches of other heads and types."""
    rng = rng_of(51)
    lens, fresh = [90, 300], [70, 150]
    caches = [Cache(rng, lens, kh, dh, 16, half) for kh, dh, half in ((2, 64, False), (4, 16, True), (1, 128, True))]
    s = caches[0].batch(hip)
    for c in caches:
        c.table = caches[0].table
    s.set(caches[0].lens, caches[0].table, fresh=fresh)
    parent = R.random_tree(rng, fresh)
    s.tree(parent)
    inv, cs, sn = hip.upload(np.ones(2, np.float32)), hip.alloc(2), hip.alloc(2)
    made = []
    for c in caches:
        q = queries(rng, fresh, 4, c.dh)
        made.append((c, c.upload(hip, pkg, mass=False, born=False), q, hip.upload(q)))
    for turn in range(2):
        outs = []
        hip.rope_table(cs.ptr, sn.ptr, inv.ptr, turn, 1, 2)
        for gap in (0, 3, 60, 200):
            for c, (g, up), q, dq in made:
                for call, p in ((hip.paged_prompt, None), (hip.paged_tree, parent)):
                    y = hip.alloc(q.size)
                    call(s, g, y.ptr, dq.ptr, heads=4, scale=0.2, gap=gap)
                    outs.append((c, q, gap, p, y))
        hip.flush()
        for c, q, gap, p, y in outs:
            want, bound = R.attend(c, fresh, q, np.float64(np.float32(0.2)), gap=gap, parent=p)
            check(y.read().reshape(q.shape), want, bound, (gap, c.dh, p is None))


@pytest.mark.parametrize("half", [False, True])
def test_a_chain_is_a_prompt(hip, pkg, half):
    """A tree that is a chain and a prompt are the same question; so are a prompt at once and in pieces."""
    rng = rng_of(61, half)
    n, f = 500, 200
    c = Cache(rng, [n], 2, 64, 16, half)
    q = queries(rng, [f], 6, 64)
    g, up = c.upload(hip, pkg, mass=False, born=False)
    s, dq, y = c.batch(hip), hip.upload(q), hip.alloc(q.size)
    s.set(c.lens, c.table, fresh=[f])
    s.tree(np.arange(f) - 1)
    want, bound = R.attend(c, [f], q, 0.125)
    for call in (hip.paged_prompt, hip.paged_tree):
        call(s, g, y.ptr, dq.ptr, heads=6, scale=0.125)
        check(y.read().reshape(q.shape), want, bound)
    at = 0
    for piece in (1, 16, 17, 100, 66):
        s.set([n - f + at + piece], c.table, fresh=[piece])
        hip.paged_prompt(s, g, y.ptr, dq.at(at * 6 * 64), heads=6, scale=0.125)
        check(y.read(piece * 6 * 64).reshape(piece, 6, 64), want[at:at + piece], bound[at:at + piece])
        at += piece


def test_new_rows_at_any_address(hip, pkg):
    """paged_store of rows that do not start at whole 16 bytes stores what aligned ones do."""
    for half in (False, True):
        got = []
        for off in (0, 1):
            c = Cache(rng_of(71), [40, 0, 33], 3, 20, 16, half)
            g, up = c.upload(hip, pkg)
            s = c.batch(hip)
            s.set(c.lens, c.table, fresh=[30, 0, 1])
            k, v = (rng_of(72, i).standard_normal((31, 3, 20)).astype(np.float32) for i in range(2))
            dk, dv = (hip.upload(np.concatenate([np.zeros(off), a.ravel()])) for a in (k, v))
            hip.paged_store(s, g, dk.at(off), dv.at(off))
            c.store([30, 0, 1], k, v)
            for name in ("k", "v", "mass"):
                assert np.array_equal(up[name].read(), getattr(c, name).ravel()), (name, off)
            assert np.array_equal(read_bits(up["born"]), c.born.ravel())


def test_refusals_leave_everything(hip, pkg):
    """(test_spans_host.py has all of the refusals)"""
    rng = rng_of(81)
    c = Cache(rng, [40, 300], 2, 64, 16)
    g, up = c.upload(hip, pkg)
    s = c.batch(hip)
    s.set(c.lens, c.table, fresh=[3, 4])
    y, q = hip.upload(np.full(7 * 256, 7.0)), hip.upload(np.ones(7 * 256))
    bits = upload_bits(hip, np.full(7, 77))
    for f in (lambda: hip.paged_prompt(s, g, y.ptr, q.ptr, 3, 1.0), lambda: hip.paged_prompt(s, g, y.ptr, q.ptr, 4, 1.0, reach=0),
              lambda: hip.paged_tree(s, g, y.ptr, q.ptr, 4, 1.0), lambda: hip.verify(s, bits.ptr, bits.ptr, bits.ptr, q.ptr, 5),
              lambda: hip.paged_keep(s, g, bits.ptr, up["k"].ptr)):
        with pytest.raises(pkg.SlmError):
            f()
    assert np.all(y.read() == 7.0) and np.all(read_bits(bits) == 77)
    for name in ("k", "v", "mass"):
        assert np.array_equal(up[name].read(), getattr(c, name).ravel())
