"""Several new tokens a sequence over paged caches: rows between the few and the many, caches of more than 2^32 values,
batches and kept steps that take turns."""

import numpy as np
import pytest

import span_ref as R
from paged_ref import Cache, read_bits, upload_bits
from test_gpu_paged import check, hip, rng_of  # noqa: F401
from test_gpu_spans import queries, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("dh", [32, 64, 100, 128, 256])
@pytest.mark.parametrize("group,fresh", [(1, [16, 3]), (1, [17, 16]), (1, [31, 0, 32]), (1, [33, 2]), (2, [16, 9, 1]), (3, [11, 1]),
                                         (17, [1, 1]), (5, [6, 7])])
def test_rows_between_few_and_many(hip, pkg, half, dh, group, fresh):
    """About 16 and 32 rows under a key head, alone, in windows, over caches that are cut and joined."""
    for old, reach, gap, tree in ((0, None, 0, False), (700, None, 0, True), (2100, 300, 0, False), (2100, 300, 2, True)):
        print(half, dh, group, fresh, old, reach, gap, tree, flush=True)
        rng = rng_of(dh, group, fresh[0], old, gap)
        c = Cache(rng, [f + old // (b + 1) for b, f in enumerate(fresh)], 2, dh, 16, half)
        q = queries(rng, fresh, 2 * group, dh)
        parent = R.random_tree(rng, fresh) if tree else None
        want, bound = R.attend(c, fresh, q, dh ** -0.5, reach, gap, False, parent)
        check(run(hip, pkg, c, fresh, q, dh ** -0.5, reach, gap, False, parent), want, bound)


@pytest.mark.parametrize("half", [False, True])
def test_cache_of_more_than_2_32_values(hip, pkg, half):
    """A prompt stored and attended, drafts stored, attended and kept, on a cache's first and last pages."""
    KH, dh, page, pages, n, f = 1, 256, 64, (1 << 32) // (256 * 64) + 40, 150, 60
    k, v = (hip.alloc_pages(pages, KH, page, dh, half=half) for _ in range(2))
    mass, born = hip.alloc(pages * page), hip.alloc(pages * page)
    g = pkg.Pages(pages=pages, page=page, key_heads=KH, dh=dh, k=k.ptr, v=v.ptr, mass=mass.ptr, born=born.ptr)
    ids = np.array([pages - 1, 0, pages - 2, pages - 7])
    rng = rng_of(9, half)
    ref = Cache(rng, [n + f], 1, dh, n + f, half=half, spare=0)  # (in a page of its own size)
    s = hip.seqs(page, 1, 4)
    for lens, fresh in ((n, n), (n + f, f)):
        s.set([lens], [ids], fresh=[fresh])
        ref.lens[:] = ref.seen[:] = lens
        kk, vv = (rng.standard_normal((fresh, KH, dh)).astype(np.float32) for _ in range(2))
        dk, dv = hip.upload(kk), hip.upload(vv)
        hip.paged_store(s, g, dk.ptr, dv.ptr)
        ref.store([fresh], kk, vv)
        parent = R.random_tree(rng, [fresh]) if fresh == f else None
        q = rng.standard_normal((fresh, 2, dh)).astype(np.float32)
        dq, y = hip.upload(q), hip.alloc(q.size)
        for reach, gap in ((None, 0), (90, 1)):
            if parent is None:
                hip.paged_prompt(s, g, y.ptr, dq.ptr, heads=2, scale=1 / 16, reach=reach, gap=gap)
            else:
                s.tree(parent)
                hip.paged_tree(s, g, y.ptr, dq.ptr, heads=2, scale=1 / 16, reach=reach, gap=gap)
            want, bound = R.attend(ref, [fresh], q, 1 / 16, reach, gap, True, parent)
            check(y.read().reshape(q.shape), want, bound)
    path = np.full(f, R.NONE, np.uint32)
    path[:20] = np.sort(rng.permutation(f)[:20])
    dc, dp = upload_bits(hip, np.array([20])), upload_bits(hip, path)
    hip.paged_keep(s, g, dc.ptr, dp.ptr)
    R.keep(ref, [f], np.array([20]), path)
    s.set([n + 20], [ids])
    ref.lens[:] = ref.seen[:] = n + 20
    q = rng.standard_normal((1, 2, dh)).astype(np.float32)
    dq, y = hip.upload(q), hip.alloc(q.size)
    hip.paged_prompt(s, g, y.ptr, dq.ptr, heads=2, scale=1 / 16)
    want, bound = R.attend(ref, [1], q, 1 / 16)
    check(y.read().reshape(q.shape), want, bound)
    s.free()
    for b in (k, v, mass, born):
        b.free()


class Turn:
    """A batch with its pages and buffers: one prompt's attention and one tree's, verified."""

    def __init__(self, hip, pkg, seed, lens, fresh, heads, KH, dh, half):
        self.hip, self.fresh, self.heads, self.dh = hip, fresh, heads, dh
        rng = rng_of(seed)
        self.c = Cache(rng, lens, KH, dh, 16, half)
        self.g, self.up = self.c.upload(hip, pkg, mass=False, born=False)
        self.s = self.c.batch(hip)
        self.parent = R.random_tree(rng, fresh)
        rows = len(self.parent)
        self.ids = rng.integers(0, 3, rows)
        self.x = rng.standard_normal((rows, 3)).astype(np.float32)
        self.q = queries(rng, fresh, heads, dh)
        self.dq, self.dx = hip.upload(self.q), hip.upload(self.x)
        self.y = [hip.alloc(self.q.size) for _ in range(2)]
        self.out = [hip.alloc(max(k, 1)) for k in (len(lens), rows, len(lens))]
        self.inv, self.cs, self.sn = hip.upload(np.ones(2, np.float32)), hip.alloc(2), hip.alloc(2)
        self.s.set(self.c.lens, self.c.table, fresh=fresh)
        self.s.tree(self.parent, self.ids)
        self.want = [R.attend(self.c, fresh, self.q, dh ** -0.5, parent=p) for p in (None, self.parent)]

    def calls(self, recorded, number):
        hip, how = self.hip, dict(heads=self.heads, scale=self.dh ** -0.5)
        if recorded:
            hip.rope_table(self.cs.ptr, self.sn.ptr, self.inv.ptr, number, 1, 2)
        hip.paged_prompt(self.s, self.g, self.y[0].ptr, self.dq.ptr, **how)
        hip.paged_tree(self.s, self.g, self.y[1].ptr, self.dq.ptr, **how)
        hip.verify(self.s, *(b.ptr for b in self.out), self.dx.ptr, 3)
        if recorded:
            hip.flush()

    def check(self):
        for y, (want, bound) in zip(self.y, self.want):
            check(y.read().reshape(want.shape), want, bound)
            self.hip.write(y, np.full(want.shape, 7.0, np.float32))
        for b, w in zip(self.out, R.verify(self.fresh, self.parent, self.ids, self.x)):
            assert np.array_equal(read_bits(b)[:len(w)], w)


@pytest.mark.parametrize("recorded", [False, True])
def test_batches_take_turns(pkg, recorded):
    """Batches of all sizes in one context, their workspace growing between kept steps: every one's results stay its own."""
    hip = pkg.Hip(0)
    small = Turn(hip, pkg, 1, [900, 40], [5, 7], 4, 2, 32, False)
    for i in range(4):
        small.calls(recorded, i)
        small.check()
    others = [Turn(hip, pkg, 2, [3000], [200], 6, 3, 64, True), Turn(hip, pkg, 3, [40] * 30, [9] * 30, 2, 1, 128, False),
              Turn(hip, pkg, 4, [6000, 5000, 10], [40, 256, 10], 8, 8, 64, False)]
    for i in range(4):
        for t in others:
            small.calls(recorded, 10 + i)
            t.calls(recorded, 10 + i)
            small.check()
            t.check()
    for t in others:  # one set anew while the others' steps are kept
        fresh = [max(f - 3, 1) for f in t.fresh]
        t.s.set(t.c.lens, t.c.table, fresh=fresh)
        small.calls(recorded, 20)
        small.check()
    hip.close()


def test_a_batch_freed_and_made_again(pkg):
    """Batches come and go, their plans and trees with them."""
    hip = pkg.Hip(0)
    before = hip.mem_info()
    for i in range(6):
        t = Turn(hip, pkg, 50 + i, [300 * (1 + i % 3)], [30], 4, 2, 64, i % 2 == 1)
        for _ in range(2):
            t.calls(False, 0)
        t.check()
        t.s.free()
        for b in (*t.up.values(), t.dq, t.dx, *t.y, *t.out, t.inv, t.cs, t.sn):
            b.free()
        if i == 2:
            before = hip.mem_info()
    assert hip.mem_info()[2] <= before[2] + (8 << 20)
    hip.close()
