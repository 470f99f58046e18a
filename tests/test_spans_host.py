"""The host side of the operators for several new tokens a sequence on the CPU (test_batch_host.py's library over
a HIP runtime without a device): which calls are refused and how, and what is queued."""

import numpy as np
import pytest

from span_ref import random_tree
from test_batch_host import host, hip, refused  # noqa: F401



class Set:
    """Three sequences of 40, 0 and 300 tokens, 7, 0 and 130 of them new, in pages of 16, 4 query heads over 2 of 64."""

    def __init__(self, host, hip, half=False):
        self.pages, self.lens, self.fresh = 25, [40, 0, 300], [7, 0, 130]
        self.table = np.zeros((3, 20), np.uint32)
        self.table[0, :3], self.table[2, :19] = [24, 1, 2], np.arange(3, 22)
        self.k, self.v = (hip.alloc_pages(self.pages, 2, 16, 64, half=half) for _ in range(2))
        self.mass, self.born = hip.alloc(self.pages * 32), hip.alloc(self.pages * 32)
        self.g = host.Pages(pages=self.pages, page=16, key_heads=2, dh=64, k=self.k.ptr, v=self.v.ptr,
                            mass=self.mass.ptr, born=self.born.ptr)
        self.s = hip.seqs(16, 3, 20)
        self.s.set(self.lens, self.table, fresh=self.fresh)
        self.parent = random_tree(np.random.default_rng(0), self.fresh)
        self.s.tree(self.parent, np.arange(137))
        self.q, self.y = hip.alloc(137 * 256), hip.alloc(137 * 256)
        self.x, self.count, self.path, self.next = hip.alloc(137 * 50), hip.alloc(3), hip.alloc(137), hip.alloc(3)
        self.hip = hip

    def attend(self, call, **a):
        getattr(self.hip, call)(self.s, self.g, **dict(dict(y=self.y.ptr, q=self.q.ptr, heads=4, scale=1.0), **a))

    def prompt(self, **a):
        self.attend("paged_prompt", **a)

    def tree(self, **a):
        self.attend("paged_tree", **a)

    def verify(self, **a):
        self.hip.verify(self.s, **dict(dict(count=self.count.ptr, path=self.path.ptr, next=self.next.ptr,
                                            logits=self.x.ptr, vocab=50), **a))

    def keep(self, **a):
        a = dict(dict(count=self.count.ptr, path=self.path.ptr), **a)
        self.hip.paged_keep(self.s, self.g, a["count"], a["path"])

    def all(self):
        return self.prompt, self.tree, self.verify, self.keep


def test_calls_that_run(host, hip):
    for half in (False, True):
        t = Set(host, hip, half)
        for f in t.all():
            before = host.lib.stub_launches()
            f()
            assert host.lib.stub_launches() > before, f
        for f in (t.prompt, t.tree):
            for a in (dict(reach=1), dict(gap=1 << 62), dict(reach=1 << 40, gap=3), dict(heads=2), dict(scale=-1.0)):
                f(**a) if a.get("heads") != 2 else f(heads=2, y=t.y.ptr, q=t.q.ptr)
        for f in t.all():  # no new tokens, then no sequences
            t.s.set(t.lens, t.table, fresh=[0, 0, 0])
            t.s.tree([], [])
            before = host.lib.stub_launches()
            f()
            assert host.lib.stub_launches() == before + (f == t.verify), f
            t.s.set([], np.zeros((0, 1)))
            t.s.tree([], [])
            before = host.lib.stub_launches()
            f()
            assert host.lib.stub_launches() == before


def test_attention(host, hip):
    t = Set(host, hip)
    big = hip.alloc(137 * 256 + 4)
    for f in (t.prompt, t.tree):
        refused(host, -1, f, heads=0)
        refused(host, -1, f, heads=3)
        refused(host, -5, f, heads=6)
        refused(host, -3, f, heads=1 << 17)
        refused(host, -1, f, reach=0)
        refused(host, -5, f, y=None)
        refused(host, -5, f, q=None)
        refused(host, -5, f, y=t.y.at(4))
        refused(host, -3, f, q=big.at(1))
        f(y=big.at(1))
        for y in (t.q.ptr, t.k.ptr, t.v.ptr):
            refused(host, -1, f, y=y)
        for field, value, code in (("pages", 24, -5), ("page", 32, -1), ("dh", 66, -3), ("dh", 260, -3), ("k", None, -5),
                                   ("v", t.k.ptr, -1), ("key_heads", 0, -1)):
            old = getattr(t.g, field)
            setattr(t.g, field, value)
            refused(host, code, f)
            setattr(t.g, field, old)
        f()
    t.s.set([33, 32], [[1, 2, 3], [1, 2, 0]])  # a page twice: attention alone reads it
    t.s.tree([-1, -1])
    t.prompt(), t.tree()
    refused(host, -1, t.keep)


def test_trees(host, hip):
    t = Set(host, hip)
    refused(host, -1, t.s.tree, np.full(137, 200))
    bad = t.parent.copy()
    bad[5] = 5
    refused(host, -1, t.s.tree, bad)
    bad[5] = -2  # (no place among the new tokens)
    refused(host, -1, t.s.tree, bad)
    t.tree(), t.verify()  # (the tree is what it was)
    with pytest.raises(ValueError):
        t.s.tree(t.parent[1:])
    with pytest.raises(ValueError):
        t.s.tree(t.parent, np.arange(3))
    assert host.lib.slm_hip_seqs_tree(hip.ctx, t.s.h, None, None) == -1
    t.s.tree(t.parent)  # no tokens
    t.tree()
    refused(host, -1, t.verify)
    t.s.set(t.lens, t.table, fresh=t.fresh)  # the batch anew: no tree
    refused(host, -1, t.tree)
    refused(host, -1, t.verify)
    t.prompt()
    t.s.set([0, 0, 300], t.table, fresh=[0, 0, 257])
    refused(host, -3, t.s.tree, np.full(257, -1))
    t.s.set([0, 0, 300], t.table, fresh=[0, 0, 256])
    t.s.tree(np.arange(256) - 1, np.arange(256))


def test_verify(host, hip):
    t = Set(host, hip)
    refused(host, -1, t.verify, vocab=0)
    refused(host, -5, t.verify, vocab=51)
    refused(host, -3, t.verify, vocab=(1 << 28) + 1)
    for name in ("count", "path", "next", "logits"):
        refused(host, -5, t.verify, **{name: None})
    refused(host, -1, t.verify, count=t.next.ptr)
    refused(host, -1, t.verify, count=t.path.ptr)
    refused(host, -1, t.verify, path=t.x.ptr)
    refused(host, -5, t.verify, path=t.count.ptr)


def test_keep(host, hip):
    t = Set(host, hip)
    refused(host, -5, t.keep, count=None)
    refused(host, -5, t.keep, path=None)
    refused(host, -5, t.keep, path=t.count.ptr)
    refused(host, -1, t.keep, path=t.k.ptr)
    refused(host, -1, t.keep, count=t.born.ptr)
    t.g.mass = t.g.born = None
    t.keep()


def test_gone_foreign_or_captured(host, hip):
    t = Set(host, hip)
    host.lib.stub_set_capturing(1)
    for f in t.all():
        refused(host, -3, f)
    refused(host, -3, t.s.tree, t.parent)
    host.lib.stub_set_capturing(0)
    other = host.Hip(0)
    old, t.s = t.s, other.seqs(16, 3, 20)
    for f in t.all():
        refused(host, -1, f)
    foreign, t.s = t.s, old
    foreign.free()
    other.close()
    h = t.s.h
    t.s.free()
    t.s.h = h
    for f in t.all():
        refused(host, -1, f)
    refused(host, -1, t.s.tree, t.parent)
    t.s.h = None
    for f in t.all():
        refused(host, -1, f)


def test_in_a_recorded_step(host, hip):
    """Recorded, then run at flush; a new batch, a new tree or more kinds of attention than are kept run what
    was recorded."""
    t = Set(host, hip)
    inv, cs, sn = hip.alloc(2), hip.alloc(2), hip.alloc(2)
    for end in (hip.flush, lambda: t.s.tree(t.parent, np.arange(137)), lambda: t.s.set(t.lens, t.table, fresh=t.fresh)):
        hip.rope_table(cs.ptr, sn.ptr, inv.ptr, 0, 1, 2)
        before = host.lib.stub_launches()
        for f in t.all():
            f()
        assert host.lib.stub_launches() == before
        end()
        assert host.lib.stub_launches() >= before + 5
        hip.flush()
    t.s.tree(t.parent, np.arange(137))
    hip.rope_table(cs.ptr, sn.ptr, inv.ptr, 0, 1, 2)
    before = host.lib.stub_launches()
    for gap in range(8):
        t.prompt(gap=gap)
    assert host.lib.stub_launches() == before
    t.prompt(gap=8)
    assert host.lib.stub_launches() >= before + 8
    hip.flush()


def test_parents_of_more_than_32_bits(host, hip):
    """Not taken for what their lower bits name."""
    t = Set(host, hip)
    for bad in (1 << 32, -(1 << 32)):
        parent = t.parent.astype(np.int64)
        parent[5] = bad
        with pytest.raises(ValueError):
            t.s.tree(parent, np.zeros(len(parent)))
    t.tree(), t.verify()


def test_batches_that_grow_and_go_leave_nothing(host, hip):
    """What a batch's trees and plans outgrew goes back with it (memory is held in slabs of 128 MiB)."""
    n = 1024
    k, v = (hip.alloc_pages(n, 1, 256, 4) for _ in range(2))
    g = host.Pages(pages=n, page=256, key_heads=1, dh=4, k=k.ptr, v=v.ptr)
    q, y = hip.alloc(n * 256 * 4), hip.alloc(n * 256 * 4)
    held = []
    for _ in range(120):
        s = hip.seqs(256, n, 1)
        for f in (100, 256):
            s.set([f] * n, np.arange(n)[:, None], fresh=[f] * n)
            s.tree(np.full(n * f, -1))
            hip.paged_tree(s, g, y.ptr, q.ptr, heads=1, scale=1.0)
        s.free()
        held.append(hip.mem_info()[2])
    assert held[-1] == held[1]


def test_tokens_that_are_no_32_bits(host, hip):
    """Not taken for what their lower bits, or their whole part, name; nor a parent for its whole part."""
    t = Set(host, hip)
    for bad in (1 << 32, (1 << 32) + 5, -1, 5.5, float("nan"), float("inf"), 1e30):
        ids = np.arange(137).astype(np.float64 if isinstance(bad, float) else np.int64)
        ids[5] = bad
        with pytest.raises(ValueError):
            t.s.tree(t.parent, ids)
    for bad in (0.5, float("nan")):
        parent = t.parent.astype(np.float64)
        parent[5] = bad
        with pytest.raises(ValueError):
            t.s.tree(parent, np.arange(137))
    t.tree(), t.verify()
    for ids in (np.arange(137), np.arange(137.0), np.arange(137, dtype=np.uint64), [0xffffffff] * 137, np.full(137, (1 << 32) - 1, np.uint64)):
        t.s.tree(t.parent, ids)
    t.s.tree(t.parent.astype(np.float64), np.arange(137))
