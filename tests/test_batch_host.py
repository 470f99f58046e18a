"""The host side of the operators over paged caches and rows of logits on the CPU: the host
runtime's own sources over a HIP runtime without a device (hip_stub.cpp). Which calls are refused
and how, that a refused call queues nothing, and the batch as it goes to the device."""

import ctypes
import subprocess
import types

import numpy as np
import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The package's binding over the test library."""
    out = tmp_path_factory.mktemp("host") / "libslm_host.so"
    src = ROOT / "slm.use_amd" / "csrc"
    subprocess.run(["/opt/rocm/llvm/bin/clang++", "-O1", "-std=c++17", "-fPIC", "-shared", "-Wl,-Bsymbolic",
                    "-ffp-contract=off", "-D__HIP_PLATFORM_AMD__", "-w", "-I", "/opt/rocm/include", "-I", str(ROOT / "include"), "-I", str(src),
                    str(src / "runtime.cpp"), str(src / "model.cpp"), str(ROOT / "tests" / "hip_stub.cpp"), "-o", str(out)],
                   check=True)
    mod = types.ModuleType("slm_host")
    mod.__file__ = str(ROOT / "slm.use_amd" / "__init__.py")
    text = (ROOT / "slm.use_amd" / "__init__.py").read_text()
    assert text.count('PKG / "libslm_hip.so"') == 1
    text = text.replace('PKG / "libslm_hip.so"', f'Path({str(out)!r})')
    import sys
    sys.modules["slm_host"] = mod
    exec(compile(text, mod.__file__, "exec"), mod.__dict__)
    mod.lib.stub_launches.restype = ctypes.c_long
    return mod


@pytest.fixture()
def hip(host):
    h = host.Hip(0)
    yield h
    host.lib.stub_set_capturing(0)
    h.close()


class Set:
    """Three sequences of 40, 0 and 300 tokens in pages of 16, 4 query heads over 2 of 64."""

    def __init__(self, host, hip, half=False):
        self.pages, self.lens = 25, [40, 0, 300]
        self.table = np.zeros((3, 20), np.uint32)
        self.table[0, :3], self.table[2, :19] = [24, 1, 2], np.arange(3, 22)
        self.k, self.v = (hip.alloc_pages(self.pages, 2, 16, 64, half=half) for _ in range(2))
        self.mass, self.born = hip.alloc(self.pages * 32), hip.alloc(self.pages * 32)
        self.g = host.Pages(pages=self.pages, page=16, key_heads=2, dh=64, k=self.k.ptr, v=self.v.ptr,
                            mass=self.mass.ptr, born=self.born.ptr)
        self.s = hip.seqs(16, 3, 20)
        self.s.set(self.lens, self.table)
        self.q, self.y = hip.alloc(3 * 4 * 64), hip.alloc(3 * 4 * 64)
        self.new = [hip.alloc(2 * 2 * 64) for _ in range(2)]
        self.mass2, self.born2 = hip.alloc(self.pages * 32), hip.alloc(self.pages * 32)
        self.hip = hip

    def store(self, **a):
        a = dict(dict(k=self.new[0].ptr, v=self.new[1].ptr), **a)
        self.hip.paged_store(self.s, self.g, a["k"], a["v"])

    def attend(self, **a):
        self.hip.paged_attend(self.s, self.g, **dict(dict(y=self.y.ptr, q=self.q.ptr, heads=4, scale=1.0), **a))

    def evict(self, **a):
        self.hip.paged_evict(self.s, self.g, **dict(dict(mass_out=self.mass2.ptr, born_out=self.born2.ptr, keep=100,
                                                         recent=10), **a))


def refused(host, code, f, *a, **k):
    before = host.lib.stub_launches()
    with pytest.raises(host.SlmError) as e:
        f(*a, **k)
    assert e.value.code == code, str(e.value)
    assert host.lib.stub_launches() == before


def test_calls_that_run(host, hip):
    for half in (False, True):
        t = Set(host, hip, half)
        for f in (t.store, t.attend, t.evict):
            before = host.lib.stub_launches()
            f()
            assert host.lib.stub_launches() > before, f
        t.attend(mass_out=t.mass.ptr)
        t.attend(mass_out=t.mass2.ptr, gap=1 << 62)
        t.evict(mass_out=t.mass.ptr, born_out=t.born.ptr)
        before = host.lib.stub_launches()
        t.evict(mass_out=t.mass.ptr, born_out=t.born.ptr, keep=300)  # nothing to give up
        assert host.lib.stub_launches() == before
        t.s.set([], np.zeros((0, 1)))
        for f in (t.store, t.attend, t.evict):
            f()
        assert host.lib.stub_launches() == before


@pytest.mark.parametrize("field,value,code", [
    ("pages", 24, -5), ("pages", 26, -5), ("pages", 0, -1), ("pages", 1 << 40, -3), ("page", 32, -1), ("page", 0, -1),
    ("key_heads", 0, -1), ("key_heads", 1 << 40, -3), ("key_heads", 3, -5), ("dh", 66, -3), ("dh", 260, -3), ("dh", 0, -1),
    ("dh", 68, -5), ("k", None, -5), ("v", None, -5)])
def test_caches(host, hip, field, value, code):
    t = Set(host, hip)
    setattr(t.g, field, value)
    heads = t.g.key_heads if 0 < t.g.key_heads < 9 else 4
    for f in (t.store, t.evict):
        refused(host, code, f)
    refused(host, code, t.attend, heads=heads)


def test_buffers_that_meet(host, hip):
    t = Set(host, hip)
    for field, other in (("v", t.k.ptr), ("v", t.k.ptr), ("mass", t.k.ptr), ("born", t.v.ptr), ("mass", t.born.ptr)):
        old = getattr(t.g, field)
        setattr(t.g, field, other)
        for f in (t.store, t.attend, t.evict):
            refused(host, -1, f)
        setattr(t.g, field, old)
    t.g.k = t.k.ptr + 4
    refused(host, -5, t.attend)  # (past the end)
    t.g.k, half = t.k.ptr, hip.alloc_pages(t.pages, 2, 16, 64, half=True)
    t.g.v = half.ptr
    refused(host, -1, t.attend)  # fp32 keys and fp16 values
    t.g.k = half.ptr + 2
    refused(host, -1, t.attend)
    small = hip.alloc_pages(t.pages - 1, 2, 16, 64, half=True)
    t.g.k = small.ptr
    refused(host, -5, t.attend)
    big = hip.alloc(t.pages * 2 * 16 * 64 + 4)
    t.g.k, t.g.v = big.at(1), t.v.ptr
    refused(host, -3, t.attend)  # not aligned


def test_attend(host, hip):
    t = Set(host, hip)
    refused(host, -1, t.attend, heads=0)
    refused(host, -1, t.attend, heads=3)
    refused(host, -3, t.attend, heads=34)
    refused(host, -5, t.attend, heads=6)
    refused(host, -5, t.attend, y=None)
    refused(host, -5, t.attend, q=None)
    refused(host, -5, t.attend, y=t.y.at(4))
    big = hip.alloc(3 * 4 * 64 + 4)
    refused(host, -3, t.attend, q=big.at(1))
    t.attend(y=big.at(1))
    for y in (t.q.ptr, t.k.ptr, t.v.ptr, t.mass.ptr, t.born.ptr):
        refused(host, -1, t.attend, y=y)
    for out in (t.k.ptr, t.v.ptr, t.born.ptr):
        refused(host, -1, t.attend, mass_out=out)
    refused(host, -5, t.attend, mass_out=t.mass.at(1))
    refused(host, -5, t.attend, mass_out=t.y.ptr)
    t.g.mass = None
    refused(host, -1, t.attend, mass_out=t.mass2.ptr)
    t.attend()


def test_store(host, hip):
    t = Set(host, hip)
    refused(host, -5, t.store, k=None)
    refused(host, -5, t.store, v=t.new[1].at(1))
    refused(host, -1, t.store, k=t.k.ptr)
    t.s.set(t.lens, t.table, fresh=[2, 0, 1])
    refused(host, -5, t.store)  # three rows
    t.s.set(t.lens, t.table, fresh=[0, 0, 0])
    t.store(k=None, v=None)


def test_evict(host, hip):
    t = Set(host, hip)
    refused(host, -1, t.evict, keep=0, recent=0)
    refused(host, -1, t.evict, keep=5, recent=6)
    refused(host, -1, t.evict, mass_out=None)
    refused(host, -1, t.evict, born_out=None)
    refused(host, -1, t.evict, mass_out=t.mass.ptr)  # one of them the cache's own
    refused(host, -1, t.evict, born_out=t.born.ptr)
    refused(host, -1, t.evict, mass_out=t.born.ptr, born_out=t.mass.ptr)
    refused(host, -1, t.evict, mass_out=t.k.ptr)
    refused(host, -1, t.evict, mass_out=t.mass2.ptr, born_out=t.mass2.ptr)
    refused(host, -5, t.evict, mass_out=t.y.ptr)
    for field in ("mass", "born"):
        old = getattr(t.g, field)
        setattr(t.g, field, None)
        refused(host, -1, t.evict)
        setattr(t.g, field, old)


def test_batches(host, hip):
    t = Set(host, hip)
    set_ = t.s.set
    refused(host, -5, set_, [1] * 4, np.zeros((4, 1)))
    refused(host, -5, set_, [321], np.zeros((1, 30)))
    refused(host, -5, set_, [33], np.zeros((1, 2)))
    refused(host, -1, set_, [33], [[1, 2, 3]], fresh=[34])
    refused(host, -1, set_, [33], [[1, 2, 3]], seen=[32])
    refused(host, -3, set_, [33], [[1, 2, 1 << 27]])
    t.attend()  # (the batch is what it was)
    set_([33, 16], [[1, 2, t.pages], [4, 0xffffffff, 0xffffffff]])
    for f in (t.store, t.attend, t.evict):
        refused(host, -5, f)
    # a page twice: attention alone reads it
    set_([33, 20], [[1, 2, 3], [4, 3, 0]])
    t.attend()
    refused(host, -1, t.attend, mass_out=t.mass.ptr)
    refused(host, -1, t.store)
    refused(host, -1, t.evict)
    set_([33, 32], [[1, 2, 3], [1, 5, 0]])  # a shared prefix: the new tokens go elsewhere
    t.store()
    refused(host, -1, t.evict)
    set_([33, 32], [[1, 2, 3], [1, 2, 0]])
    refused(host, -1, t.store)
    set_([33], [[1, 2, 1]])  # within a sequence
    refused(host, -1, t.store)
    for args in ((0, 1, 1), (16, 0, 1), (16, 1, 0), (16, 1 << 20, 1), (1 << 31, 1, 1), (16, 65536, 1 << 20), (1 << 62, 1, 4)):
        with pytest.raises(host.SlmError):
            hip.seqs(*args)
    with pytest.raises(host.SlmError):
        hip.alloc_pages(1 << 40, 1 << 40, 16, 64)


def test_a_batch_that_is_gone_or_another_contexts(host, hip):
    t = Set(host, hip)
    other = host.Hip(0)
    foreign = other.seqs(16, 3, 20)
    old, t.s = t.s, foreign
    for f in (t.store, t.attend, t.evict):
        refused(host, -1, f)
    t.s = old
    h = t.s.h
    t.s.free()
    t.s.h = h
    for f in (t.store, t.attend, t.evict):
        refused(host, -1, f)
    refused(host, -1, t.s.set, [1], [[0]])
    refused(host, -1, t.s.free)
    t.s.h = None
    refused(host, -1, t.attend)
    foreign.free()
    other.close()


def test_under_a_callers_capture(host, hip):
    t = Set(host, hip)
    x, lp = hip.alloc(100), hip.alloc(1)
    host.lib.stub_set_capturing(1)
    for f in (t.store, t.attend, t.evict):
        refused(host, -3, f)
    refused(host, -3, t.s.set, t.lens, t.table)
    refused(host, -3, hip.seqs, 16, 1, 1)
    refused(host, -3, t.s.free)
    refused(host, -3, hip.logprobs, lp.ptr, x.ptr, [0], 100)
    host.lib.stub_set_capturing(0)
    t.attend()


def test_in_a_recorded_step(host, hip):
    """Recorded, then run at flush; a new batch, or the batch's end, runs what was recorded."""
    t = Set(host, hip)
    inv, cs, sn = hip.alloc(2), hip.alloc(2), hip.alloc(2)
    x, lp = hip.alloc(100), hip.alloc(1)
    for end in (hip.flush, lambda: t.s.set(t.lens, t.table), t.s.free):
        hip.rope_table(cs.ptr, sn.ptr, inv.ptr, 0, 1, 2)
        before = host.lib.stub_launches()
        t.store()
        t.attend()
        t.evict()
        hip.logprobs(lp.ptr, x.ptr, [7], 100)
        assert host.lib.stub_launches() == before
        end()
        assert host.lib.stub_launches() >= before + 4
        hip.flush()


def test_the_batch_on_the_device(host, hip):
    """Lengths, positions, row and superblock offsets, superblocks and the table as the kernels read
    them; the superblocks' count rounded up with places for none."""
    s = hip.seqs(16, 70, 40)
    rng = np.random.default_rng(0)
    for n in (1, 3, 70):
        lens = rng.integers(0, 640, n)
        fresh = np.minimum(lens, rng.integers(0, 5, n))
        seen = lens + rng.integers(0, 9, n)
        table = rng.integers(0, 1 << 20, (n, 40))
        s.set(lens, table, fresh=fresh, seen=seen)
        dev = ctypes.c_void_p.from_address(s.h + 32).value  # slm_seqs: four sizes, then the block
        u = np.ctypeslib.as_array((ctypes.c_uint32 * 4096).from_address(dev))
        m = 70
        assert np.array_equal(u[:n], lens) and np.array_equal(u[m:m + n], seen)
        assert np.array_equal(u[2 * m:2 * m + n + 1], np.concatenate([[0], np.cumsum(fresh)]))
        nsb = np.maximum(1, -(-lens // 256))
        assert np.array_equal(u[3 * m + 1:3 * m + n + 2], np.concatenate([[0], np.cumsum(nsb)]))
        want = [(b, z, lens[b], 0) for b in range(n) for z in range(nsb[b])]
        i0 = (16 * m + 8 + 15) // 16 * 4
        assert np.array_equal(u[i0:i0 + 4 * len(want)].reshape(-1, 4), want)
        most = ctypes.c_size_t.from_address(s.h + 24).value
        at = i0 + 4 * most
        w = min(40, -(-int(max(1, (-(-lens // 16)).max())) // 16) * 16)
        got = np.ctypeslib.as_array((ctypes.c_uint32 * (n * w)).from_address(dev + 4 * at)).reshape(n, w)
        for b in range(n):
            used = -(-lens[b] // 16)
            assert np.array_equal(got[b, :used], table[b, :used]) and not got[b, used:].any()


def test_logprobs(host, hip):
    x, lp, ti, tl = hip.alloc(200), hip.alloc(4), hip.alloc(200), hip.alloc(200)
    f = hip.logprobs
    f(lp.ptr, x.ptr, [0, 49, 7, 1], 50)
    f(lp.ptr, x.ptr, [0], 50, top=32, top_ids=ti.ptr, top_lp=tl.ptr)
    refused(host, -5, f, lp.ptr, x.ptr, [50], 50)
    refused(host, -5, f, lp.ptr, x.ptr, [0] * 5, 50)
    refused(host, -5, f, lp.ptr, x.ptr, [0] * 5, 40)  # five rows, four results
    refused(host, -5, f, None, x.ptr, [0], 50)
    refused(host, -5, f, lp.ptr, None, [0], 50)
    refused(host, -1, f, lp.ptr, x.ptr, [0], 0)
    refused(host, -1, f, lp.ptr, x.ptr, [0], 20, top=21, top_ids=ti.ptr, top_lp=tl.ptr)
    refused(host, -3, f, lp.ptr, x.ptr, [0], 50, top=33, top_ids=ti.ptr, top_lp=tl.ptr)
    refused(host, -1, f, lp.ptr, x.ptr, [0], 50, top=3, top_ids=ti.ptr)
    refused(host, -1, f, lp.ptr, x.ptr, [0], 50, top=3, top_lp=ti.ptr)
    refused(host, -1, f, lp.ptr, x.ptr, [0], 50, entropy=lp.ptr)
    refused(host, -1, f, x.ptr, x.ptr, [0], 50)
    refused(host, -1, f, lp.ptr, x.ptr, [0], 50, top=3, top_ids=ti.ptr, top_lp=ti.at(2))
    refused(host, -5, f, lp.ptr, x.ptr, [0, 1], 100, top=32, top_ids=tl.at(137), top_lp=ti.ptr)
    refused(host, -3, f, lp.ptr, x.ptr, [0], (1 << 28) + 1)
    before = host.lib.stub_launches()
    f(lp.ptr, x.ptr, [], 50)
    assert host.lib.stub_launches() == before
    assert host.lib.slm_hip_logprobs(hip.ctx, lp.ptr, None, None, None, 0, x.ptr, None, 1, 50) == -1


def test_many_rows_of_logits(host, hip):
    """More rows than the tokens' way to the device takes at once; the most there may be, and one more."""
    for m in (1 << 20, (1 << 20) + 1, (1 << 22) - 1):
        x, lp = hip.alloc(2 * m), hip.alloc(m)
        before = host.lib.stub_launches()
        hip.logprobs(lp.ptr, x.ptr, np.ones(m), 2)
        assert host.lib.stub_launches() == before + -(-m // (1 << 20))
        ids = np.zeros(m)
        ids[-1] = 2
        refused(host, -5, hip.logprobs, lp.ptr, x.ptr, ids, 2)
        x.free()
        lp.free()
    refused(host, -3, hip.logprobs, None, None, np.zeros(1 << 22), 2)
