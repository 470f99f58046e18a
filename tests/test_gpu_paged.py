"""Attention of one new token over paged caches, the store before it and the eviction behind it,
against plain 64-bit implementations (paged_ref.py)."""

import numpy as np
import pytest

from paged_ref import U, U16, Cache, read_bits, upload_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip(pkg):
    h = pkg.Hip(0)
    yield h
    h.close()


def rng_of(*key):
    return np.random.default_rng(list(key))


def check(got, want, bound, what=""):
    with np.errstate(invalid="ignore"):
        err = np.abs(got.astype(np.float64) - want)
    bad = np.where(np.isfinite(want), ~(err <= bound), ~((got == want) | (np.isnan(got) & np.isnan(want))))
    assert not bad.any(), (what, np.argwhere(bad)[:4], err[bad][:4], np.broadcast_to(bound, err.shape)[bad][:4])


def attend(hip, pkg, c, q, gap=0, mass=True, born=False, scale=None):
    """y, and the cache's mass after it, from the device."""
    g, up = c.upload(hip, pkg, mass=mass, born=born)
    n, H, dh = q.shape
    s = c.batch(hip)
    s.set(c.lens, c.table, fresh=np.zeros(n), seen=c.seen)
    dq, y = hip.upload(q), hip.upload(np.full(q.size, 7.0, np.float32))
    out = hip.upload(np.full(c.mass.size, 5.0, np.float32)) if mass else None
    hip.paged_attend(s, g, y.ptr, dq.ptr, heads=H, gap=gap, scale=scale if scale is not None else dh ** -0.5,
                     mass_out=out.ptr if mass else None)
    got = y.read().reshape(q.shape), out.read().reshape(c.mass.shape) if mass else None
    for name in ("k", "v"):
        assert np.array_equal(up[name].read(), getattr(c, name).ravel(), equal_nan=True), name
    for b in (*up.values(), dq, y, *([out] if mass else [])):
        b.free()
    s.free()
    return got


SHAPES = [  # heads, key heads, dh, page
    (4, 2, 16, 16), (12, 4, 64, 64), (12, 12, 64, 16), (3, 1, 64, 1), (2, 1, 4, 7), (16, 1, 80, 48), (8, 8, 128, 32),
    (10, 2, 36, 256), (32, 2, 256, 64), (5, 5, 200, 100), (16, 2, 128, 1000), (6, 6, 60, 5)]
BATCHES = [[1], [37], [256], [257], [64, 0, 65], [1, 255, 256, 257, 0, 511, 512, 513], [700, 3, 1023, 64, 0, 300]]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attend(hip, pkg, shape, half):
    H, KH, dh, page = shape
    for i, lens in enumerate(BATCHES):
        rng = rng_of(H, KH, dh, page, i)
        c = Cache(rng, lens, KH, dh, page, half)
        q = (rng.standard_normal((len(lens), H, dh)) * 1.8).astype(np.float32)
        y, mass = attend(hip, pkg, c, q)
        want, wmass, bound, mbound = c.attend(q, dh ** -0.5, born=False)
        check(y, want, bound, lens)
        used = c.used()
        check(mass[used], wmass[used], mbound[used], lens)
        assert np.all(mass[~used] == 5.0)
        plain, _ = attend(hip, pkg, c, q, mass=False)
        assert np.array_equal(plain, y)


@pytest.mark.parametrize("born", [False, True])
@pytest.mark.parametrize("gap", [1, 5, 200, 256, 300, 5000])
def test_gap(hip, pkg, gap, born):
    """Positions behind the gap alone; with `born` in any order; sequences that see nothing."""
    lens = [300, 1, 0, 256, 257, 700, 6]
    rng = rng_of(gap, born)
    seen = np.array(lens) + ([0, 3, 0, 100, 2, 4000, 0] if born else [0] * 7)
    c = Cache(rng, lens, 2, 64, 16, seen=seen)
    if born:
        for b, n in enumerate(lens):
            pg, sl = c.where(b)
            for h in range(2):
                c.born[pg, h, sl] = rng.permutation(int(seen[b]))[:n]
    # what is not seen may hold anything
    for b in range(len(lens)):
        pg, sl = c.where(b)
        for h in range(2):
            pos = c.born[pg, h, sl].astype(np.int64) if born else np.arange(len(pg))
            hid = pos + gap >= int(c.seen[b] if born else c.lens[b])
            c.k[pg[hid], h, sl[hid]] = np.nan
            c.v[pg[hid], h, sl[hid]] = np.inf
    q = rng.standard_normal((len(lens), 6, 64)).astype(np.float32)
    want, wmass, bound, mbound = c.attend(q, 0.125, gap, born)
    g, up = c.upload(hip, pkg, born=born)
    s = c.batch(hip)
    s.set(c.lens, c.table, fresh=np.zeros(len(lens)), seen=c.seen)
    dq, y = hip.upload(q), hip.upload(np.full(q.size, 7.0, np.float32))
    hip.paged_attend(s, g, y.ptr, dq.ptr, heads=6, gap=gap, scale=0.125, mass_out=up["mass"].ptr)  # in place
    check(y.read().reshape(q.shape), want, bound)
    check(up["mass"].read().reshape(c.mass.shape), wmass, mbound)


@pytest.mark.parametrize("half", [False, True])
def test_same_bits_in_any_batch(hip, pkg, half):
    """A sequence alone, among others, on other pages and in another order: the same bits."""
    lens = [1500, 1, 256, 700, 0, 2049]
    rng = rng_of(9, half)
    c = Cache(rng, lens, 4, 64, 48, half)
    q = rng.standard_normal((len(lens), 12, 64)).astype(np.float32)
    y, mass = attend(hip, pkg, c, q)
    for b in range(len(lens)):
        one = Cache(rng_of(1), [lens[b]], 4, 64, 48, half)
        (p0, s0), (p1, s1) = c.where(b), one.where(0)
        for name in ("k", "v", "mass"):
            getattr(one, name)[p1, :, s1] = getattr(c, name)[p0, :, s0]
        y1, m1 = attend(hip, pkg, one, q[b:b + 1])
        assert np.array_equal(y1[0], y[b])
        assert np.array_equal(m1[p1, :, s1], mass[p0, :, s0])


@pytest.mark.parametrize("half", [False, True])
def test_infinities_and_nan_in_visible_keys(hip, pkg, half):
    """Where the formula takes them: a NaN key, infinite scores of both signs (all of them, one
    superblock's, one key's), infinite values under weight and under none."""
    lens = [600] * 7
    c = Cache(rng_of(4), lens, 1, 16, 16, half)
    q = np.abs(rng_of(5).standard_normal((7, 2, 16))).astype(np.float32) + 0.1
    q[2] = q[2].astype(np.float16)  # (fp16 mode's queries: what is past fp16 in them is zero)
    at = [c.where(b) for b in range(7)]
    c.k[at[0][0][400], 0, at[0][1][400]] = np.nan
    c.k[at[1][0], 0, at[1][1]] = -np.inf                          # every score -inf
    c.k[at[2][0][256:512], 0, at[2][1][256:512]] = -np.inf        # a superblock of them
    c.k[at[3][0][5], 0, at[3][1][5]] = np.inf
    c.v[at[4][0][10], 0, at[4][1][10], 3] = np.inf                # weighed
    c.k[at[5][0][20], 0, at[5][1][20]] = -np.inf                  # no weight, an infinite value
    c.v[at[5][0][20], 0, at[5][1][20], 2] = np.inf
    y, _ = attend(hip, pkg, c, q, mass=False)
    want, _, bound, _ = c.attend(q, 0.25, born=False)
    want[1] = np.nan
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(y[np.isinf(want)], want[np.isinf(want)])
    assert np.all(np.isnan(y[0])) and np.all(np.isnan(y[1])) and np.all(np.isfinite(y[2]))
    check(y[[2, 6]], want[[2, 6]], bound[[2, 6]])
    assert fine[4].sum() == 2 * 15


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads", [7, 16])
def test_infinities_under_many_heads(hip, pkg, heads, half):
    """The same with more query heads on the key head; queries of both signs where a key is infinite."""
    c = Cache(rng_of(41, heads), [600] * 5, 1, 64, 16, half)
    q = np.abs(rng_of(42, heads).standard_normal((5, heads, 64))).astype(np.float32) + 0.1
    q[2] = q[2].astype(np.float16)
    at = [c.where(b) for b in range(5)]
    bound = c.attend(q, 0.125, born=False)[2]  # (of all the keys: no less than of those that weigh)
    c.k[at[0][0][400], 0, at[0][1][400]] = np.nan
    c.k[at[1][0], 0, at[1][1]] = -np.inf
    c.k[at[2][0][256:512], 0, at[2][1][256:512]] = -np.inf
    c.k[at[3][0][5], 0, at[3][1][5], 9] = -np.inf                 # no weight: its infinite score is one element's
    c.v[at[4][0][10], 0, at[4][1][10], 3] = np.inf
    y, _ = attend(hip, pkg, c, q, mass=False)
    want = c.attend(q, 0.125, born=False)[0]
    assert np.all(np.isnan(y[:2])) and np.all(want[4, :, 3] == np.inf)
    check(y[2:], want[2:], bound[2:])


@pytest.mark.parametrize("qs,ks,scale", [(1e-6, 1.0, 3e5), (3e6, 1.0, 1e-6), (1e30, 1.0, 1e-30), (1.0, 2e-7, 1e6),
                                         (1.0, 2e4, 2e-5), (1.0, 1e4, 4e-5), (1e-9, 1e-6, 1e15), (0.0, 1.0, 1.0)])
def test_fp16_keys_and_queries_of_any_size(hip, pkg, qs, ks, scale):
    """fp32 queries over fp16 keys: small ones, past fp16's range, keys below its normal numbers and at
    its largest (some of them infinite once rounded)."""
    c = Cache(rng_of(17), [300, 90], 2, 64, 16, True, scale=1.0)
    c.k = c.values(c.k * ks)
    q = (rng_of(18).standard_normal((2, 12, 64)) * qs).astype(np.float32)
    q[..., ::7] *= np.float32(1e-4)
    y, mass = attend(hip, pkg, c, q, scale=scale)
    want, wmass, bound, mbound = c.attend(q, np.float64(np.float32(scale)), born=False)
    check(y, want, bound)
    check(mass[c.used()], wmass[c.used()], mbound[c.used()])


@pytest.mark.parametrize("qs,ks,scale", [(1e-6, 1.0, 3e5), (3e6, 1.0, 1e-6), (1e30, 1.0, 1e-30), (1.0, 2e-7, 1e6),
                                         (1.0, 2e4, 2e-5), (1.0, 1e4, 4e-5), (1e-9, 1e-6, 1e15), (0.0, 1.0, 1.0)])
def test_fp16_keys_and_twelve_heads_of_any_size(hip, pkg, qs, ks, scale):
    """The same with twelve query heads on one key head."""
    c = Cache(rng_of(17), [300, 90], 1, 64, 16, True, scale=1.0)
    c.k = c.values(c.k * ks)
    q = (rng_of(18).standard_normal((2, 12, 64)) * qs).astype(np.float32)
    q[..., ::7] *= np.float32(1e-4)
    y, mass = attend(hip, pkg, c, q, scale=scale)
    want, wmass, bound, mbound = c.attend(q, np.float64(np.float32(scale)), born=False)
    check(y, want, bound)
    check(mass[c.used()], wmass[c.used()], mbound[c.used()])


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(hip, pkg, scale):
    """No scale (the mean), a negative one, one that leaves a single key all the weight."""
    c = Cache(rng_of(6), [300, 40], 2, 32, 16)
    q = rng_of(7).standard_normal((2, 4, 32)).astype(np.float32) * 3
    y, mass = attend(hip, pkg, c, q, scale=scale)
    want, wmass, bound, mbound = c.attend(q, np.float64(np.float32(scale)), born=False)
    check(y, want, bound)
    check(mass[c.used()], wmass[c.used()], mbound[c.used()])


def test_long_cache(hip, pkg):
    """A cache whose values pass 2^32 bytes: a sequence on its last pages and its first."""
    KH, dh, page, pages = 1, 256, 64, (1 << 32) // (256 * 4 * 64) + 40
    g = pkg.Pages(pages=pages, page=page, key_heads=KH, dh=dh)
    k, v = (hip.alloc_pages(pages, KH, page, dh) for _ in range(2))
    g.k, g.v = k.ptr, v.ptr
    rng = rng_of(8)
    n = 200
    kk, vv = (rng.standard_normal((n, dh)).astype(np.float32) for _ in range(2))
    s = hip.seqs(page, 1, 4)
    s.set([n], [[pages - 1, 0, pages - 2, 7]], fresh=[n])
    dk, dv = hip.upload(kk), hip.upload(vv)
    hip.paged_store(s, g, dk.ptr, dv.ptr)
    got = hip.read(k.at((pages - 1) * page * dh), page * dh)
    assert np.array_equal(got, kk[:64].ravel())
    q = rng.standard_normal((1, 1, dh)).astype(np.float32)
    dq, y = hip.upload(q), hip.alloc(dh)
    hip.paged_attend(s, g, y.ptr, dq.ptr, heads=1, scale=1 / 16)
    ref = Cache(rng, [n], 1, dh, n, spare=0)
    ref.k[0, 0], ref.v[0, 0] = kk, vv
    want, _, bound, _ = ref.attend(q, 1 / 16, born=False)
    check(y.read().reshape(q.shape), want, bound)
    for b in (k, v):
        b.free()


@pytest.mark.parametrize("half", [False, True])
def test_cache_of_more_than_2_32_values(hip, pkg, half):
    """Stored, attended, evicted and attended again on a cache's first and last pages."""
    KH, dh, page, pages, n, keep = 1, 256, 64, (1 << 32) // (256 * 64) + 40, 200, 100
    k, v = (hip.alloc_pages(pages, KH, page, dh, half=half) for _ in range(2))
    mass, born = hip.alloc(pages * page), hip.alloc(pages * page)
    g = pkg.Pages(pages=pages, page=page, key_heads=KH, dh=dh, k=k.ptr, v=v.ptr, mass=mass.ptr, born=born.ptr)
    ids = np.array([pages - 1, 0, pages - 2, 7])
    rng = rng_of(9, half)
    ref = Cache(rng, [n], 1, dh, n, half=half, spare=0)
    s = hip.seqs(page, 1, 4)
    s.set([n], [ids], fresh=[n])
    dk, dv = hip.upload(ref.k), hip.upload(ref.v)
    hip.paged_store(s, g, dk.ptr, dv.ptr)
    ref.mass[:] = 0
    for lens in (n, keep):
        q = rng.standard_normal((1, 1, dh)).astype(np.float32)
        dq, y = hip.upload(q), hip.alloc(dh)
        s.set([lens], [ids], seen=[n])
        hip.paged_attend(s, g, y.ptr, dq.ptr, heads=1, scale=1 / 16, mass_out=mass.ptr)
        ref.lens[:] = lens
        want, wmass, bound, mbound = ref.attend(q, 1 / 16)
        check(y.read().reshape(q.shape), want, bound)
        got = mass.read().reshape(pages, page)[ids].ravel()[:n]
        check(got[:lens], wmass.ravel()[:lens], mbound.ravel()[:lens])
        if lens == n:
            ref.mass[:] = got.reshape(ref.mass.shape)
            hip.paged_evict(s, g, mass.ptr, born.ptr, keep=keep, recent=10)
            ref.evict(keep, 10)
            got = read_bits(born).reshape(pages, page)[ids].ravel()[:keep]
            assert np.array_equal(got, ref.born.ravel()[:keep])
    s.free()
    for b in (k, v, mass, born):
        b.free()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("page,dh,KH", [(1, 4, 1), (16, 64, 4), (7, 80, 3), (100, 256, 2)])
def test_store(hip, pkg, page, dh, KH, half):
    """New tokens of several sequences, none to a whole prompt: their slots alone change."""
    lens, fresh = [5, 0, 130, 64, 33, 1], [1, 0, 130, 20, 0, 1]
    rng = rng_of(page, dh, half)
    c = Cache(rng, lens, KH, dh, page, half, seen=[5, 0, 130, 70, 4000, 9])
    g, up = c.upload(hip, pkg)
    s = c.batch(hip)
    s.set(c.lens, c.table, fresh=fresh, seen=c.seen)
    k, v = (rng.standard_normal((sum(fresh), KH, dh)).astype(np.float32) for _ in range(2))
    dk, dv = hip.upload(k), hip.upload(v)
    hip.paged_store(s, g, dk.ptr, dv.ptr)
    c.store(fresh, k, v)
    for name in ("k", "v", "mass"):
        assert np.array_equal(up[name].read(), getattr(c, name).ravel()), name
    assert np.array_equal(read_bits(up["born"]), c.born.ravel())
    # by default one new token each, none in an empty sequence; a cache without mass and born
    s.set(c.lens, c.table)
    g.mass = g.born = None
    fresh = [1, 0, 1, 1, 1, 1]
    k, v = (rng.standard_normal((5, KH, dh)).astype(np.float32) for _ in range(2))
    dk, dv = hip.upload(k), hip.upload(v)
    hip.paged_store(s, g, dk.ptr, dv.ptr)
    mass, born = c.mass.copy(), c.born.copy()
    c.store(fresh, k, v)
    assert np.array_equal(up["k"].read(), c.k.ravel()) and np.array_equal(up["v"].read(), c.v.ravel())
    assert np.array_equal(up["mass"].read(), mass.ravel()) and np.array_equal(read_bits(up["born"]), born.ravel())


def evict(hip, pkg, c, keep, recent, in_place):
    g, up = c.upload(hip, pkg)
    s = c.batch(hip)
    s.set(c.lens, c.table, fresh=np.zeros(len(c.lens)), seen=c.seen)
    mass, born = up["mass"], up["born"]
    if not in_place:
        mass, born = hip.upload(np.full(c.mass.size, 5.0)), upload_bits(hip, np.full(c.born.size, 77))
    hip.paged_evict(s, g, mass.ptr, born.ptr, keep=keep, recent=recent)
    before = c.mass.copy(), c.born.copy()
    c.evict(keep, recent)
    for name in ("k", "v"):
        assert np.array_equal(up[name].read(), getattr(c, name).ravel()), name
    gm, gb = mass.read().reshape(c.mass.shape), read_bits(born).reshape(c.born.shape)
    written = np.zeros(c.mass.shape, bool)
    for b in range(len(c.lens)):
        pg, sl = c.where(b, min(int(c.lens[b]), keep))
        written[pg, :, sl] = True
    rest = (c.mass, c.born) if in_place else (np.full_like(c.mass, 5.0), np.full_like(c.born, 77))
    assert np.array_equal(gm, np.where(written, c.mass, rest[0]), equal_nan=True)
    assert np.array_equal(gb, np.where(written, c.born, rest[1]))
    if not in_place:
        assert np.array_equal(up["mass"].read(), before[0].ravel(), equal_nan=True)
    for b in (*up.values(), *(() if in_place else (mass, born))):
        b.free()
    s.free()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (64, 10), (100, 100), (300, 17), (1000, 1), (5000, 9)])
def test_evict(hip, pkg, keep, recent, half, in_place):
    """Ragged lengths around the budget, weights with ties, zeros, infinities and NaN."""
    lens = [1100, 0, 301, 300, 299, 1, 64, 65, 2, 1025]
    rng = rng_of(keep, recent)
    c = Cache(rng, lens, 3, 20, 16, half, seen=np.array(lens) + [50, 0, 7, 0, 0, 3, 0, 0, 0, 1])
    c.mass = np.exp(2 * rng.standard_normal(c.mass.shape)).astype(np.float32)
    c.mass[rng.random(c.mass.shape) < 0.3] = 0.25
    c.mass[rng.random(c.mass.shape) < 0.1] = 0.0
    c.mass[rng.random(c.mass.shape) < 0.05] = -0.0
    c.mass[rng.random(c.mass.shape) < 0.02] = np.nan
    c.mass[rng.random(c.mass.shape) < 0.02] = np.inf
    c.mass[rng.random(c.mass.shape) < 0.02] = -np.inf
    c.mass[rng.random(c.mass.shape) < 0.02] = -1.5
    for b, n in enumerate(lens):
        pg, sl = c.where(b)
        for h in range(3):
            c.born[pg, h, sl] = rng.permutation(int(c.seen[b]))[:n]
    evict(hip, pkg, c, keep, recent, in_place)


@pytest.mark.parametrize("mass", ["equal", "rising", "falling", "nan"])
def test_evict_orders(hip, pkg, mass):
    """All weights equal (the lower slots stay), rising (the upper ones, all move), falling (none
    does), all NaN; a length past a workgroup's reach at once."""
    lens = [70001, 4097]
    c = Cache(rng_of(3), lens, 1, 4, 64)
    for b, n in enumerate(lens):
        pg, sl = c.where(b)
        c.mass[pg, 0, sl] = dict(equal=np.full(n, 0.5), rising=np.arange(n), falling=-np.arange(n),
                                 nan=np.full(n, np.nan))[mass]
    evict(hip, pkg, c, 3001, 100, True)


def test_shared_pages(hip, pkg):
    """Two sequences with one prefix: attention reads it for both."""
    c = Cache(rng_of(11), [40, 32], 2, 64, 16)
    c.table[1, :2] = c.table[0, :2]
    q = rng_of(12).standard_normal((2, 4, 64)).astype(np.float32)
    y, _ = attend(hip, pkg, c, q, mass=False)
    want, _, bound, _ = c.attend(q, 0.125, born=False)
    check(y, want, bound)


def test_fp16_mode(hip, pkg):
    """y rounded as slm_hip_attend rounds it, the scale too; the weights are not."""
    h = pkg.Hip(0)
    try:
        h.set_fp16(True)
        for lens in ([200, 30], [900, 257]):
            c = Cache(rng_of(13), lens, 2, 64, 16, half=True)
            c.mass = c.mass.astype(np.float16).astype(np.float32)
            q = rng_of(14).standard_normal((2, 4, 64)).astype(np.float16).astype(np.float32)
            y, mass = attend(h, pkg, c, q, scale=0.1)
            want, wmass, bound, mbound = c.attend(q, float(np.float16(0.1)), born=False)
            check(y, want, bound + U16 * np.abs(want) + 2.0 ** -25)
            assert np.array_equal(y, y.astype(np.float16).astype(np.float32))
            used = c.used()
            check(mass[used], wmass[used], mbound[used])
    finally:
        h.close()


def test_agrees_with_attend_over_a_ring(hip, pkg):
    """The same keys in pages and in slm_hip_attend's cache: both within the bound of 64 bits."""
    n, H, KH, dh = 700, 12, 4, 64
    c = Cache(rng_of(15), [n], KH, dh, 64)
    q = rng_of(16).standard_normal((1, H, dh)).astype(np.float32)
    pg, sl = c.where(0)
    k, v = (hip.upload(np.pad(a[pg, :, sl].transpose(1, 0, 2), ((0, 0), (0, 68), (0, 0)))) for a in (c.k, c.v))
    dq, y = hip.upload(q), hip.alloc(q.size)
    hip.attend(y.ptr, dq.ptr, k.ptr, v.ptr, pos=n - 1, m=1, reach=pkg.USIZE_MAX, gap=0, cap=n + 68, heads=H,
               key_heads=KH, dh=dh, scale=0.125)
    got, _ = attend(hip, pkg, c, q, mass=False)
    want, _, bound, _ = c.attend(q, 0.125, born=False)
    check(got, want, bound)
    check(y.read().reshape(q.shape), want, bound)


def serve(hip, pkg, c, steps, keep, recent, recorded):
    """A batch stepped: store, attend with weights noted, evict where it is over its budget, and the
    tokens picked from logits with their log probabilities. Returns what came out, and holds every
    step to the plain implementation."""
    rng = rng_of(21)
    n, H, KH, dh, vocab = len(c.lens), 4, c.KH, c.dh, 97
    g, up = c.upload(hip, pkg)
    s = c.batch(hip, max_pages=c.width + 4)
    head = rng.standard_normal((vocab, H * dh)).astype(np.float32)
    w = hip.upload(head)
    dq, dk, dv, y = (hip.alloc(n * x * dh) for x in (H, KH, KH, H))
    lg, lp, ent, tl = hip.alloc(n * vocab), hip.alloc(n), hip.alloc(n), hip.alloc(n * 3)
    ti = hip.alloc(n * 3)
    inv, cs, sn = hip.upload(np.ones(2, np.float32)), hip.alloc(2), hip.alloc(2)
    free = [p for p in range(c.pages) if p not in set(c.table[c.table < c.pages].tolist())]
    outs = []
    for step in range(steps):
        c.lens, c.seen = c.lens + 1, c.seen + 1
        for b in range(n):
            need = -(-int(c.lens[b]) // c.page)
            if c.table[b, need - 1] >= c.pages:
                c.table[b, need - 1] = free.pop()
        s.set(c.lens, c.table, seen=c.seen)
        q, k, v = (rng.standard_normal((n, x, dh)).astype(np.float32) for x in (H, KH, KH))
        hip.write(dq, q), hip.write(dk, k), hip.write(dv, v)
        ids = rng.integers(0, vocab, n)
        if recorded:
            hip.rope_table(cs.ptr, sn.ptr, inv.ptr, step, 1, 2)
        hip.paged_store(s, g, dk.ptr, dv.ptr)
        hip.paged_attend(s, g, y.ptr, dq.ptr, heads=H, scale=dh ** -0.5, mass_out=up["mass"].ptr)
        hip.linear(lg.ptr, w.ptr, vocab, H * dh, y.ptr, n)
        hip.logprobs(lp.ptr, lg.ptr, ids, vocab, entropy=ent.ptr, top=3, top_ids=ti.ptr, top_lp=tl.ptr)
        hip.paged_evict(s, g, up["mass"].ptr, up["born"].ptr, keep=keep, recent=recent)
        if recorded:
            hip.flush()
        c.store([1] * n, k, v)
        want, wmass, bound, mbound = c.attend(q, dh ** -0.5)
        got = y.read().reshape(q.shape)
        check(got, want, bound)
        x = lg.read().reshape(n, vocab).astype(np.float64)
        l = x - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)) - x.max(1, keepdims=True)
        assert np.abs(lp.read() - l[np.arange(n), ids]).max() < 64 * U * 16
        assert np.array_equal(read_bits(ti).reshape(n, 3), np.argsort(-x, 1, kind="stable")[:, :3])
        # the weights as the device noted them decide what goes
        c.mass = wmass.astype(np.float32)
        gone = c.lens > keep
        if gone.any():
            # (the plain eviction by the device's own weights: they differ in their last bits)
            c.lens = np.minimum(c.lens, keep).astype(np.uint32)
            k1, v1, m1 = (up[i].read().reshape(getattr(c, i).shape) for i in ("k", "v", "mass"))
            b1 = read_bits(up["born"]).reshape(c.born.shape)
            for b in range(n):
                pg, sl = c.where(b)
                for h in range(KH):
                    born = b1[pg, h, sl].astype(int)
                    assert len(set(born.tolist())) == len(born)
                    newest = set(range(max(0, int(c.seen[b]) - recent), int(c.seen[b])))
                    assert newest <= set(born.tolist())
            c.k, c.v, c.mass, c.born = k1, v1, m1, b1
        else:
            check(up["mass"].read().reshape(wmass.shape)[c.used()], wmass[c.used()], mbound[c.used()])
        outs.append((got, lp.read(), m1 if gone.any() else None))
    return outs


@pytest.mark.parametrize("page,lens", [(16, [60, 61, 3]), (64, [300, 200, 290])])
def test_served_together(hip, pkg, page, lens):
    """The operators as a server uses them, call by call and as recorded steps: the same bits."""
    keep = max(lens) + 4
    runs = []
    for recorded in (False, True):
        c = Cache(rng_of(20), lens, 2, 16, page, spare=12)
        c.table = np.concatenate([c.table, np.full((3, 4), 0xfffffff0, np.uint32)], 1)
        runs.append(serve(hip, pkg, c, 12, keep, 8, recorded))
    for a, b in zip(*runs):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
        assert (a[2] is None) == (b[2] is None) and (a[2] is None or np.array_equal(a[2], b[2]))


def test_kept_steps_follow_the_batch(hip, pkg):
    """A recorded step kept as a graph runs again with other lengths, pages and new tokens."""
    c = Cache(rng_of(30), [50, 20, 90], 2, 32, 16, spare=6)
    c.table = np.concatenate([c.table, np.full((3, 2), 0xfffffff0, np.uint32)], 1)
    free = [p for p in range(c.pages) if p not in set(c.table[c.table < c.pages].tolist())]
    g, up = c.upload(hip, pkg, born=False)
    s = c.batch(hip, max_pages=16)
    rng = rng_of(31)
    dq, dk, dv, y = (hip.alloc(3 * x * 32) for x in (4, 2, 2, 4))
    inv, cs, sn = hip.upload(np.ones(2, np.float32)), hip.alloc(2), hip.alloc(2)
    before = hip.graph_stats()["captured"]
    for step in range(9):
        if step:
            c.lens, c.seen = c.lens + 1, c.seen + 1
        if step == 5:  # the batch's order changes, and with it every row of the table
            c.lens, c.seen, c.table = c.lens[::-1].copy(), c.seen[::-1].copy(), c.table[::-1].copy()
        for b in range(3):
            need = -(-int(c.lens[b]) // 16)
            if c.table[b, need - 1] >= c.pages:
                c.table[b, need - 1] = free.pop()
        q, k, v = (rng.standard_normal((3, x, 32)).astype(np.float32) for x in (4, 2, 2))
        hip.write(dq, q), hip.write(dk, k), hip.write(dv, v)
        s.set(c.lens, c.table)
        hip.rope_table(cs.ptr, sn.ptr, inv.ptr, step, 1, 2)
        hip.paged_store(s, g, dk.ptr, dv.ptr)
        hip.paged_attend(s, g, y.ptr, dq.ptr, heads=4, scale=0.2, mass_out=up["mass"].ptr)
        hip.flush()
        c.store([1] * 3, k, v)
        want, wmass, bound, mbound = c.attend(q, np.float64(np.float32(0.2)), born=False)
        check(y.read().reshape(q.shape), want, bound)
        got = up["mass"].read().reshape(wmass.shape)
        check(got, wmass, mbound)
        c.mass = got
    assert hip.graph_stats()["captured"] > before


def test_kept_steps_share_the_workspace(pkg):
    """Two recorded steps kept as graphs, run in turn, and between them calls of their own that need
    more of the workspace than either: every run gives what the first gave."""
    hip = pkg.Hip(0)
    rng = rng_of(32)
    H, KH, dh, vocab = 4, 2, 64, 40000
    sets, x = [], hip.upload(rng.standard_normal((2, vocab)))
    for lens in ([700, 90], [1500, 3, 400], [3000] * 6):
        c = Cache(rng, lens, KH, dh, 16)
        g, up = c.upload(hip, pkg, born=False)
        q, n = rng.standard_normal((len(lens), H, dh)).astype(np.float32), len(lens)
        s = c.batch(hip)
        s.set(c.lens, c.table, fresh=np.zeros(n))
        sets.append((c, g, s, q, hip.upload(q), hip.alloc(q.size), hip.alloc(c.mass.size), up))
    inv, cs, sn = hip.upload(np.ones(2, np.float32)), hip.alloc(2), hip.alloc(2)
    lp, ti, tl = hip.alloc(2), hip.alloc(64), hip.alloc(64)
    first = {}

    def run(i, recorded, step):
        c, g, s, q, dq, y, mass, up = sets[i]
        hip.write(y, np.zeros(q.size)), hip.write(lp, np.zeros(2)), hip.write(tl, np.zeros(64))
        if recorded:
            hip.rope_table(cs.ptr, sn.ptr, inv.ptr, step, 1, 2)
        hip.paged_attend(s, g, y.ptr, dq.ptr, heads=H, scale=0.1, mass_out=mass.ptr)
        hip.logprobs(lp.ptr, x.ptr, [5, 39999], vocab, top=32, top_ids=ti.ptr, top_lp=tl.ptr)
        if recorded:
            hip.flush()
        out = [b.read() for b in (y, lp, ti, tl)] + [mass.read().reshape(c.mass.shape)[c.used()]]
        if i not in first:
            want, wmass, bound, mbound = c.attend(q, np.float64(np.float32(0.1)), born=False)
            check(out[0].reshape(q.shape), want, bound)
            check(out[4], wmass[c.used()], mbound[c.used()])
            first[i] = out
        for a, b in zip(out, first[i]):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))

    before = hip.graph_stats()["captured"]
    for step in range(8):
        run(0, True, step)
        if step >= 4:
            run(2, False, step)
        run(1, True, step)
        run(0, False, step)
    assert hip.graph_stats()["captured"] >= before + 2
    hip.close()


def test_refusals(hip, pkg):
    """Refused calls leave every buffer as it was (test_batch_host.py has all of the refusals)."""
    c = Cache(rng_of(40), [40, 300], 2, 64, 16)
    g, up = c.upload(hip, pkg)
    s = c.batch(hip)
    q, y = hip.upload(np.ones(2 * 4 * 64)), hip.upload(np.full(2 * 4 * 64, 7.0))
    k = hip.upload(np.ones(2 * 2 * 64))

    def bad(code, f, *a, **k):
        with pytest.raises(pkg.SlmError) as e:
            f(*a, **k)
        assert e.value.code == code, e.value

    def unchanged():
        assert np.all(y.read() == 7.0) and np.array_equal(read_bits(up["born"]), c.born.ravel())
        for name in ("k", "v", "mass"):
            assert np.array_equal(up[name].read(), getattr(c, name).ravel())

    s.set(c.lens, c.table)
    bad(-1, hip.paged_attend, s, g, y.ptr, q.ptr, 3, 1.0)
    bad(-5, hip.paged_attend, s, g, y.ptr, q.ptr, 6, 1.0)
    bad(-1, hip.paged_evict, s, g, up["mass"].ptr, up["born"].ptr, 5, 6)
    s.set([33, 20], [[1, 2, 3], [4, c.pages, 0]])  # a page that the cache does not have
    bad(-5, hip.paged_attend, s, g, y.ptr, q.ptr, 4, 1.0)
    bad(-5, hip.paged_store, s, g, k.ptr, k.ptr)
    bad(-5, hip.paged_evict, s, g, up["mass"].ptr, up["born"].ptr, 5, 1)
    s.set([33, 20], [[1, 2, 3], [4, 3, 0]])  # a page twice
    bad(-1, hip.paged_attend, s, g, y.ptr, q.ptr, 4, 1.0, mass_out=up["mass"].ptr)
    bad(-1, hip.paged_store, s, g, k.ptr, k.ptr)
    bad(-1, hip.paged_evict, s, g, up["mass"].ptr, up["born"].ptr, 8, 2)
    unchanged()
    s.set([], np.zeros((0, 1)))  # no sequences: nothing to do
    hip.paged_attend(s, g, y.ptr, q.ptr, 4, 1.0, mass_out=up["mass"].ptr)
    hip.paged_evict(s, g, up["mass"].ptr, up["born"].ptr, 8, 2)
    unchanged()
