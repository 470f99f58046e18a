"""The forms of the paged operators that sizes choose: every number of query heads on a key head in
every class of head sizes, both joins of long caches' superblocks on both sides of their rule, and
evictions of more slots than a workgroup's memory holds. Against plain 64-bit implementations
(paged_ref.py)."""

import numpy as np
import pytest

from paged_ref import Cache
from test_gpu_paged import attend, check, evict, rng_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip(pkg):
    h = pkg.Hip(0)
    yield h
    h.close()


def hold(hip, pkg, c, q):
    y, mass = attend(hip, pkg, c, q)
    want, wmass, bound, mbound = c.attend(q, q.shape[2] ** -0.5, born=False)
    check(y, want, bound)
    used = c.used()
    check(mass[used], wmass[used], mbound[used])
    assert np.all(mass[~used] == 5.0)
    plain, _ = attend(hip, pkg, c, q, mass=False)
    assert np.array_equal(plain, y)
    return y, mass


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 9, 13])
@pytest.mark.parametrize("dh", [8, 64, 68, 128, 132, 256])
def test_every_group_and_head_size(hip, pkg, dh, group, half):
    for i, lens in enumerate(([255, 1, 0], [257, 700, 0, 66])):
        rng = rng_of(dh, group, half, i)
        c = Cache(rng, lens, 2, dh, 16, half)
        hold(hip, pkg, c, (rng.standard_normal((len(lens), 2 * group, dh)) * 1.8).astype(np.float32))


# up to 256 / (head size / 4) superblocks each has a group of a four-wave join's threads of its own; past 64
# and 512 superblocks the sums are read in more rounds
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("H,KH,dh,n", [(4, 2, 64, 4096), (4, 2, 64, 4097), (5, 1, 64, 17000), (2, 1, 256, 1024),
                                       (2, 1, 256, 1025), (6, 1, 256, 5000), (2, 2, 4, 16384), (3, 1, 4, 17000),
                                       (2, 1, 4, 65536), (2, 1, 4, 65537), (3, 1, 4, 131072), (3, 1, 4, 131600),
                                       (6, 1, 12, 140000)])
def test_joins(hip, pkg, H, KH, dh, n, half):
    rng = rng_of(H, dh, n, half)
    c = Cache(rng, [300, n, 5], KH, dh, 64, half)
    hold(hip, pkg, c, rng.standard_normal((3, H, dh)).astype(np.float32))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lens", [[200, 300, 5000], [4096, 4097], [100, 256, 131]])
def test_same_bits_beside_longer_ones(hip, pkg, lens, half):
    """A sequence alone has the bits that it has beside one long enough for the other join."""
    c = Cache(rng_of(50, half), lens, 2, 64, 48, half)
    q = rng_of(51).standard_normal((len(lens), 6, 64)).astype(np.float32)
    y, mass = attend(hip, pkg, c, q)
    for b in range(len(lens)):
        one = Cache(rng_of(1), [lens[b]], 2, 64, 48, half)
        (p0, s0), (p1, s1) = c.where(b), one.where(0)
        for name in ("k", "v", "mass"):
            getattr(one, name)[p1, :, s1] = getattr(c, name)[p0, :, s0]
        y1, m1 = attend(hip, pkg, one, q[b:b + 1])
        assert np.array_equal(y1[0], y[b]) and np.array_equal(m1[p1, :, s1], mass[p0, :, s0])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page", [7, 64])
@pytest.mark.parametrize("keep,recent", [(39900, 0), (36300, 100), (30000, 29999), (5, 2), (50000, 40)])
def test_long_evictions(hip, pkg, keep, recent, page, in_place):
    """Sequences about and past the 36352 slots whose ranks a workgroup holds: few moves and many, more
    kept than there are, weights with ties at the border, infinities and NaN, positions in any order."""
    lens = [40000, 36353, 36352, 36351, 100]
    rng = rng_of(keep, page)
    c = Cache(rng, lens, 2, 4, page, seen=np.array(lens) + [900, 0, 3, 0, 0])
    c.mass = np.round(rng.random(c.mass.shape) * 20).astype(np.float32)
    c.mass[rng.random(c.mass.shape) < 0.02] = np.nan
    c.mass[rng.random(c.mass.shape) < 0.02] = np.inf
    for b, n in enumerate(lens):
        pg, sl = c.where(b)
        for h in range(2):
            c.born[pg, h, sl] = rng.permutation(int(c.seen[b]))[:n]
    evict(hip, pkg, c, keep, recent, in_place)


@pytest.mark.parametrize("page", [7, 64])
def test_long_evictions_of_weights_that_differ(hip, pkg, page):
    """No two weights alike: no ties at the border."""
    lens = [40001, 300]
    c = Cache(rng_of(60, page), lens, 2, 4, page)
    for b, n in enumerate(lens):
        pg, sl = c.where(b)
        for h in range(2):
            c.mass[pg, h, sl] = rng_of(61, b, h).permutation(n).astype(np.float32) * 0.37
    evict(hip, pkg, c, 39990, 7, False)
