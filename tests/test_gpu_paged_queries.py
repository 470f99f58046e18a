"""Attention over paged caches with queries whose sizes lie far apart: a head's result is that of its
own query, whatever its siblings on the key head hold, and an element's part is its own. Against
plain 64-bit implementations (paged_ref.py), whose bounds go by each head's own query."""

import numpy as np
import pytest

from paged_ref import Cache
from test_gpu_paged import attend, check, rng_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip(pkg):
    h = pkg.Hip(0)
    yield h
    h.close()


# heads, key heads, head size: 1, 2, 3, 4, 5 to 8 and more query heads a key head, three classes of
# head sizes and odd ones
SHAPES = [(2, 1, 4), (3, 1, 64), (8, 2, 64), (6, 3, 20), (12, 2, 36), (8, 1, 64), (12, 1, 64), (8, 2, 128), (5, 1, 100),
          (16, 1, 128), (3, 1, 256), (4, 1, 200), (16, 2, 256), (12, 1, 256)]
LENS = [[300, 90], [90, 40]]  # some superblocks a sequence, one each


def case(shape, lens, half, *key):
    H, KH, dh = shape
    rng = rng_of(H, KH, dh, len(key), *key)
    c = Cache(rng, lens, KH, dh, 16, half)
    return c, rng.standard_normal((len(lens), H, dh)).astype(np.float32)


def hold(hip, pkg, c, q, bounds=None):
    """Checks y and the noted weights. bounds: (of y, of the weights), where the cache's own have none."""
    dh = q.shape[2]
    y, mass = attend(hip, pkg, c, q)
    with np.errstate(all="ignore"):
        want, wmass, bound, mbound = c.attend(q, dh ** -0.5, born=False)
    if bounds:
        bound, mbound = bounds
    check(y, want, bound)
    used = c.used()
    check(mass[used], wmass[used], mbound[used])
    return y, want


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [1e-30, 1e-9, 1e9, 1e15, 1e20, 1e30])
def test_heads_of_different_sizes(hip, pkg, shape, size, half):
    """One head's query far larger or smaller than its siblings'."""
    for i, lens in enumerate(LENS):
        c, q = case(shape, lens, half, i)
        q[:, 1] *= np.float32(size)
        y, want = hold(hip, pkg, c, q)
        assert np.isfinite(want).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_a_head_that_is_no_number(hip, pkg, shape, what, half):
    """An infinite or NaN element makes NaNs of its own head (its scores are infinite, of both signs),
    and of the weights, which are sums over heads; the siblings' outputs are their own."""
    for i, lens in enumerate(LENS):
        c, q = case(shape, lens, half, i)
        q[0, 1, 2] = what
        y, want = hold(hip, pkg, c, q)
        assert np.isnan(want[0, 1]).all() and np.isfinite(want[0, 0]).all() and np.isfinite(want[1]).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [1e10, 1e20, 1e38])
def test_a_large_element_that_meets_zeros(hip, pkg, shape, size, half):
    """A query element of any size against keys that are zero there: the others decide."""
    for i, lens in enumerate(LENS):
        c, q = case(shape, lens, half, i)
        c.k[..., 1] = 0
        q[:, 0, 1] = size
        q[:, 1, 1] = -size
        hold(hip, pkg, c, q)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_small_elements_at_infinite_keys(hip, pkg, shape, half):
    """An infinite key element counts with the query element's sign, however small that is: a score of
    -inf (no weight) for positive ones at -inf, +inf (a NaN) for negative ones, NaN for zeros."""
    for i, lens in enumerate(LENS):
        c, q = case(shape, lens, half, i)
        q[:, :, 3] = 1e-12
        q[0, 0, 3] = 1e-39
        with np.errstate(all="ignore"):
            _, _, *bounds = c.attend(q, shape[2] ** -0.5, born=False)  # (of all the keys: no less than of those that weigh)
        pg, sl = c.where(0)
        c.k[pg[5], :, sl[5], 3] = -np.inf
        c.k[pg[-1], :, sl[-1], 3] = -np.inf
        y, want = hold(hip, pkg, c, q, bounds)
        assert np.isfinite(want).all()
        q[0, 1, 3] = -1e-12
        y, want = hold(hip, pkg, c, q, bounds)
        assert np.isnan(want[0, 1]).all() and np.isfinite(want[0, 0]).all()
        q[0, 1, 3] = 0
        y, want = hold(hip, pkg, c, q, bounds)
        assert np.isnan(want[0, 1]).all() and np.isfinite(want[0, 0]).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_infinite_keys_under_full_queries(hip, pkg, shape, half):
    """A superblock (and a whole wave's part of one) of keys that are -inf throughout, under positive
    queries with all of fp32's digits: no weight. Under queries of both signs: NaN."""
    c, q = case(shape, [600, 90], half)
    with np.errstate(all="ignore"):
        q = np.abs(q) + np.float32(0.1)
        _, _, *bounds = c.attend(q, shape[2] ** -0.5, born=False)
    for b, part in ((0, slice(256, 512)), (1, slice(0, 64))):
        pg, sl = c.where(b)
        c.k[pg[part], :, sl[part]] = -np.inf
    y, want = hold(hip, pkg, c, q, bounds)
    assert np.isfinite(want).all()
    q[:, 1, 1] *= -1
    y, want = hold(hip, pkg, c, q, bounds)
    assert np.isnan(want[:, 1]).all() and np.isfinite(want[:, 0]).all()
