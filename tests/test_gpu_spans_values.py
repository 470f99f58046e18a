"""Several new tokens a sequence over paged caches: values whose sizes lie far apart, each channel held to what its own
values are."""

import numpy as np
import pytest

import span_ref as R
from paged_ref import U, Cache
from test_gpu_paged import check, hip, rng_of  # noqa: F401
from test_gpu_spans import queries, run

pytestmark = pytest.mark.gpu


def attend(c, fresh, q, scale, reach=None, gap=0, parent=None):
    """A prompt's (a tree's, with parents) y [rows][H][dh] in 64 bits, and a bound for each element: r sum w |v| + 2^-36 sum |v| + m 2^-118, over the
    channel's m values that the row sees.

    r as in span_ref.attend: a weight's relative error is the score's, twice (its own and the sum's: 2 d), the exponential's and
    division's (8 U), its two fp16 parts' (a rounding to 22 bits, 4 U); a value's two parts' are 4 U, the product of
    second parts that is left out 4 U, and the sums' chains of all slots, rescaled once every 16 at most, and trees of 32 steps. The
    weights' parts are off by 2^-37 of the largest weight at least, the first one's 2^-11 (for the values' second parts)
    by as much: 2^-36 times the value. Where weights are 2^-32 (fp32 products, by element), a sum of values below
    2^-94 is rounded to fp32's least step, 2^-149, a slot: half of it times 2^32 is 2^-118."""
    rows, H, dh = q.shape
    y, bound, at = np.zeros((rows, H, dh)), np.zeros((rows, H, dh)), 0
    for b, f in enumerate(fresh):
        pg, sl = c.where(b)
        old, step = len(pg) - f, np.arange(f)
        sees = np.arange(len(pg)) <= old + step[:, None]
        if parent is not None:
            line, step = R.lines(parent[at:at + f], [f])[0]
            sees[:, old:] = line
        back = old + step[:, None] - np.concatenate([np.arange(old), old + step])
        sees &= (back >= gap) & (back < (1 << 62 if reach is None else reach))
        m = sees.sum(1, keepdims=True)
        for h in range(H):
            k, v = (a[pg, h // (H // c.KH), sl].astype(np.float64) for a in (c.k, c.v))
            qq = q[at:at + f, h].astype(np.float64)
            s = np.where(sees, qq @ k.T * scale, -np.inf)
            e = np.exp(s - np.where(m, s.max(1, keepdims=True), 0))
            w = e / np.where(m, e.sum(1, keepdims=True), 1)
            largest = np.where(sees, np.abs(qq) @ np.abs(k).T * abs(scale), 0).max(1, keepdims=True)
            d = U * ((dh + 10) * largest + 3 * np.abs(np.where(sees, s, 0)).max(1, keepdims=True))
            r = 2 * d + U * (8 + 4 + 4 + 4 + m + m / 16 + 32)
            y[at:at + f, h] = w @ v
            bound[at:at + f, h] = r * (w @ np.abs(v)) + 2.0 ** -36 * (sees @ np.abs(v)) + m * 2.0 ** -118
        at += f
    return y, bound


# heads, key heads, head size, lengths, new tokens: rows of each kind (few, between, many), stretches that are joined
KINDS = [(4, 2, 20, [90], [90]), (2, 1, 32, [150, 70], [16, 9]), (6, 2, 64, [300, 70], [90, 70]), (3, 1, 64, [200], [20]),
         (3, 1, 64, [1500], [120]), (2, 2, 64, [40, 300], [7, 3]), (4, 2, 128, [200, 90], [90, 60]), (2, 1, 256, [150], [40])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size,half", [(1e-3, True), (1e-5, True), (1e-3, False), (1e-6, False), (1e-8, False), (1e-10, False),
                                       (1e-12, False), (1e-14, False), (1e-16, False), (1e-30, False), (1e12, False)])
def test_channels_of_another_size(hip, pkg, kind, size, half):
    """One channel of four."""
    H, KH, dh, lens, fresh = kind
    rng = rng_of(dh, lens[0])
    c = Cache(rng, lens, KH, dh, 16, half)
    c.v[..., 1::4] *= np.float32(size)
    c.v = c.values(c.v)
    q = queries(rng, fresh, H, dh)
    want, bound = attend(c, fresh, q, dh ** -0.5)
    check(run(hip, pkg, c, fresh, q, dh ** -0.5), want, bound, (kind, size))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("smallest,share", [(9, 1.0), (9, 0.001), (15, 0.01), (35, 0.5)])
def test_elements_of_other_sizes(hip, pkg, kind, smallest, share):
    """A share of the values has powers of ten down to 10^-smallest, each its own: early rows, which see few slots, see
    nothing larger in some channels."""
    H, KH, dh, lens, fresh = kind
    rng = rng_of(dh, lens[0], smallest)
    c = Cache(rng, lens, KH, dh, 16)
    power = np.where(rng.random(c.v.shape) < share, -smallest * rng.random(c.v.shape), 0.0)
    c.v = (c.v * 10.0 ** power).astype(np.float32)
    q = queries(rng, fresh, H, dh)
    want, bound = attend(c, fresh, q, dh ** -0.5)
    check(run(hip, pkg, c, fresh, q, dh ** -0.5), want, bound, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("powers", [(0, 10, -10, 0), (-30, 0), (0, -30), (0, 30), (-12, -8, -4, 0, 4, 8, 12), (30, 20, 10, 0)])
def test_tokens_of_other_sizes(hip, pkg, kind, powers):
    """Values of 50 slots after another of a size of their own, in every channel but one."""
    H, KH, dh, lens, fresh = kind
    rng = rng_of(dh, lens[0], len(powers))
    c = Cache(rng, lens, KH, dh, 16)
    for b in range(len(lens)):
        pg, sl = c.where(b)
        size = 10.0 ** np.array(powers, float)[np.arange(len(pg)) // 50 % len(powers)]
        for h in range(KH):
            c.v[pg, h, sl, 1:] = (c.v[pg, h, sl, 1:] * size[:, None]).astype(np.float32)
    q = queries(rng, fresh, H, dh)
    want, bound = attend(c, fresh, q, dh ** -0.5)
    check(run(hip, pkg, c, fresh, q, dh ** -0.5), want, bound, kind)


@pytest.mark.parametrize("size", [1e6, 1e12, 1e30])
@pytest.mark.parametrize("kind", KINDS)
def test_one_value_far_larger_that_few_rows_see(hip, pkg, kind, size):
    """The newest token's in one channel: the rows before it have results of their own size in all of them."""
    H, KH, dh, lens, fresh = kind
    rng = rng_of(dh, lens[0], 5)
    c = Cache(rng, lens, KH, dh, 16)
    for b in range(len(lens)):
        pg, sl = c.where(b)
        c.v[pg[-1], :, sl[-1], 2] = np.float32(size)
    q = queries(rng, fresh, H, dh)
    want, bound = attend(c, fresh, q, dh ** -0.5)
    check(run(hip, pkg, c, fresh, q, dh ** -0.5), want, bound, kind)


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_are_zero(hip, pkg, kind):
    """Channels, tokens and a first stretch of nothing but zeros, of both signs."""
    H, KH, dh, lens, fresh = kind
    rng = rng_of(dh, lens[0], 6)
    c = Cache(rng, lens, KH, dh, 16)
    c.v[..., ::8] = 0.0
    for b in range(len(lens)):
        pg, sl = c.where(b)
        c.v[pg[:70], :, sl[:70]] = -0.0
        c.v[pg[100::9], :, sl[100::9]] = 0.0
    q = queries(rng, fresh, H, dh)
    want, bound = attend(c, fresh, q, dh ** -0.5)
    check(run(hip, pkg, c, fresh, q, dh ** -0.5), want, bound, kind)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("odd", [20, 400])
def test_long_stretches_with_small_values(hip, pkg, dh, odd):
    """Small values in some slots of 1100 that a workgroup has alone, or in most of its tiles."""
    rng = rng_of(dh, odd, 7)
    lens, fresh = [1100] * 16, [64] * 16
    c = Cache(rng, lens, 2, dh, 16)
    for b in range(16):
        pg, sl = c.where(b)
        at = rng.permutation(1036)[:odd]
        c.v[pg[at], :, sl[at], 1:3] *= np.float32(1e-11)
    q = queries(rng, fresh, 32, dh)
    want, bound = attend(c, fresh, q, dh ** -0.5)
    check(run(hip, pkg, c, fresh, q, dh ** -0.5), want, bound)


@pytest.mark.parametrize("scale", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_a_scale_that_is_not_finite(hip, pkg, kind, half, scale):
    """NaN for every row that sees a token, as paged_attend's; zeros for one that sees none."""
    H, KH, dh, lens, fresh = kind
    rng = rng_of(dh, lens[0], 8)
    c = Cache(rng, lens, KH, dh, 16, half)
    q = queries(rng, fresh, H, dh)
    for gap in (0, 30):
        y = run(hip, pkg, c, fresh, q, scale, gap=gap)
        sees = np.concatenate([np.arange(n - f, n) >= gap for n, f in zip(lens, fresh)])
        assert np.isnan(y[sees]).all() and not y[~sees].any()
    g, up = c.upload(hip, pkg, mass=False, born=False)
    s = c.batch(hip)
    s.set(c.lens, c.table, fresh=np.zeros(len(lens)))
    dq, one = hip.upload(q[:len(lens)]), hip.alloc(len(lens) * H * dh)
    hip.paged_attend(s, g, one.ptr, dq.ptr, heads=H, scale=scale)
    assert np.isnan(one.read()).all()


def check_by_largest_score(hip, pkg, kind, half, size):
    """A row's result is the value of its largest score, where that lies above the others by more than scores may be off."""
    H, KH, dh, lens, fresh = kind
    rng = rng_of(dh, lens[0], 9)
    c = Cache(rng, lens, KH, dh, 16, half)
    q = (rng.standard_normal((sum(fresh), H, dh)) * size).astype(np.float32)
    y, at, sure = run(hip, pkg, c, fresh, q, 0.125), 0, 0
    for b, f in enumerate(fresh):
        pg, sl = c.where(b)
        for h in range(H):
            k, v = (a[pg, h // (H // KH), sl] for a in (c.k, c.v))
            qq = q[at:at + f, h].astype(np.float64)
            s, error = qq @ k.T.astype(np.float64), U * (dh + 13) * (np.abs(qq) @ np.abs(k.T))
            for i in range(f):
                m = lens[b] - f + i + 1
                first = int(s[i, :m].argmax())
                rest = np.delete(s[i, :m] + error[i, :m], first)
                if not rest.size or (s[i, first] - error[i, first] - rest.max()) * 0.125 > 40:  # (e^-40 of the others)
                    err = np.abs(y[at + i, h] - v[first]).max()
                    assert err <= 32 * U * np.abs(v[first]).max(), (b, h, i, err)
                    sure += 1
        at += f
    assert sure > 0.9 * sum(fresh) * H


ALONE = [(1, 1, 64, [50] * 24, [1] * 24), (1, 1, 200, [50] * 24, [1] * 24)]  # a row to a workgroup


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e8, 1e9, 1e10, 1e12, 1e30])
@pytest.mark.parametrize("kind", KINDS + ALONE)
def test_large_scores(hip, pkg, kind, half, size):
    """Scores whose last bit is worth many powers of two."""
    check_by_largest_score(hip, pkg, kind, half, size)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("size", [1e35, 2e37])
@pytest.mark.parametrize("kind", KINDS + ALONE)
def test_the_largest_queries(hip, pkg, kind, half, size):
    """Near the end of fp32, with scores that it holds."""
    check_by_largest_score(hip, pkg, kind, half, size)


@pytest.mark.parametrize("share", [0.0002, 0.3])
@pytest.mark.parametrize("reach,gap", [(None, 0), (90, 0), (None, 40), (70, 11)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_small_values_in_windows_and_trees(hip, pkg, kind, tree, reach, gap, share):
    """In some tiles or all of them, seen by some rows."""
    H, KH, dh, lens, fresh = kind
    rng = rng_of(dh, lens[0], gap, tree)
    c = Cache(rng, lens, KH, dh, 16)
    c.v = np.where(rng.random(c.v.shape) < share, c.v * np.float32(1e-12), c.v)
    q = queries(rng, fresh, H, dh)
    parent = R.random_tree(rng, fresh) if tree else None
    want, bound = attend(c, fresh, q, dh ** -0.5, reach, gap, parent)
    check(run(hip, pkg, c, fresh, q, dh ** -0.5, reach, gap, False, parent), want, bound, kind)
