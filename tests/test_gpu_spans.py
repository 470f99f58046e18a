"""Several new tokens a sequence over paged caches: attention of prompts and of trees of drafted tokens, the
trees' verification and the path that is kept, against plain 64-bit implementations (span_ref.py)."""

import numpy as np
import pytest

import span_ref as R
from paged_ref import U16, Cache, read_bits, upload_bits
from test_gpu_paged import check, hip, rng_of  # noqa: F401

pytestmark = pytest.mark.gpu


def run(hip, pkg, c, fresh, q, scale, reach=None, gap=0, born=False, parent=None, extra=3):
    """y from the device; the cache and the rows of y behind the last new token stay as they were."""
    g, up = c.upload(hip, pkg, mass=False, born=born)
    rows, H, dh = q.shape
    s = c.batch(hip)
    s.set(c.lens, c.table, fresh=fresh, seen=c.seen)
    if parent is not None:
        s.tree(parent)
    dq, y = hip.upload(q), hip.upload(np.full((rows + extra) * H * dh, 7.0, np.float32))
    call = hip.paged_prompt if parent is None else hip.paged_tree
    call(s, g, y.ptr, dq.ptr, heads=H, scale=scale, reach=reach, gap=gap)
    got = y.read().reshape(rows + extra, H, dh)
    assert np.all(got[rows:] == 7.0)
    for name in ("k", "v"):
        assert np.array_equal(up[name].read(), getattr(c, name).ravel(), equal_nan=True), name
    for b in (*up.values(), dq, y):
        b.free()
    s.free()
    return got[:rows]


def queries(rng, fresh, H, dh):
    return (rng.standard_normal((int(np.sum(fresh)), H, dh)) * 1.8).astype(np.float32)


SHAPES = [  # heads, key heads, dh, page
    (4, 2, 16, 16), (12, 4, 64, 64), (12, 12, 64, 16), (3, 1, 64, 1), (2, 1, 4, 7), (16, 1, 80, 48), (8, 8, 128, 32),
    (10, 2, 36, 256), (32, 2, 256, 64), (5, 5, 200, 100), (20, 1, 64, 1000), (6, 6, 60, 5), (48, 1, 32, 64)]
BATCHES = [  # lengths, new tokens
    ([1], [1]), ([37], [37]), ([20], [3]), ([300], [1]), ([131], [130]), ([64, 0, 65], [1, 0, 65]),
    ([40, 7, 1, 0, 129, 500], [0, 7, 1, 0, 33, 5]), ([700, 3, 520, 64], [129, 3, 257, 16])]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_prompt(hip, pkg, shape, half):
    H, KH, dh, page = shape
    for i, (lens, fresh) in enumerate(BATCHES):
        print(shape, half, lens, fresh, flush=True)
        rng = rng_of(H, KH, dh, page, i)
        c = Cache(rng, lens, KH, dh, page, half)
        q = queries(rng, fresh, H, dh)
        y = run(hip, pkg, c, fresh, q, dh ** -0.5)
        want, bound = R.attend(c, fresh, q, dh ** -0.5)
        check(y, want, bound, lens)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_tree(hip, pkg, shape, half):
    H, KH, dh, page = shape
    for i, (lens, fresh) in enumerate(BATCHES + [([256, 300], [256, 200])]):
        if max(fresh) > 256:
            fresh = [min(f, 256) for f in fresh]
        print(shape, half, lens, fresh, flush=True)
        rng = rng_of(H, KH, dh, page, i, 1)
        c = Cache(rng, lens, KH, dh, page, half)
        q = queries(rng, fresh, H, dh)
        parent = R.random_tree(rng, fresh, roots=i % 2 == 1)
        y = run(hip, pkg, c, fresh, q, dh ** -0.5, parent=parent)
        want, bound = R.attend(c, fresh, q, dh ** -0.5, parent=parent)
        check(y, want, bound, lens)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("born", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("reach,gap", [(1, 0), (2, 0), (40, 0), (None, 1), (None, 3), (200, 37), (None, 300), (5, 5), (3, 7),
                                       (None, 5000), (2 ** 40, 2 ** 40), (300, 0)])
def test_reach_and_gap(hip, pkg, half, born, tree, reach, gap):
    """What lies between them alone; positions in any order; rows that see nothing; what no row sees may
    hold anything."""
    lens, fresh = [300, 1, 0, 256, 300, 6, 90], [40, 1, 0, 3, 200, 6, 17]
    rng = rng_of(reach or 0, gap, born, tree)
    seen = np.array(lens) + ([0, 3, 0, 100, 2, 0, 4000] if born else [0] * 7)
    c = Cache(rng, lens, 2, 64, 16, half, seen=seen)
    parent = R.random_tree(rng, fresh) if tree else None
    if born:
        for b, n in enumerate(lens):
            pg, sl = c.where(b)
            for h in range(2):
                old = n - fresh[b]
                c.born[pg[:old], h, sl[:old]] = rng.permutation(int(seen[b]) - fresh[b])[:old]
                c.born[pg[old:], h, sl[old:]] = int(seen[b]) - fresh[b] + np.arange(fresh[b])
    q = queries(rng, fresh, 6, 64)
    want, bound = R.attend(c, fresh, q, 0.125, reach, gap, born, parent)
    check(run(hip, pkg, c, fresh, q, 0.125, reach, gap, born, parent), want, bound)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("heads", [2, 6])
def test_what_is_not_seen_may_hold_anything(hip, pkg, half, tree, heads):
    """Infinities and NaN in new tokens that some rows do not see, in slots behind a window and behind the
    sequences' ends, and in pages of no sequence."""
    lens, fresh = [300, 140, 33], [40, 140, 1]
    rng = rng_of(half, tree, heads)
    c = Cache(rng, lens, 2, 64, 16, half)
    parent = R.random_tree(rng, fresh) if tree else None
    used = c.used()
    for a, x in ((c.k, np.nan), (c.v, np.inf)):
        a[~used] = x
    for b, n in enumerate(lens):  # the last new tokens
        pg, sl = c.where(b)
        last = [n - 1, n - 2][:fresh[b] - 1]
        c.k[pg[last], :, sl[last]] = np.inf
        c.v[pg[last], :, sl[last]] = np.nan
    pg, sl = c.where(0)  # behind the window of all
    c.k[pg[:100], :, sl[:100]] = np.nan
    c.v[pg[:100], :, sl[:100]] = -np.inf
    q = queries(rng, fresh, heads, 64)
    want, bound = R.attend(c, fresh, q, 0.125, 150, 0, False, parent)
    y = run(hip, pkg, c, fresh, q, 0.125, 150, 0, False, parent)
    check(y, want, bound)
    assert np.isfinite(want).any() and not np.isfinite(want).all()


@pytest.mark.parametrize("size", [1e4, 1e6, 3e8, 1e30])
@pytest.mark.parametrize("which", ["keys", "values", "both"])
@pytest.mark.parametrize("seen", [False, True])
def test_far_larger_keys_and_values_beside_others(hip, pkg, size, which, seen):
    """Finite ones many times the others' size in the same tile: of tokens that a row does not see, and of
    tokens that rows see (then without weight for most rows, or all of it)."""
    lens, fresh = [300, 70], [90, 70]
    rng = rng_of(int(np.log10(size)), seen)
    c = Cache(rng, lens, 2, 64, 16)
    for b, n in enumerate(lens):
        pg, sl = c.where(b)
        at = [3, 65, 130][:n // 60] if seen else [n - 1, n - 30]
        for name, x in (("k", c.k), ("v", c.v)):
            if which in ("both", "keys" if name == "k" else "values"):
                x[pg[at], :, sl[at]] *= np.float32(size)
    q = queries(rng, fresh, 6, 64)
    want, bound = R.attend(c, fresh, q, 0.125)
    check(run(hip, pkg, c, fresh, q, 0.125), want, bound)


@pytest.mark.parametrize("fresh", [3, 130])
@pytest.mark.parametrize("n", [200, 5000])
def test_the_largest_values(hip, pkg, fresh, n):
    """fp32's largest: no sum of weighted ones overflows."""
    rng = rng_of(n, fresh)
    c = Cache(rng, [n], 1, 64, 16)
    c.v = (np.sign(c.v) * np.float32(3.3e38)).astype(np.float32)
    q = queries(rng, [fresh], 3, 64)
    want, bound = R.attend(c, [fresh], q, 0.125)
    check(run(hip, pkg, c, [fresh], q, 0.125), want, bound)


@pytest.mark.parametrize("half", [False, True])
def test_infinities_and_nan_in_visible_keys(hip, pkg, half):
    lens, fresh = [600] * 7, [20] * 7
    c = Cache(rng_of(4), lens, 1, 16, 16, half)
    q = np.abs(rng_of(5).standard_normal((140, 2, 16))).astype(np.float32) + 0.1
    at = [c.where(b) for b in range(7)]
    c.k[at[0][0][400], 0, at[0][1][400]] = np.nan
    c.k[at[1][0], 0, at[1][1]] = -np.inf                          # every score -inf
    c.k[at[2][0][256:512], 0, at[2][1][256:512]] = -np.inf
    c.k[at[3][0][5], 0, at[3][1][5]] = np.inf
    c.v[at[4][0][10], 0, at[4][1][10], 3] = np.inf                # weighed
    c.k[at[5][0][20], 0, at[5][1][20]] = -np.inf                  # no weight, an infinite value
    c.v[at[5][0][20], 0, at[5][1][20], 2] = np.inf
    want, bound = R.attend(c, fresh, q, 0.25)
    check(run(hip, pkg, c, fresh, q, 0.25), want, bound)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("sizes", [(1.0, 20000.0, 2e-5), (1e4, 1e-7, 1.0), (1e-30, 1e-30, 1.0), (1e30, 1e-4, 1e-27),
                                   (3e38, 1e-38, 1e-39), (0.0, 0.0, 1.0)])
@pytest.mark.parametrize("fresh", [3, 130])
def test_queries_of_any_size(hip, pkg, half, sizes, fresh):
    """Elements of a query (and of the heads beside it) whose sizes lie far apart, and keys that bring the
    small ones up."""
    a, b, scale = sizes
    rng = rng_of(7, half, fresh)
    c = Cache(rng, [200], 1, 64, 16, half)
    q = queries(rng, [fresh], 3, 64)
    q[:, 0, :32] *= a
    q[:, 0, 32:] *= b
    q[:, 1] *= np.float32(a) * np.float32(1e-3)
    big = max(a, b, 1e-30) / max(min(a, b), 1e-30)
    c.k[..., (0 if a < b else 32):(32 if a < b else 64)] *= np.float32(min(big, 2e4))
    c.k = c.values(np.clip(c.k, -6e4, 6e4))
    want, bound = R.attend(c, [fresh], q, scale)
    with np.errstate(all="ignore"):
        check(run(hip, pkg, c, [fresh], q, scale), want, bound + 1e-37)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 30.0])
def test_scales(hip, pkg, half, scale):
    rng = rng_of(11)
    c = Cache(rng, [150, 40], 2, 64, 16, half)
    q = queries(rng, [70, 5], 4, 64)
    want, bound = R.attend(c, [70, 5], q, scale)
    check(run(hip, pkg, c, [70, 5], q, scale), want, bound)


@pytest.mark.parametrize("half", [False, True])
def test_long_caches(hip, pkg, half):
    """Rows whose slots are cut over many workgroups, and prompts of several tiles beside single tokens."""
    for lens, fresh, H, KH in (([9001], [25], 12, 4), ([4000, 1, 900, 2500], [3, 1, 800, 1], 6, 2), ([20000, 10], [1, 1], 4, 4)):
        rng = rng_of(lens[0], half)
        c = Cache(rng, lens, KH, 64, 64, half)
        q = queries(rng, fresh, H, 64)
        for parent in (None, R.random_tree(rng, fresh)) if max(fresh) <= 256 else (None,):
            want, bound = R.attend(c, fresh, q, 0.125, parent=parent)
            check(run(hip, pkg, c, fresh, q, 0.125, parent=parent), want, bound)


def test_a_row_alone_is_paged_attend(hip, pkg):
    """A prompt token by token through slm_hip_paged_attend gives what it gives at once."""
    rng = rng_of(21)
    c = Cache(rng, [60, 33], 4, 64, 16)
    q = queries(rng, [20, 33], 12, 64)
    y = run(hip, pkg, c, [20, 33], q, 0.125)
    g, up = c.upload(hip, pkg, mass=False, born=False)
    s = c.batch(hip)
    at = 0
    for b, f in enumerate([20, 33]):
        for i in range(f):
            lens = np.zeros(2, np.uint32)
            lens[b] = c.lens[b] - f + i + 1
            s.set(lens, c.table, fresh=np.zeros(2))
            dq, out = hip.upload(np.repeat(q[at + i][None], 2, 0)), hip.alloc(2 * 12 * 64)
            hip.paged_attend(s, g, out.ptr, dq.ptr, heads=12, scale=0.125)
            one = out.read().reshape(2, 12, 64)[b]
            assert np.abs(one - y[at + i]).max() < 3e-6
        at += f


def test_fp16_mode(pkg):
    hip = pkg.Hip(0)
    hip.set_fp16(True)
    rng = rng_of(31)
    c = Cache(rng, [90, 10], 2, 64, 16, half=True)
    q = queries(rng, [50, 10], 6, 64).astype(np.float16).astype(np.float32)
    parent = R.random_tree(rng, [50, 10])
    for p in (None, parent):
        y = run(hip, pkg, c, [50, 10], q, 0.125, parent=p)
        want, bound = R.attend(c, [50, 10], q, 0.125, parent=p)
        assert np.array_equal(y, y.astype(np.float16).astype(np.float32))
        check(y, want, bound + U16 * np.abs(want) + 2.0 ** -25)
    hip.close()


@pytest.mark.parametrize("seed", range(6))
def test_verify(hip, pkg, seed):
    rng = rng_of(41, seed)
    vocab = [1, 5, 97, 2049, 32000, 65003][seed]
    for fresh in ([1], [25], [3, 0, 64, 1, 256], [0, 0], [7] * 40):
        rows = int(np.sum(fresh))
        parent = R.random_tree(rng, fresh, roots=seed % 2 == 1)
        ids = rng.integers(0, min(vocab, 4 if seed % 2 else vocab), rows).astype(np.uint32)
        x = (np.round(rng.standard_normal((rows, vocab)) * 2) / 2).astype(np.float32)  # (ties)
        first = np.repeat(np.cumsum(fresh) - fresh, fresh)
        on = (parent >= 0) & (rng.random(rows) < 0.8)
        x[(first + parent)[on], ids[on]] = 30.0
        if seed == 2 and rows:
            x[rng.integers(rows), 0] = np.nan
            x[rng.integers(rows)] = np.nan
            x[rng.integers(rows)] = -np.inf
            x[rng.integers(rows), vocab - 1] = np.inf
            x[rng.integers(rows), 1:] = np.nan
        s = hip.seqs(16, len(fresh), 40)
        s.set(np.array(fresh) + 5, np.zeros((len(fresh), 40)), fresh=fresh)
        s.tree(parent, ids)
        dx = hip.upload(x) if rows else hip.alloc(1)
        n = len(fresh)
        count, path, after = (upload_bits(hip, np.full(k + 2, 77)) for k in (n, rows, n))
        hip.verify(s, count.ptr, path.ptr, after.ptr, dx.ptr, vocab)
        got = [read_bits(b) for b in (count, path, after)]
        for a, w in zip(got, R.verify(fresh, parent, ids, x)):
            assert np.array_equal(a[:-2], w), (fresh, a[:-2], w)
            assert np.all(a[-2:] == 77)
        for b in (dx, count, path, after):
            b.free()
        s.free()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shape", [(4, 64, 64), (2, 16, 16), (1, 4, 7), (12, 256, 16), (3, 36, 5), (2, 252, 64)])
def test_keep(hip, pkg, shape, half):
    KH, dh, page = shape
    rng = rng_of(KH, dh, page)
    for trial in range(4):
        fresh = [[25], [1, 0, 40, 7], [256, 3], [60] * 9][trial]
        lens = np.array(fresh) + rng.integers(0, 50, len(fresh))
        c = Cache(rng, lens, KH, dh, page, half)
        path, count = [], []
        for b, f in enumerate(fresh):
            k = int(rng.integers(0, f + 1))
            p = np.full(f, R.NONE, np.uint32)
            p[:k] = np.sort(rng.permutation(f)[:k])
            if trial == 1 and f > 5:  # paths that end where they do not rise, or leave the tokens
                p[3], k = [f + 9, 0][b % 2], f + 100
            if trial == 2 and f > 5:
                p[:], k = np.arange(f), f
            path.append(p)
            count.append(k)
        path = np.concatenate(path)
        g, up = c.upload(hip, pkg)
        s = c.batch(hip)
        s.set(lens, c.table, fresh=fresh)
        dc, dp = upload_bits(hip, np.array(count, np.uint32)), upload_bits(hip, path)
        hip.paged_keep(s, g, dc.ptr, dp.ptr)
        R.keep(c, fresh, np.array(count), path)
        for name in ("k", "v", "mass"):
            assert np.array_equal(up[name].read(), getattr(c, name).ravel()), (name, trial)
        assert np.array_equal(read_bits(up["born"]), c.born.ravel())
        for b in (*up.values(), dc, dp):
            b.free()
        s.free()
