"""Log probabilities of given tokens, entropy and alternatives against 64 bits (paged_ref.py)."""

import numpy as np
import pytest

from paged_ref import U, logprobs, read_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip(pkg):
    h = pkg.Hip(0)
    yield h
    h.close()


def run(hip, x, ids, top, entropy=True, off=0):
    m, n = x.shape
    dx = hip.upload(np.concatenate([np.full(off, 9.0, np.float32), x.ravel(), np.full(8, 9.0, np.float32)]))
    lp, ent, ti, tl = (hip.upload(np.full(max(k, 1), 5.0)) for k in (m, m, m * top, m * top))
    hip.logprobs(lp.ptr, dx.at(off), ids, n, entropy=ent.ptr if entropy else None, top=top,
                 top_ids=ti.ptr if top else None, top_lp=tl.ptr if top else None)
    out = (lp.read(), ent.read(), read_bits(ti)[:m * top].reshape(m, top).astype(int),
           tl.read()[:m * top].reshape(m, top))
    for b in (dx, lp, ent, ti, tl):
        b.free()
    return out


def check(x, got, ids, top):
    lp, ent, ti, tl = got
    wl, we, wi, wt, bl, be = logprobs(x, ids, top)
    assert np.array_equal(ti, wi)

    def near(a, b, bound):
        fine = np.isfinite(b)
        assert np.array_equal(a[~fine], b[~fine].astype(np.float32), equal_nan=True), (a[~fine], b[~fine])
        # the last rounding, and that of x - M before it, go by the result's size
        err = np.abs(a[fine].astype(np.float64) - b[fine])
        bad = err > (bound + 4 * U * np.abs(np.where(np.isfinite(b), b, 0)))[fine]
        assert not bad.any(), (err[bad][:4], bound[fine][bad][:4])

    near(lp, wl, bl)
    near(ent, we, be)
    near(tl, wt, np.broadcast_to(bl[:, None], wt.shape))


@pytest.mark.parametrize("m,n,top", [(1, 1, 0), (1, 1, 1), (3, 2, 2), (1, 32000, 20), (5, 97, 32), (2, 63, 32), (7, 64, 5),
                                     (3, 65, 1), (4, 1023, 3), (4, 1025, 32), (2, 4099, 31), (300, 1000, 2),
                                     (33, 32003, 20), (2, 131071, 32), (1, 300001, 7), (9, 16384, 0), (6, 32768, 32),
                                     (5, 65537, 32)])
def test_random(hip, m, n, top):
    rng = np.random.default_rng([m, n, top])
    x = (rng.standard_normal((m, n)) * 3).astype(np.float32)
    ids = rng.integers(0, n, m)
    ids[0] = int(x[0].argmax())
    check(x, run(hip, x, ids, top), ids, top)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_any_alignment(hip, off):
    """Rows at every offset from 16 bytes: the neighbours' values do not come in."""
    rng = np.random.default_rng(off)
    for n in (5, 1022, 4097):
        x = (rng.standard_normal((6, n)) * 2 - 30).astype(np.float32)  # (9.0 lies around them)
        ids = rng.integers(0, n, 6)
        check(x, run(hip, x, ids, 5, off=off), ids, 5)


def test_ties_and_order(hip):
    """Equal logits: the lower token first, however many there are; fp16 values; signed zeros."""
    n = 5000
    rng = np.random.default_rng(1)
    x = np.stack([np.full(n, 1.5), np.arange(n) % 7, -(np.arange(n) % 3), rng.standard_normal(n).astype(np.float16),
                  np.where(np.arange(n) % 2, 0.0, -0.0), np.arange(n), -np.arange(n),
                  np.where(np.arange(n) == 4999, 2.0, 1.0), np.sort(rng.standard_normal(n))]).astype(np.float32)
    ids = rng.integers(0, n, len(x))
    for top in (1, 31, 32):
        check(x, run(hip, x, ids, top), ids, top)


def test_peaked(hip):
    """One token with nearly all the probability: its log probability keeps its digits."""
    n = 32000
    x = np.full((3, n), -20.0, np.float32)
    x[0, 77], x[1, 5], x[2, 31999] = 0.0, 40.0, 3.0
    ids = np.array([77, 5, 31999])
    lp, ent, _, tl = run(hip, x, ids, 2)
    rest = (n - 1) * np.exp(np.array([-20.0, -60.0, -23.0]))
    want = -np.log1p(rest)
    assert np.all(np.abs(lp - want) <= 200 * U * np.abs(want))
    assert np.array_equal(tl[:, 0], lp)
    assert np.all(ent >= 0) and np.all(np.abs(ent - (np.log1p(rest) + rest * np.array([20, 60, 23]) / (1 + rest)))
                                       <= 400 * U * (ent + np.abs(want)))


def test_impossible_tokens_infinities_and_nan(hip):
    n = 3000
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((8, n)) * 2).astype(np.float32)
    x[0, rng.random(n) < 0.9] = -np.inf
    x[1] = -np.inf                    # no token is possible
    x[2] = -np.inf
    x[2, 2999] = -1e30                # one is
    x[3, 17] = np.inf
    x[4, 18] = np.nan
    x[5] = np.nan
    x[6] = -np.inf
    x[6, 5] = np.nan
    x[7, :] = np.finfo(np.float32).min
    ids = np.array([int(x[0].argmax()), 4, 2999, 3, 7, 0, 6, 9])
    check(x, run(hip, x, ids, 4), ids, 4)
    ids = np.array([int(np.flatnonzero(x[0] == -np.inf)[0]), 0, 0, 17, 18, 1, 5, 0])
    check(x, run(hip, x, ids, 32), ids, 32)


def test_same_bits_alone(hip):
    """A row's results are those it has alone (rows of whole 16 bytes)."""
    x = (np.random.default_rng(4).standard_normal((40, 32000)) * 3).astype(np.float32)
    ids = np.arange(40)
    all_ = run(hip, x, ids, 5)
    for i in (0, 13, 39):
        one = run(hip, x[i:i + 1], ids[i:i + 1], 5)
        for a, b in zip(all_, one):
            assert np.array_equal(a[i], b[0])


def test_without_entropy_and_in_a_step(hip):
    """No entropy asked for; inside a recorded step, behind the linear that makes the logits, with
    other tokens on each run of the kept step."""
    rng = np.random.default_rng(5)
    w = rng.standard_normal((500, 64)).astype(np.float32)
    dw, dx, y = hip.upload(w), hip.alloc(64), hip.alloc(500)
    lp, ti, tl = hip.alloc(1), hip.alloc(4), hip.alloc(4)
    inv, cs, sn = hip.upload(np.ones(2, np.float32)), hip.alloc(2), hip.alloc(2)
    for step in range(6):
        hip.write(dx, rng.standard_normal(64))
        ids = rng.integers(0, 500, 1)
        hip.rope_table(cs.ptr, sn.ptr, inv.ptr, step, 1, 2)
        hip.linear(y.ptr, dw.ptr, 500, 64, dx.ptr, 1)
        hip.logprobs(lp.ptr, y.ptr, ids, 500, top=4, top_ids=ti.ptr, top_lp=tl.ptr)
        hip.flush()
        x = y.read()[None]
        wl, _, wi, wt, bl, _ = logprobs(x, ids, 4)
        assert np.abs(lp.read() - wl)[0] <= bl[0] + 4 * U * np.abs(wl)[0]
        assert np.array_equal(read_bits(ti), wi[0])
        assert np.all(np.abs(tl.read() - wt[0]) <= bl[0] + 4 * U * np.abs(wt[0]))


def test_first_alternative_is_the_greedy_pick(hip):
    x = np.random.default_rng(6).standard_normal((1, 32000)).astype(np.float16).astype(np.float32)
    _, _, ti, _ = run(hip, x, [0], 1)
    tok, dx = hip.alloc(2), hip.upload(x)
    hip.argmax(tok.ptr, None, 0, 0, dx.ptr, 32000)
    assert tok.read().view(np.int64)[0] == ti[0, 0]


def test_refusals(hip, pkg):
    x, lp, ti, tl = hip.alloc(200), hip.upload(np.full(4, 7.0)), hip.alloc(200), hip.alloc(200)

    def bad(code, *a, **k):
        with pytest.raises(pkg.SlmError) as e:
            hip.logprobs(*a, **k)
        assert e.value.code == code, e.value

    bad(-5, lp.ptr, x.ptr, [0, 50], 50)              # a token past the row
    bad(-5, lp.ptr, x.ptr, [0] * 5, 50)              # more rows than x holds
    bad(-1, lp.ptr, x.ptr, [0], 0)
    bad(-1, lp.ptr, x.ptr, [0], 50, top=51, top_ids=ti.ptr, top_lp=tl.ptr)
    bad(-3, lp.ptr, x.ptr, [0], 50, top=33, top_ids=ti.ptr, top_lp=tl.ptr)
    bad(-1, lp.ptr, x.ptr, [0], 50, top=3, top_ids=ti.ptr)
    bad(-1, lp.ptr, x.ptr, [0], 50, entropy=lp.ptr)
    bad(-1, x.ptr, x.ptr, [0], 50)
    bad(-1, lp.ptr, x.ptr, [0], 50, top=3, top_ids=ti.ptr, top_lp=ti.at(1))
    assert np.all(lp.read() == 7.0)
    hip.logprobs(lp.ptr, x.ptr, [], 50)              # no rows: nothing to do
    assert np.all(lp.read() == 7.0)
