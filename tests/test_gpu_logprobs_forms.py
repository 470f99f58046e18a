"""Log probabilities where sizes choose other forms: many long rows (a workgroup a row, some panels of
it), a row over workgroups of some panels each. Against 64 bits (paged_ref.py)."""

import numpy as np
import pytest

from paged_ref import U, read_bits
from test_gpu_logprobs import check, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip(pkg):
    h = pkg.Hip(0)
    yield h
    h.close()


@pytest.mark.parametrize("m,n", [(65, 8193), (70, 32003), (66, 70001), (65, 32768), (64, 8193), (1, 524289), (2, 600001),
                                 (64, 8192), (200, 8191)])
@pytest.mark.parametrize("top", [0, 1, 20, 32])
def test_random(hip, m, n, top):
    rng = np.random.default_rng([m, n, top])
    x = (rng.standard_normal((m, n)) * 3).astype(np.float32)
    ids = rng.integers(0, n, m)
    check(x, run(hip, x, ids, top, off=top % 4), ids, top)


def orders(n, panel):
    """Rows whose first `panel` logits say little of the rest."""
    rng = np.random.default_rng(n)
    r = (rng.standard_normal(n) * 2).astype(np.float32)
    first = np.arange(n) < panel
    return np.stack([np.sort(r), np.sort(r)[::-1], np.full(n, -1.5), np.where(first, -np.inf, r), np.where(first, np.nan, r),
                     np.where(first, r, -np.inf), np.where(first, r, np.nan), np.where(first, -1e30, r),
                     np.arange(n) // 7, np.where(np.arange(n) == n - 1, np.inf, r), np.full(n, -np.inf),
                     np.where(np.arange(n) == n - 1, 5.0, -np.inf), np.where(first, r, 100 + r)]).astype(np.float32)


@pytest.mark.parametrize("top", [0, 3, 32])
@pytest.mark.parametrize("off", [0, 3])
@pytest.mark.parametrize("n", [32769, 70001])
def test_orders_over_the_panels_of_many_rows(hip, n, off, top):
    """Rising and falling rows, equal logits, impossible tokens and NaN in whole panels."""
    x = np.tile(orders(n, 32768), (6, 1))  # (78 rows: not split)
    ids = np.random.default_rng(top).integers(0, n, len(x))
    check(x, run(hip, x, ids, top, off=off), ids, top)


@pytest.mark.parametrize("top", [0, 3, 32])
@pytest.mark.parametrize("n,panel", [(532500, 8192), (600001, 16384)])
def test_orders_over_the_panels_of_a_part(hip, n, panel, top):
    x = orders(n, panel)
    ids = np.random.default_rng(top).integers(0, n, len(x))
    check(x, run(hip, x, ids, top, off=1), ids, top)


@pytest.mark.parametrize("recorded", [False, True])
def test_more_rows_than_go_up_at_once(hip, recorded):
    """Past 2^20 rows, call by call and where a step is being recorded. Bounds as paged_ref's, for rows of 3."""
    m, n, top = (1 << 20) + 5, 3, 2
    rng = np.random.default_rng(7)
    x = (rng.standard_normal((m, n)) * 3).astype(np.float32)
    ids = rng.integers(0, n, m)
    dx, lp, ent, ti, tl = hip.upload(x), hip.alloc(m), hip.alloc(m), hip.alloc(m * top), hip.alloc(m * top)
    if recorded:
        inv, cs, sn = hip.upload(np.ones(2, np.float32)), hip.alloc(2), hip.alloc(2)
        hip.rope_table(cs.ptr, sn.ptr, inv.ptr, 0, 1, 2)
    hip.logprobs(lp.ptr, dx.ptr, ids, n, entropy=ent.ptr, top=top, top_ids=ti.ptr, top_lp=tl.ptr)
    hip.flush()
    r = x.astype(np.float64)
    d = r.max(1, keepdims=True) - r
    l = -d - np.log(np.exp(-d).sum(1, keepdims=True))
    p = np.exp(l)
    rel = (p * (2 * d + 2)).sum(1) + 33
    bl = U * (rel + 4 + 2 * np.log(n))
    be = bl + U * ((p * d * (2 * d + 4)).sum(1) + 2 * (p * d).sum(1) * (33 + rel))
    order = np.argsort(-r, 1, kind="stable")[:, :top]
    assert np.array_equal(read_bits(ti).reshape(m, top), order)
    want = l[np.arange(m), ids]
    assert np.all(np.abs(lp.read() - want) <= bl + 4 * U * np.abs(want))
    want = -(p * l).sum(1)
    assert np.all(np.abs(ent.read() - want) <= be + 4 * U * want)
    want = np.take_along_axis(l, order, 1)
    assert np.all(np.abs(tl.read().reshape(m, top) - want) <= bl[:, None] + 4 * U * np.abs(want))
