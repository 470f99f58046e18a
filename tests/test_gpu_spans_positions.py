"""Several new tokens a sequence over paged caches whose slots have positions of their own."""

import numpy as np
import pytest

import span_ref as R
from paged_ref import Cache
from test_gpu_paged import attend, check, hip, rng_of  # noqa: F401
from test_gpu_spans import queries, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("reach,gap", [(None, 1), (None, 40), (2 ** 32 + 5, 3), (60, 2)])
@pytest.mark.parametrize("group", [1, 3, 20])
def test_positions_behind_a_rows_own(hip, pkg, half, tree, reach, gap, group):
    """Slots before the new tokens' whose position lies behind a row's: not seen, as by paged_attend."""
    lens, fresh = [300, 90], [20, 9]
    rng = rng_of(gap, tree, group)
    c = Cache(rng, lens, 2, 64, 16, half)
    for b, n in enumerate(lens):
        pg, sl = c.where(b)
        ahead = rng.permutation(n - fresh[b])[:40]
        c.born[pg[ahead], :, sl[ahead]] += np.uint32(500)
        c.born[pg[ahead[:4]], :, sl[ahead[:4]]] = np.uint32(0xffffffff)
    q = queries(rng, fresh, 2 * group, 64)
    parent = R.random_tree(rng, fresh) if tree else None
    want, bound = R.attend(c, fresh, q, 0.125, reach, gap, True, parent)
    y = run(hip, pkg, c, fresh, q, 0.125, reach, gap, True, parent)
    check(y, want, bound)
    if not tree and reach is None and group <= 16:
        last = np.cumsum(fresh) - 1
        one, _ = attend(hip, pkg, c, np.ascontiguousarray(q[last]), gap, mass=False, born=True, scale=0.125)
        check(one, want[last], bound[last])
