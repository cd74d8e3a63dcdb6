"""Shared pages on the GPU where the caller's table has holes."""
import pytest

import kv_q4_ref as R
import vsl
from test_kv_q4_gpu import Gpu, ints

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("at,entry", [(2, -1), (2, 16), (2, 1 << 30), (0, -1), (1, 99)])
def test_fork_of_a_source_that_misses_a_page(at, entry):
    """The fork has the source's hole, is told of it, and gets no page with another sequence's content for it."""
    g = Gpu(R.Pages(4, 4, 64, 16), 2, 64, 7)
    vsl.kv_extend(g.kv, ints(0, 1), ints(150, 30), 2, g.ws, g.n, status=g.status)
    g.ref.extend([(0, 150), (1, 30)])
    g.same()
    g.table[0, at] = entry
    vsl.kv_fork(g.kv, ints(0, 1), ints(2, 3), 2, g.ws, g.n, status=g.status)
    assert g.status.item() == -5
    assert g.lens.tolist() == [150, 30, 150, 30]
    t = g.table.tolist()
    free = 4  # the lowest free pages, in the forks' order
    want = [0, 1, free, -1]
    want[at] = entry
    assert t[2] == want and t[3] == [free + 1, -1, -1, -1]
    count = [0] * 16
    for row in t:
        for p in set(row):
            if 0 <= p < 16:
                count[p] += 1
    count[at] += 1  # the page that the source lost is still counted for it
    assert g.count.tolist() == count
    want = g.mirror.copy()
    if at != 2:
        want[:, free] = want[:, 2]
    want[:, free + 1] = want[:, 3]
    assert (g.pool.cpu().numpy() == want).all()
