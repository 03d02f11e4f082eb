"""GPU tests of the serving step's operators at values that FP32 or the pool cannot hold: queries that are not finite, and
rows that leave the range as they are rotated. Oracle and tolerances are test_gpu_serving.py's."""
import numpy as np
import pytest

import cmachine_b200 as cm
from test_gpu_paged import BYTES, KINDS, QWEN, download, widen
from test_gpu_serving import Served

pytestmark = pytest.mark.gpu

WILD = [np.nan, np.inf, -np.inf, 3e38, -3e38]


@KINDS
@pytest.mark.parametrize("value", WILD)
@pytest.mark.parametrize("news", [[1, 2, 1], [301, 3]], ids=["single", "pairs"])
def test_queries_that_are_not_finite_touch_no_other(kind, value, news):
    """One KV head's queries of one row, or one element of them: its pages are some of the sequence, in order; every other
    row and head has its own, and its attention."""
    p = Served(kind, QWEN, 16, news, [700, 500, 400][:len(news)], seed=31)
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    wild = int(p.starts[0])
    at = int(p.lengths[0]) - news[0]
    plain = p.queries()
    for elements in (slice(0, 6 * 128), 2 * 128 + 5):
        q = plain.copy()
        q[wild, elements] = value
        got, which = p.sparse(q, 10, 1, 2)
        w = which[wild, 0]
        assert np.all(np.diff(w) > 0) and w[0] == 0 and w[-1] == at // 16 and w[-2] == at // 16 - 1
        # The row's other KV head: the same as with the plain queries.
        want, pages = p.sparse(plain, 10, 1, 2)
        assert np.array_equal(which[wild, 1], pages[wild, 1]) and np.array_equal(got[wild, 6 * 128:], want[wild, 6 * 128:])
        assert np.array_equal(np.delete(which, wild, 0), np.delete(pages, wild, 0))
        assert np.array_equal(np.delete(got, wild, 0), np.delete(want, wild, 0))
    q = plain.copy()
    q[wild, :6 * 128] = value
    got, which = p.sparse(q, 10, 1, 2)
    every = list(p.places())
    p.places = lambda: (x for x in every if x[1] != wild)
    p.check_sparse(got, which, q, 10, 1, 2, marks)
    assert p.flags() == 0
    p.free()


@KINDS
@pytest.mark.parametrize("value", WILD)
@pytest.mark.parametrize("bound", [0x7f80, 0xff80, 0x7fc0, 0xffff, 0x0000])
def test_queries_and_bounds_that_are_not_finite(kind, value, bound):
    p = Served(kind, QWEN, 16, [2, 1], [700, 900], seed=32)
    marks = p.rng.integers(0, 65536, p.marks.shape).astype(np.uint16)
    marks[::2] = bound
    cm.lib().gpu_write(p.bounds, cm.ptr(marks), marks.nbytes)
    q = p.queries()
    q[0] = value
    q[2, ::7] = value
    _, which = p.sparse(q, 10, 1, 2)
    for s, r, at in p.places():
        for h in range(2):
            w = which[r, h]
            assert np.all(np.diff(w) > 0) and w[0] == 0 and w[-1] == at // 16 and w[-2] == at // 16 - 1
    p.free()
