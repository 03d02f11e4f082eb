"""GPU tests of the serving step's operators at values that FP32 or the pool cannot hold, and at calls of unusual shape: queries
that are not finite, rows that leave the range as they are rotated, pages named twice, pools of more than 2^32 elements,
clusters of every size. Oracle and tolerances are test_gpu_serving.py's."""
import numpy as np
import pytest

import cmachine_b200 as cm
from test_gpu_paged import BYTES, KINDS, QWEN, download, upload, widen
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


@KINDS
@pytest.mark.parametrize("most", [4, 640], ids=["single", "tiles"])
@pytest.mark.parametrize("which", ["key", "value"])
def test_a_row_that_its_rotation_takes_out_of_range_is_zeros(kind, most, which):
    """3.4e38 (cos 2 - sin 2) = -4.5e38, beyond FP32: the only row of the batch that cannot be stored. As a value it is not
    rotated: bytes hold it, and BF16 does not (3.4e38 is above 2^128 - 2^119)."""
    p = Served(kind, QWEN, 16, [most], [most], seed=33)
    rng = np.random.default_rng(4)
    x = (1 + rng.random((p.rows, 16 * 128))).astype(np.float32)
    row, head = int(p.starts[0]) + 2, 13 if which == "key" else 15
    x[row, head * 128:(head + 1) * 128] = 3.4e38
    p.rotate(x, (None, None, 1e-6, 1e6, 128))
    side = 0 if which == "key" else 1
    lost = which == "key" or kind != BYTES
    assert p.flags() == (1 if lost else 0)
    host, scales = p.get()
    page = int(p.table[0, 0])
    stored = host[side][page, :, 2]  # the row's two heads
    stored = stored.astype(np.float64) * scales[side][page, :, 2, None] if kind == BYTES else widen(stored)
    assert np.all(stored[0] != 0) if which == "value" else np.any(stored[0] != 0)
    if lost:
        assert np.all(stored[1] == 0)
        if kind == BYTES:
            assert scales[side][page, 1, 2] == 1
    else:
        assert np.all(np.abs(stored[1] / float(np.float32(3.4e38)) - 1) <= 2.0**-22)
    for j in (1, 3):  # the rows beside it
        assert np.any(host[side][page, 1, j] != 0)
    p.free()


@KINDS
def test_a_page_that_is_named_more_than_once(kind):
    """Two sequences of one length that share all their pages, and a table that names a page at several places."""
    p = Served(kind, QWEN, 16, [1, 1], [640, 640], seed=34)
    p.table[0, 5:9] = p.table[0, 4]
    p.table[0, 30] = p.table[0, 4]
    p.table[1] = p.table[0]
    p.put()
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    for blocks in (4, 12):
        q = p.queries()
        got, which = p.sparse(q, blocks, 1, 2)
        p.check_sparse(got, which, q, blocks, 1, 2, marks)
    assert p.flags() == 0
    p.free()


@KINDS
def test_a_pool_of_more_than_2_32_elements(kind):
    """The same batch in a small pool and at the end of one of 4.5e9 elements a side: the same queries, rows, bounds, pages and
    attention, bit for bit."""
    heads, page, news, lengths = (16, 8, 128), 128, [1, 5], [700, 400]
    L = cm.lib()
    p = Served(kind, heads, page, news, lengths, seed=35, extra=0)
    x = np.random.default_rng(5).standard_normal((p.rows, 32 * 128)).astype(np.float32)
    w = np.ones(128, np.float32)
    turn = (w, w, 1e-6, 1e6, 128)

    def serve():
        y = p.rotate(x, turn)
        p.whole()
        assert L.gpu_paged_bounds(p.cache, p.batch, p.bounds, p.status) == 0
        got, which = p.sparse(y, 4, 1, 1)
        assert p.flags() == 0
        return y, got, which

    want = serve()
    small = (p.get(), download(p.bounds, p.marks.shape, np.uint16))
    pages, far = 34500, 34500 - p.pages
    a_page, es = 8 * page * 128, 1 if kind == BYTES else 2
    pool = [L.gpu_alloc(pages * a_page * es) for _ in range(2)]
    scales, bounds = L.gpu_alloc(2 * pages * 8 * page * 4), L.gpu_alloc(pages * 8 * 2 * 128 * 2)
    for side in range(2):
        L.gpu_write(pool[side] + far * a_page * es, cm.ptr(p.host[side]), p.host[side].nbytes)
        if kind == BYTES:
            L.gpu_write(scales + (side * pages + far) * 8 * page * 4, cm.ptr(np.ascontiguousarray(p.scales[side])), p.scales[side].nbytes)
    table = p.table.copy()
    table[table >= 0] += far
    t = upload(table)
    p.cache = cm.PagedCache(kind, pages, page, 8, 128, *pool, scales if kind == BYTES else None)
    p.batch.table, near, p.bounds = t, p.bounds, bounds
    assert all(np.array_equal(a, b) for a, b in zip(serve(), want))
    for side in range(2):
        assert np.array_equal(download(pool[side] + far * a_page * es, small[0][0][side].shape, small[0][0][side].dtype), small[0][0][side])
        if kind == BYTES:
            assert np.array_equal(download(scales + (side * pages + far) * 8 * page * 4, p.scales[side].shape), small[0][1][side])
    assert np.array_equal(download(bounds + far * 8 * 2 * 128 * 2, small[1].shape, np.uint16), small[1])
    for y in (*pool, scales, bounds, t):
        L.gpu_free(y)
    p.bounds = near
    p.free()


@pytest.mark.parametrize("dim", [64, 128])
@KINDS
def test_clusters_of_every_size(kind, dim):
    """One query row over rows enough that 9 to 16 CTAs share them, so that no warp sums more than one chain of steps."""
    for ctas in range(9, 17):
        page, rows = 256, ctas * 128 * 16 - 40
        p = Served(kind, (2, 1, dim), page, [1], [rows + 3 * page], seed=ctas)
        p.whole()
        marks = download(p.bounds, p.marks.shape, np.uint16)
        q, blocks = p.queries(0.1), -(-rows // page)
        got, which = p.sparse(q, blocks, 1, 1)
        p.check_sparse(got, which, q, blocks, 1, 1, marks)
        p.free()
