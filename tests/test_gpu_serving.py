"""GPU tests of the rotated append, the page bounds and the attention over chosen pages (include/gpu.h) against float64.

Rotated rows are carried in 64 bits and rounded once: half a step of FP32, 2^-24 |y|. The kernel's angle is a 64-bit
product of a place and a 64-bit rate, each rounded, in half turns, so it is off by 2^-52 place; its cosines, the norm
(a sum of dim squares, a reciprocal root) and the rotation add fewer than dim / 4 + 32 roundings of 2^-53 of the pair's
size. The oracle's angles are 80-bit numbers. So

    |y - exact| <= 2^-24 |exact| + 2^-149 + (2^-52 place + 2^-46) |pair|

Stored rows are the codec's of the FP32 row, checked bit for bit through gpu_paged_append.

Bounds and the choice of pages are exact: the oracle's scores are 64-bit sums in another order, and a choice between
scores closer than 2^-40 of their terms' sum would be reported as a tie of the test's own making (none is).
The attention over what was chosen is held to the bound of test_gpu_paged.py: a kernel of its own does it, with the parts
and sums of that file's few-row kernel.
"""
import numpy as np
import pytest

import cmachine_b200 as cm
from test_gpu_paged import BF16, BYTES, KINDS, QWEN, SENTINEL, Pool, bf16, download, upload, widen

pytestmark = pytest.mark.gpu

MHA64, GROUP4, MQA, ODD64, GROUP3 = (4, 4, 64), (32, 8, 128), (8, 1, 128), (14, 2, 64), (9, 3, 64)


class Served(Pool):
    """A pool with its bounds; the bounds of pages that nothing has brought up to date hold junk."""

    def put(self):
        super().put()
        junk = self.rng.integers(0, 0x7f80, (self.pages, self.kvheads, 2, self.dim)).astype(np.uint16)
        self.marks = junk
        self.bounds = upload(junk)
        self.live.append(self.bounds)

    def rotate(self, x, turn, inplace=False, pad=0, qheads=None):
        """gpu_paged_rotate_append of fused rows x [rows][(qheads + 2 kvheads) dim]; returns the queries."""
        L, qh = cm.lib(), qheads or self.qheads
        width, n = (qh + 2 * self.kvheads) * self.dim, max(self.rows, 1)
        wide = np.full((n, width + pad), np.nan, np.float32)
        wide[:x.shape[0], :width] = x
        dx = upload(wide)
        norms = [upload(w) if w is not None else None for w in turn[:2]]
        t = cm.HeadRotation(*norms, *turn[2:])
        k = dx + qh * self.dim * 4
        if inplace:
            out, stride = dx, width + pad
        else:
            stride = qh * self.dim + pad
            out = upload(np.full((n, stride), SENTINEL, np.float32))
        assert L.gpu_paged_rotate_append(self.cache, self.batch, t, out, stride, dx, k, k + self.kvheads * self.dim * 4,
                                         width + pad, qh, self.status) == 0
        got = download(out, (n, stride))
        after = download(dx, wide.shape)
        same = slice(qh * self.dim, None) if inplace else slice(None)
        assert np.array_equal(after[:, same], wide[:, same], equal_nan=True)  # the input is left alone
        if not inplace:
            assert np.all(got[:, qh * self.dim:] == SENTINEL)
            L.gpu_free(out)
        for p in [dx, *[p for p in norms if p]]:
            L.gpu_free(p)
        return got[:, :qh * self.dim]

    def places(self):
        """(sequence, row, place) of every new row of a sequence with good extents."""
        for s in range(len(self.news)):
            for i in range(int(self.news[s])):
                yield s, int(self.starts[s]) + i, int(self.lengths[s] - self.news[s]) + i

    def update(self):
        assert cm.lib().gpu_paged_bounds(self.cache, self.batch, self.bounds, self.status) == 0
        return download(self.bounds, self.marks.shape, np.uint16)

    def whole(self):
        """The same cache with every row new."""
        starts = np.concatenate([[0], np.cumsum(self.lengths)]).astype(np.int32)
        p = upload(starts)
        self.live.append(p)
        b = cm.PagedBatch(len(self.news), int(starts[-1]), int(self.lengths.max(initial=0)), int(self.lengths.max(initial=0)), p,
                          self.batch.lengths, self.batch.table, self.stride)
        assert cm.lib().gpu_paged_bounds(self.cache, b, self.bounds, self.status) == 0

    def sparse(self, q, blocks, first, recent, gpu=None, pad=0, chosen=True):
        L = cm.lib()
        n, width = max(self.rows, 1), self.qheads * self.dim
        out = upload(np.full((n, width + pad), SENTINEL, np.float32))
        wide = np.full((n, width + pad), np.nan, np.float32)
        wide[:q.shape[0], :width] = q
        dq, sel = upload(wide), upload(np.full((n, self.kvheads, blocks), -77, np.int32))
        g = gpu or L.gpu_open()
        assert L.gpu_paged_sparse_attention(g, out, width + pad, dq, width + pad, self.cache, self.batch, self.bounds, self.qheads,
                                            blocks, first, recent, sel if chosen else None, self.status) == 0
        got, which = download(out, (n, width + pad)), download(sel, (n, self.kvheads, blocks), np.int32)
        for p in (out, dq, sel):
            L.gpu_free(p)
        if not gpu:
            L.gpu_close(g)
        assert np.all(got[:, width:] == SENTINEL)
        return got[:, :width], which

    def choose(self, x, s, h, at, blocks, first, recent, marks):
        """The pages of one query row x [qheads][dim] of KV head h at place `at`, ascending."""
        own, group = at // self.page, self.qheads // self.kvheads
        if own < blocks:
            return list(range(own + 1))
        low, high, want = first, own - recent + 1, blocks - first - recent
        ids = self.table[s, low:high]
        good = (ids >= 0) & (ids < self.pages)
        b = widen(marks[np.where(good, ids, 0), h]).astype(np.float64)  # [pages][2][dim]
        y = x[h * group:(h + 1) * group].astype(np.float64)
        score = (np.maximum(y, 0) @ b[:, 1].T + np.minimum(y, 0) @ b[:, 0].T).max(0)
        score = np.where(good, score, -np.inf)
        order = np.argsort(-score, kind="stable")
        if want and len(order) > want:
            edge = order[want - 1:want + 1]  # the last page in and the first one out
            gap, size = score[edge[0]] - score[edge[1]], (np.abs(y) @ np.abs(b[edge]).max(1).T).max()
            if np.isfinite(gap):
                assert gap == 0 or gap > 2.0**-40 * size, "a tie of the test's making"
        return sorted([*range(low), *(order[:want] + low).tolist(), *range(high, own + 1)])

    def check_sparse(self, got, which, q, blocks, first, recent, marks, skip=()):
        d, group = self.dim, self.qheads // self.kvheads
        held = {}
        for s, r, at in self.places():
            if s in skip:
                continue
            if s not in held:
                held[s] = (*self.held(s, 0), self.held(s, 1)[0])
            k, there, v = held[s]
            for h in range(self.kvheads):
                if at < 0:
                    assert np.all(which[r, h] == -1) and np.all(got[r, h * group * d:(h + 1) * group * d] == 0)
                    continue
                pages = self.choose(q[r].reshape(self.qheads, d), s, h, at, blocks, first, recent, marks)
                assert which[r, h].tolist() == pages + [-1] * (blocks - len(pages)), (s, r, h)
                j = np.concatenate([np.arange(p * self.page, min((p + 1) * self.page, at + 1)) for p in pages])
                j = j[there[j]]
                kk, vv = k[h, j], v[h, j]
                for g in range(h * group, (h + 1) * group):
                    x, o = q[r, g * d:(g + 1) * d].astype(np.float64), got[r, g * d:(g + 1) * d]
                    if not len(j):
                        assert np.all(o == 0)
                        continue
                    t = kk @ x / np.sqrt(d)
                    p = np.exp(t - t.max())
                    p /= p.sum()
                    big = (np.maximum(np.abs(x), np.abs(x).max() / 16) @ np.abs(kk).T / np.sqrt(d)).max()
                    tol = 2.0**-23 * (64 * big + 128 + len(j) / 8) * (p @ np.abs(vv)) + 2.0**-36 * len(j) * np.abs(vv).max()
                    assert np.all(np.abs(o - p @ vv) <= tol), (s, r, g, float(np.abs(o - p @ vv).max()))


def turned(x, weight, at, eps, theta, rotary):
    """One head's row, normed and rotated to place `at`, in float64, and each element's pair's size."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt(np.mean(y * y) + np.float64(np.float32(eps))) * weight.astype(np.float64)
    size, half = np.abs(y), rotary // 2
    if half:
        rate = np.longdouble(np.float32(theta)) ** (-np.arange(half, dtype=np.longdouble) / half)
        angle = np.longdouble(at) * rate
        c, s = np.cos(angle), np.sin(angle)
        a, b = y[:half].copy(), y[half:rotary].copy()
        y = np.concatenate([(a * c - b * s).astype(np.float64), (b * c + a * s).astype(np.float64), y[rotary:]])
        size = np.concatenate([np.hypot(a, b), np.hypot(a, b), size[rotary:]])
    return y, size


def check_turned(p, got, x, weight, turn, qheads):
    worst = 0.0
    for s, r, at in p.places():
        for h in range(qheads):
            d = slice(h * p.dim, (h + 1) * p.dim)
            exact, size = turned(x[r, d], weight, at, *turn)
            off = np.abs(got[r, d] - exact)
            tol = 2.0**-24 * np.abs(exact) + 2.0**-149 + (2.0**-52 * abs(at) + 2.0**-46) * size
            assert np.all(off <= tol), (s, r, h, at)
            worst = max(worst, float((off / tol).max()))
    return worst


ROTATIONS = [(None, None, 1e-6, 1e6, 128), ("w", "w", 1e-6, 1e6, 128), ("w", None, 1e-5, 1e4, 64), (None, "w", 0.0, 5e5, 20),
             ("w", "w", 1e-6, 1e4, 0), (None, None, 0.0, 1.0, 4)]


@KINDS
@pytest.mark.parametrize("rotation", ROTATIONS, ids=range(len(ROTATIONS)))
@pytest.mark.parametrize("shape", [(QWEN, 16, [1], [1]), (QWEN, 64, [1, 1, 1], [300, 31, 32768]), (ODD64, 7, [3, 0, 5, 17], [3, 9, 90, 400]),
                                   (GROUP3, 24, [2, 9], [40, 9]), (MQA, 100, [130], [130]), (MHA64, 3, [33, 40], [100, 64]),
                                   # rows enough for tiles of four: whole ones, and sequences that leave one to three
                                   (QWEN, 16, [650, 2], [700, 900]), (ODD64, 7, [601, 1, 0, 6], [601, 40, 3, 90]),
                                   (GROUP3, 24, [299, 303, 5], [400, 303, 5]), (MQA, 100, [700], [1000])],
                         ids=["first", "single", "ragged", "odd", "chunk", "small", "tiles", "ragged-tiles", "odd-tiles", "chunk-tiles"])
def test_rotated_rows_match_float64(kind, rotation, shape):
    heads, page, news, lengths = shape
    p = Served(kind, heads, page, news, lengths, seed=sum(lengths), gap=2)
    qh, kv, d = heads
    rng = np.random.default_rng(11)
    x = (rng.standard_normal((p.rows, (qh + 2 * kv) * d)) * np.exp(rng.standard_normal((p.rows, 1)))).astype(np.float32)
    w = [(1 + 0.2 * rng.standard_normal(d)).astype(np.float32) if n else None for n in rotation[:2]]
    turn = (*w, *rotation[2:4], min(rotation[4], d))
    before = p.get()
    got = p.rotate(x, turn, pad=4)
    assert np.all(got[:2] == SENTINEL)  # rows of no sequence
    check_turned(p, got, x, w[0], turn[2:], qh)
    assert p.flags() == 0
    # The keys, as rows of another call's queries, appended by gpu_paged_append: the same pool, bit for bit.
    k = x[:, qh * d:(qh + kv) * d]
    keys = p.rotate(np.concatenate([k, k, k], 1), (w[1], None, *turn[2:]), qheads=kv)
    check_turned(p, keys, k, w[1], turn[2:], kv)
    host, p.host, scales, p.scales = p.host, before[0], p.scales, before[1]
    p.put()
    p.rotate(x, turn)
    got = p.get()
    p.put()
    L, dk, dv = cm.lib(), upload(keys), upload(x[:, (qh + kv) * d:])
    assert L.gpu_paged_append(p.cache, p.batch, dk, dv, kv * d, p.status) == 0
    want = p.get()
    for a, b in zip((*got[0], got[1]), (*want[0], want[1])):
        assert np.array_equal(a, b)
    assert any(not np.array_equal(a, b) for a, b in zip(got[0], before[0]))
    for y in (dk, dv):
        L.gpu_free(y)
    p.free()


@KINDS
@pytest.mark.parametrize("heads", [QWEN, GROUP3])
@pytest.mark.parametrize("most", [40, 603])
def test_rotation_in_place(kind, heads, most):
    p = Served(kind, heads, 16, [5, 1, most], [5, 900, most + 37], seed=2)
    rng = np.random.default_rng(3)
    d = heads[2]
    x = rng.standard_normal((p.rows, (heads[0] + 2 * heads[1]) * d)).astype(np.float32)
    w = np.ones(d, np.float32)
    turn = (w, w, 1e-6, 1e6, d)
    a = p.rotate(x, turn, pad=8)
    first = p.get()
    b = p.rotate(x, turn, inplace=True, pad=8)
    assert np.array_equal(a, b) and np.array_equal(first[0][0], p.get()[0][0])
    p.free()


@pytest.mark.parametrize("place", [2**20 - 1, 2**30 - 1])
def test_far_places(place):
    """Sequences as long as the interface allows, whose last page alone exists."""
    page = 65536
    table = np.full((1, 2**30 // page), -1, np.int32)
    table[0, place // page] = 0
    p = Served(BF16, (1, 1, 64), page, [1], [1], table=table, extra=0)
    p.lengths, p.stride = np.array([place + 1]), table.shape[1]
    p.put()
    p.batch.max_length = 2**30
    x = np.random.default_rng(5).standard_normal((1, 192)).astype(np.float32)
    got = p.rotate(x, (None, None, 0.0, 1e6, 64))
    check_turned(p, got, x, None, (0.0, 1e6, 64), 1)
    y, _ = turned(x[0, 64:128], None, place, 0.0, 1e6, 64)
    assert p.flags() == 0
    stored = widen(download(p.live[0], p.host[0].shape, np.uint16)[0, 0, place % page])
    assert np.all(np.abs(stored - y) <= 2.0**-8 * np.abs(y) + 1e-6)
    p.free()


@KINDS
@pytest.mark.parametrize("more", [[], [600]], ids=["few", "tiles"])
def test_rotation_reports_what_it_cannot_store(kind, more):
    p = Served(kind, QWEN, 16, [3, 2, 4] + more, [40, 1, 4] + more, seed=8)  # the second has a row at place -1
    p.table[0, 2] = p.pages  # places 32 .. 47 of the first
    p.put()
    x = np.random.default_rng(4).standard_normal((p.rows, 16 * 128)).astype(np.float32)
    r = int(p.starts[2])
    x[r, 12 * 128 + 5] = np.nan       # a key of the first KV head
    x[r + 1, 15 * 128 + 9] = np.inf   # a value of the second
    x[r + 2, 13 * 128:14 * 128] = 3.4e38  # its rotation leaves FP32's range somewhere
    x[r + 3, 7] = np.nan              # a query head
    before = p.get()
    got = p.rotate(x, (None, None, 1e-6, 1e6, 128))
    assert p.flags() == 1 | 2
    y = np.where(np.isfinite(x), x, 0)
    for s, row, at in p.places():
        for h in range(12):
            d = slice(h * 128, h * 128 + 128)
            if row == r + 3 and h == 0:
                continue
            exact, size = turned(y[row, d], None, at, 0, 1e6, 128)
            assert np.all(np.abs(got[row, d] - exact) <= 2.0**-24 * np.abs(exact) + 2.0**-45 * size)
    after = p.get()
    ids = p.table[2, 0]
    val = (lambda kk, j, h: after[0][kk][ids, h, j].astype(np.int64)) if kind == BYTES else (lambda kk, j, h: widen(after[0][kk][ids, h, j]))
    assert np.all(val(0, 0, 0) == 0) and np.any(val(0, 0, 1) != 0) and np.any(val(1, 0, 0) != 0)
    assert np.all(val(1, 1, 1) == 0) and np.any(val(0, 1, 1) != 0)
    assert np.all(val(0, 2, 1) == 0) or np.all(np.isfinite(val(0, 2, 1)))
    for kk in range(2):  # rows without a page went nowhere
        changed = np.argwhere((after[0][kk] != before[0][kk]).any(-1))
        assert {int(c[0]) for c in changed} <= {int(p.table[1, 0]), int(p.table[2, 0]), *p.table[3:].reshape(-1).tolist()}
    p.free()


@KINDS
def test_rows_of_zeros_and_extremes(kind):
    """Zero rows with and without an eps, and rows whose squares leave FP32's range."""
    p = Served(kind, (2, 1, 128), 16, [4], [4], seed=1)
    x = np.random.default_rng(6).standard_normal((4, 512)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-30)
    x[2] *= np.float32(1e30)
    w = np.full(128, 1.5, np.float32)
    got = p.rotate(x, (w, w, 1e-6, 1e6, 128))
    check_turned(p, got, x, w, (1e-6, 1e6, 128), 2)
    assert np.all(got[0] == 0)
    got = p.rotate(x[:, :], (w, w, 0.0, 1e6, 128))
    assert np.all(np.isnan(got[0]))  # 0 / 0
    check = Served(kind, (2, 1, 128), 16, [3], [4], seed=1)
    check_turned(check, got[1:], x[1:], w, (0.0, 1e6, 128), 2)
    assert p.flags() == 1  # the zero key
    p.free()
    check.free()


# ---------------------------------------------------------------- bounds
def bounds_of(p, s, page):
    """Exact bounds of one page of a sequence as BF16 bits [kvheads][2][dim], and the page's id."""
    n = min(p.page, int(p.lengths[s]) - page * p.page)
    ids = int(p.table[s, page])
    x = p.values(0)[ids, :, :n]
    out = np.empty((p.kvheads, 2, p.dim), np.uint16)
    for side, y in enumerate((x.min(1), x.max(1))):
        near = bf16(y.astype(np.float32))
        wrong = widen(near) < y if side else widen(near) > y
        steps = np.where((near >> 15) == (0 if side else 1), 1, -1)  # in magnitude
        out[:, side] = np.where(wrong, near + steps * wrong, near).astype(np.uint16)
    return ids, out


@KINDS
@pytest.mark.parametrize("shape", [(QWEN, 16, [1, 1, 1, 1], [1, 16, 17, 300]), (MHA64, 1, [3, 1], [9, 5]), (ODD64, 24, [5, 60, 0, 100], [90, 60, 7, 100]),
                                   (GROUP4, 100, [250, 1], [250, 1000]), (MQA, 300, [700], [1000])], ids=["one", "page1", "ragged", "long", "big"])
def test_bounds_are_exact(kind, shape):
    p = Served(kind, *shape, seed=3)
    if kind == BYTES:  # products that FP32 rounds
        p.scales *= (1 + 2.0**-9 * p.rng.standard_normal(p.scales.shape)).astype(np.float32)
        p.put()
    got = p.update()
    want = p.marks.copy()
    for s in range(len(p.news)):
        n, c = int(p.lengths[s]), int(p.news[s])
        if c:
            for page in range((n - c) // p.page, (n - 1) // p.page + 1):
                ids, b = bounds_of(p, s, page)
                want[ids] = b
    assert np.array_equal(widen(got), widen(want))  # zeros of either sign
    assert p.flags() == 0
    p.free()


@KINDS
def test_bounds_pass_over_nan_and_report_bad_pages(kind):
    p = Served(kind, QWEN, 16, [40, 3], [40, 2], seed=5)
    p.table[0, 1] = -1
    ids = p.table[0, 0]
    if kind == BYTES:
        p.scales[0][ids, 0, 3] = np.nan
    else:
        p.host[0][ids, 0, 3] = 0x7fc0
    p.put()
    got = p.update()
    assert p.flags() == 2
    x = p.values(0)[ids, 0]
    x = x[np.isfinite(x).all(1)]
    assert len(x) == 15 and np.all(widen(got[ids, 0, 0]) <= x.min(0)) and np.all(widen(got[ids, 0, 1]) >= x.max(0))
    free = np.setdiff1d(np.arange(p.pages), p.table)
    assert len(free) and np.array_equal(got[free], p.marks[free])
    p.free()


# ---------------------------------------------------------------- chosen pages
CHOICES = [(QWEN, 16, [1], [1], 4, 1, 1), (QWEN, 16, [1, 1, 1], [64, 65, 80], 4, 1, 2), (QWEN, 64, [1] * 4, [4000, 31, 1025, 64], 6, 1, 2),
           (ODD64, 24, [1, 3, 7], [900, 700, 7], 5, 0, 1), (GROUP4, 32, [5, 5], [900, 300], 9, 2, 2), (MQA, 1, [1, 2], [200, 33], 40, 3, 5),
           (MHA64, 7, [40, 1], [300, 129], 12, 1, 4), (GROUP3, 100, [1, 130], [2000, 1500], 4, 0, 4), (QWEN, 16, [1], [5000], 100, 1, 1),
           (QWEN, 16, [200, 1], [333, 1000], 3, 1, 1), (QWEN, 48, [3], [2], 5, 1, 1), ((1, 1, 64), 16, [1], [20000], 1, 0, 1),
           # rows enough to go in pairs, which sequences' ends part
           (QWEN, 16, [299, 1, 4], [900, 333, 40], 5, 1, 1), (GROUP3, 24, [201], [1500], 6, 0, 2), (QWEN, 16, [300], [3000], 150, 2, 5)]


@KINDS
@pytest.mark.parametrize("case", CHOICES, ids=lambda c: f"{c[0]}p{c[1]}n{c[2]}l{c[3]}b{c[4]}".replace(" ", ""))
def test_sparse_attention_matches_float64(kind, case):
    heads, page, news, lengths, blocks, first, recent = case
    p = Served(kind, heads, page, news, lengths, seed=sum(lengths), gap=1)
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries()
    got, which = p.sparse(q, blocks, first, recent, pad=4)
    assert np.all(got[0] == SENTINEL) and np.all(which[0] == -77)  # the row of no sequence
    p.check_sparse(got, which, q, blocks, first, recent, marks)
    assert p.flags() == 0
    again, _ = p.sparse(q, blocks, first, recent, chosen=False)
    assert np.array_equal(got, again)
    p.free()


@KINDS
def test_pages_enough_are_the_whole_attention(kind):
    p = Served(kind, QWEN, 16, [1, 1, 1], [500, 3, 64], seed=4)
    q = p.queries()
    got, which = p.sparse(q, 32, 1, 1)  # no bounds are asked for
    p.check(got, q)
    p.check(p.attend(q), q)
    p.free()


@KINDS
def test_equal_pages_go_to_the_lower(kind):
    """Pages with the same keys, so equal scores in every digit, and a query of zeros, for which all are equal."""
    p = Served(kind, QWEN, 16, [1, 1], [640, 640], seed=6)
    for s in range(2):
        for page in range(3, 39):
            for x in p.host:
                x[p.table[s, page]] = x[p.table[s, 3 + page % 4]]
            if kind == BYTES:
                p.scales[:, p.table[s, page]] = p.scales[:, p.table[s, 3 + page % 4]]
    p.put()
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries()
    q[1] = 0
    for blocks in (4, 9, 20, 39):
        got, which = p.sparse(q, blocks, 1, 1)
        p.check_sparse(got, which, q, blocks, 1, 1, marks)
    assert which[1, 0, :3].tolist() == [0, 1, 2]
    p.free()


@KINDS
def test_scores_of_unlike_size(kind):
    """Scores that fall by half from page to page, so that every pass over them cuts off few."""
    p = Served(kind, (4, 2, 64), 16, [1], [16 * 120], seed=7)
    for page in range(120):
        f = 2.0 ** -(page * 37 % 120)
        if kind == BYTES:
            p.scales[0][p.table[0, page]] *= np.float32(f)
        else:
            p.host[0][p.table[0, page]] = bf16(widen(p.host[0][p.table[0, page]]) * np.float32(f))
    p.put()
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries()
    for blocks in (3, 50, 100):
        got, which = p.sparse(q, blocks, 1, 1)
        p.check_sparse(got, which, q, blocks, 1, 1, marks)
    p.free()


@KINDS
def test_many_rows_and_more_pages_than_threads(kind):
    p = Served(kind, (2, 2, 64), 4, [150, 0, 1, 1], [1400, 8, 1400, 5], seed=8)
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries()
    got, which = p.sparse(q, 30, 2, 3)
    p.check_sparse(got, which, q, 30, 2, 3, marks)
    p.free()


@KINDS
def test_missing_pages_are_chosen_last(kind):
    """Pages without an id: those between are lowest, those that are always taken count for nothing and are reported."""
    p = Served(kind, QWEN, 16, [1, 1], [400, 400], seed=9)
    p.table[0, [5, 9, 11]] = [-1, p.pages, 2**31 - 1]
    p.table[1, 0] = -1
    p.put()
    plain = p.table.copy()
    p.whole()
    p.status_after = p.flags()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries()
    got, which = p.sparse(q, 8, 1, 2)
    p.check_sparse(got, which, q, 8, 1, 2, marks)
    assert np.array_equal(p.table, plain) and p.flags() == 2
    p.free()


@KINDS
def test_bad_extents_leave_rows_alone(kind):
    p = Served(kind, QWEN, 16, [1, 2, 1], [100, 60, 90], seed=10)
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    n = upload(np.array([100, -5, 90], np.int32))
    p.batch.lengths = n
    q = p.queries()
    got, which = p.sparse(q, 4, 1, 1)
    assert p.flags() == 4 and np.all(got[1:3] == SENTINEL) and np.all(which[1:3] == -77)
    p.check_sparse(got, which, q, 4, 1, 1, marks, skip={1})
    cm.lib().gpu_free(n)
    p.free()


def test_too_many_pages_are_reported():
    """A sequence of more pages than one choice looks at is left out, the others are not; a loose max_length is no matter."""
    table = np.tile(np.arange(8, dtype=np.int32), (2, 2049))
    p = Served(BF16, (1, 1, 64), 1, [1, 1], [16385, 16384], table=table[:, :16392], extra=0)
    p.stride = 16392
    p.put()
    p.batch.max_length = 1 << 30
    p.whole()
    q = p.queries()
    got, which = p.sparse(q, 5, 1, 1)
    assert p.flags() == 4 and np.all(got[0] == SENTINEL) and np.all(which[0] == -77)
    marks = download(p.bounds, p.marks.shape, np.uint16)
    p.check_sparse(got, which, q, 5, 1, 1, marks, skip={0})
    p.free()


@KINDS
def test_wild_bounds_and_queries_stay_inside(kind):
    """Non-finite bounds or queries make the choice unspecified: still `blocks` pages of the sequence, in order."""
    for wild in (0x7f80, 0xff80, 0x7fc0, 0xffff):
        p = Served(kind, QWEN, 16, [2, 1], [700, 900], seed=11)
        marks = p.rng.integers(0, 65536, p.marks.shape).astype(np.uint16)
        marks[::2] = wild
        cm.lib().gpu_write(p.bounds, cm.ptr(marks), marks.nbytes)
        q = p.queries()
        q[0] = [np.nan, np.inf, -np.inf, 3e38][wild % 4]
        _, which = p.sparse(q, 10, 1, 2)
        for s, r, at in p.places():
            for h in range(2):
                w = which[r, h]
                assert np.all(np.diff(w) > 0) and w[0] == 0 and w[-1] == at // 16 and w[-2] == at // 16 - 1
        p.free()


@KINDS
@pytest.mark.parametrize("page", [7, 16, 24, 48, 100])
@pytest.mark.parametrize("what", ["non-finite", "huge"])
def test_what_no_query_sees_may_hold_anything(kind, page, what):
    """Free pages and rows behind a sequence's last hold NaN and infinities, or numbers far larger than any other."""
    news, lengths = [1, 3, 1], [1111, 500, page - 1]
    p = Served(kind, QWEN, page, news, lengths, seed=20)
    plain = Served(kind, QWEN, page, news, lengths, seed=20)
    used = np.zeros((p.pages, page), bool)
    for s, n in enumerate(lengths):
        for j in range(n):
            used[p.table[s, j // page], j % page] = True
    hide = ~used[:, None, :]
    if kind == BYTES:
        for kk, bad in ((0, np.nan), (1, np.inf)) if what == "non-finite" else ((0, 1e30), (1, 1e30)):
            p.scales[kk][np.broadcast_to(hide, p.scales[kk].shape)] = bad
    else:
        for kk, bad in ((0, 0x7FC0), (1, 0xFF80)) if what == "non-finite" else ((0, 0x7149), (1, 0xF149)):
            p.host[kk][np.broadcast_to(hide, p.host[kk].shape[:3])] = bad
    p.put()
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries()
    got, which = p.sparse(q, 5, 1, 1)
    plain.check_sparse(got, which, q, 5, 1, 1, marks)
    assert p.flags() == 0
    p.free()
    plain.free()


@KINDS
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-4, 12.0, 1e20])
def test_queries_of_any_size(kind, scale):
    p = Served(kind, QWEN, 32, [1, 3], [900, 700], seed=21, spread=0.3)
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries(scale)
    q[0, :128] = 0
    got, which = p.sparse(q, 6, 1, 1)
    p.check_sparse(got, which, q, 6, 1, 1, marks)
    p.free()


@KINDS
@pytest.mark.parametrize("spread", [2.0, 5.0])
@pytest.mark.parametrize("heads", [QWEN, ODD64])
def test_rows_of_unlike_size(kind, heads, spread):
    """K and V rows whose sizes differ by many powers of two, zero rows among them; the largest V row first, or last."""
    for blocks in (5, 60):
        p = Served(kind, heads, 16, [1, 2], [1500, 1600], seed=22, spread=spread)
        for s, place in ((0, 3), (1, 1590)):
            at = p.table[s, place // 16], slice(None), place % 16
            if kind == BYTES:
                p.scales[1][at] = 1e25
            else:
                p.host[1][at] = bf16(np.full(p.host[1][at].shape, 1e25, np.float32))
        if kind == BYTES:
            p.host[0][:, 0, 3], p.host[1][:, 1, 5] = 0, 0
        else:
            p.host[0][:, 0, 3], p.host[1][:, 1, 5] = 0, 0x8000
        p.put()
        p.whole()
        marks = download(p.bounds, p.marks.shape, np.uint16)
        q = p.queries(0.3 if spread < 3 else 0.01)
        got, which = p.sparse(q, blocks, 1, 1)
        p.check_sparse(got, which, q, blocks, 1, 1, marks)
        p.free()


@pytest.mark.parametrize("page", [16, 24, 64])
def test_scales_at_any_float(page):
    """Scales that start next to a 16-byte boundary."""
    p = Served(BYTES, QWEN, page, [1, 2], [1000, 777], seed=23)
    p.whole()
    q = p.queries()
    want, _ = p.sparse(q, 6, 1, 1)
    for off in (1, 2, 3):
        moved = upload(np.concatenate([np.full(off, np.nan, np.float32), p.scales.reshape(-1)]))
        p.cache.scales = moved + 4 * off
        got, _ = p.sparse(q, 6, 1, 1)
        cm.lib().gpu_free(moved)
        assert np.array_equal(got, want)
    p.free()


@KINDS
@pytest.mark.parametrize("dim", [64, 128])
def test_long_sums(kind, dim):
    """So many rows of nearly equal weight that the largest cluster's warps add up more than one chain each; V of one sign."""
    p = Served(kind, (2, 1, dim), 256, [1], [60000], seed=24)
    if kind == BYTES:
        p.host[1] = np.abs(p.host[1])
    else:
        p.host[1] = p.host[1] & np.uint16(0x7fff)
    p.put()
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries(0.01)
    got, which = p.sparse(q, 200, 1, 1)
    p.check_sparse(got, which, q, 200, 1, 1, marks)
    p.free()


@KINDS
def test_more_rows_than_one_pass_has_tables_for(kind):
    p = Served(kind, (2, 2, 64), 1, [1, 1100], [9000, 1200], seed=25)
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries()
    got, which = p.sparse(q, 8192, 2, 3)
    p.check_sparse(got, which, q, 8192, 2, 3, marks)
    p.free()


@KINDS
def test_thousands_of_equal_pages(kind):
    """One row in every page: the choice goes by the ids of thousands of equal scores."""
    p = Served(kind, (4, 2, 64), 1, [1, 1], [6000, 3000], seed=26)
    for x in p.host:
        x[:] = x[:1]
    p.scales[:] = p.scales[:, :1]
    x = p.table[0, [17, 5000]]  # two above the others
    if kind == BYTES:
        p.scales[0][x] *= 1.5
    else:
        p.host[0][x] = bf16(widen(p.host[0][x]) * np.float32(1.5))
    p.put()
    p.whole()
    marks = download(p.bounds, p.marks.shape, np.uint16)
    q = p.queries()
    for blocks in (9, 1000):
        got, which = p.sparse(q, blocks, 1, 1)
        p.check_sparse(got, which, q, blocks, 1, 1, marks)
    p.free()


@KINDS
def test_a_decoding_loop(kind):
    """Rotated append, bounds and attention over chosen pages, token by token and once more in one chunk: the same cache
    and bounds, and every token's attention held to its own cache."""
    n0, steps = 77, 20
    p = Served(kind, QWEN, 16, [1, 1], [n0 + steps, 40 + steps], seed=12)
    chunk = Served(kind, QWEN, 16, [steps, steps], [n0 + steps, 40 + steps], seed=12, table=p.table)
    chunk.host, chunk.scales = [x.copy() for x in p.host], p.scales.copy()
    chunk.put()
    rng = np.random.default_rng(13)
    x = rng.standard_normal((2 * steps, 16 * 128)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(128)).astype(np.float32)
    turn = (w, w, 1e-6, 1e6, 128)
    q = chunk.rotate(x, turn)
    chunk.whole()
    final, g = chunk.get(), cm.lib().gpu_open()
    rows = np.empty((2 * steps, 12 * 128), np.float32)
    for t in range(steps):
        p.lengths = np.array([n0 + t + 1, 40 + t + 1], np.int32)
        cm.lib().gpu_write(p.batch.lengths, cm.ptr(p.lengths.astype(np.int32)), 8)
        if t == 0:
            p.whole()
        pick = [t, steps + t]
        rows[pick] = p.rotate(x[pick], turn)
        marks = p.update()
        got, which = p.sparse(rows[pick], 3, 1, 1, gpu=g)
        p.host, p.scales = p.get()
        p.check_sparse(got, which, rows[pick], 3, 1, 1, marks)
    assert np.array_equal(rows, q)
    used = np.unique(p.table[p.table >= 0])
    for a, b in zip(p.host, final[0]):
        assert np.array_equal(a[used], b[used])
    if kind == BYTES:
        assert np.array_equal(p.scales[:, used], final[1][:, used])
    last = download(chunk.bounds, chunk.marks.shape, np.uint16)
    assert np.array_equal(widen(marks[used]), widen(last[used]))
    assert p.flags() == chunk.flags() == 0
    cm.lib().gpu_close(g)
    p.free()
    chunk.free()
