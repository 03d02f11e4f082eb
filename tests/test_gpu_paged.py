"""GPU tests of the paged K/V cache (include/gpu.h) against float64.

The oracle reads the pool's own bytes, so attention is held to its arithmetic
alone, element by element, by

    |out - exact| <= 2^-23 (64 S + 128 + n / 8) sum_j p_j |v_j|,   S = max_j sum_c max(|q_c|, |q|max / 16) |k_jc| / sqrt(dim)

over the n rows a query sees. A score q.k is a sum of dim products. Either each is
carried to 22 bits or more and they are added in FP32 with truncation, at most
dim / 16 + 1 <= 9 steps a half, two halves, below 2^-23 * 20 S in all; or q_c is off by
2^-24 of the largest |q| plus a rounding of its own (2^-24 |q|max = 2^-23 * 8 |q|max / 16,
so below 2^-23 * 9 S) and the products are exact. The factor log2(e) and the scale add 4
roundings, so 24 S. Both numerator and denominator of the softmax carry it,
as a factor: 2 * 24 S < 64 S with the base-2 subtraction's rounding (at most S) and
the running maximum's. exp2, the 22-bit weights, their scales, partial sums of at
most 64 truncating steps and the merge: below 128. Adding n / 16 partial results in
sequence rounds by 2^-24 each at most: n / 8 covers both sums.

Weights have a smallest step as well. In FP32 they underflow below 2^-149 of the
largest; carried to the tensor cores as two 16-bit halves, after scaling so that the
largest weight times row size is near 2^14, they are multiples of 2^-25, hence off by
up to 2^-39 of it, and a row's size is within 2 of its largest element. So

    + 2^-36 n max_j |v_j|

which only shows where the rows that carry the weight are far smaller than others.
"""
import numpy as np
import pytest

import cmachine_b200 as cm
from cmachine_b200 import ptr

pytestmark = pytest.mark.gpu

BF16, BYTES = 2, 3
SENTINEL = np.float32(-12345.5)


def upload(a):
    L = cm.lib()
    a = np.ascontiguousarray(a)
    p = L.gpu_alloc(max(a.nbytes, 16))
    if a.nbytes:
        L.gpu_write(p, ptr(a), a.nbytes)
    return p


def download(p, shape, dtype=np.float32):
    out = np.empty(shape, dtype)
    if out.nbytes:
        cm.lib().gpu_read(ptr(out), p, out.nbytes)
    return out


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def widen(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


class Pool:
    """A paged cache and one ragged batch on the device; news and lengths a sequence."""

    def __init__(self, kind, heads, page, news, lengths, seed=0, extra=3, spread=0.3, table=None, gap=0):
        self.kind, (self.qheads, self.kvheads, self.dim), self.page = kind, heads, page
        self.news, self.lengths = np.array(news), np.array(lengths)
        rng = self.rng = np.random.default_rng(seed)
        need = -(-self.lengths // page)
        self.pages, self.stride = int(need.sum()) + extra, max(1, int(need.max(initial=0)) + 1)
        shape = (self.pages, self.kvheads, page, self.dim)
        if table is None:
            order = rng.permutation(self.pages).astype(np.int32)
            table = np.full((len(news), self.stride), -7, np.int32)
            at = 0
            for s, n in enumerate(need):
                table[s, :n] = order[at:at + n]
                at += n
        self.table = np.array(table, np.int32)
        if kind == BYTES:
            self.host = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
            self.scales = np.exp(rng.standard_normal((2, *shape[:3])) * spread).astype(np.float32) * np.float32(0.02)
        else:
            self.host = [bf16(rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:3] + (1,)) * spread))
                         for _ in range(2)]
            self.scales = np.zeros((2, 1, 1, 1), np.float32)
        self.starts = np.concatenate([[0], np.cumsum(self.news)]).astype(np.int32) + np.int32(gap)
        self.rows = int(self.starts[-1])
        self.live = []
        self.put()

    def put(self):
        """The host's copies to the device."""
        self.free()
        up = [upload(x) for x in (*self.host, self.scales, self.starts, self.lengths.astype(np.int32), self.table,
                                  np.zeros(4, np.int32))]
        self.live = up
        self.status = up[6]
        self.cache = cm.PagedCache(self.kind, self.pages, self.page, self.kvheads, self.dim, up[0], up[1],
                                   up[2] if self.kind == BYTES else None)
        self.batch = cm.PagedBatch(len(self.news), self.rows, int(self.news.max(initial=0)), int(self.lengths.max(initial=0)),
                                   up[3], up[4], up[5], self.stride)

    def get(self):
        """The device's pool: (codes or BF16 bits of K and V, scales)."""
        dt = np.int8 if self.kind == BYTES else np.uint16
        return ([download(p, h.shape, dt) for p, h in zip(self.live[:2], self.host)],
                download(self.live[2], self.scales.shape))

    def flags(self):
        return int(download(self.status, 1, np.int32)[0])

    def values(self, kind):
        if self.kind == BYTES:
            return self.host[kind].astype(np.float64) * self.scales[kind][..., None]
        return widen(self.host[kind]).astype(np.float64)

    def held(self, s, kind):
        """Sequence s's rows [kvheads][length][dim], and which of them have a page."""
        v, n = self.values(kind), int(self.lengths[s])
        out, there = np.zeros((self.kvheads, n, self.dim)), np.zeros(n, bool)
        for j in range(n):
            page = self.table[s, j // self.page]
            if 0 <= page < self.pages:
                out[:, j] = v[page, :, j % self.page]
                there[j] = True
        return out, there

    def attend(self, q, window=0, sinks=0, pad=0, gpu=None, rows=None):
        """gpu_paged_attention of q [rows][qheads * dim]; out comes from a buffer of sentinels."""
        L = cm.lib()
        n, width = rows or max(self.rows, 1), self.qheads * self.dim
        out = upload(np.full((n, width + pad), SENTINEL, np.float32))
        wide = np.full((n, width + pad), np.nan, np.float32)
        wide[:q.shape[0], :width] = q
        dq = upload(wide)
        g = gpu or L.gpu_open()
        assert L.gpu_paged_attention(g, out, width + pad, dq, width + pad, self.cache, self.batch, self.qheads, window,
                                     sinks, self.status) == 0
        got = download(out, (n, width + pad))
        for p in (out, dq):
            L.gpu_free(p)
        if not gpu:
            L.gpu_close(g)
        assert np.all(got[:, width:] == SENTINEL)
        return got[:, :width]

    def queries(self, scale=1.0):
        return (self.rng.standard_normal((max(self.rows, 1), self.qheads * self.dim)) * scale).astype(np.float32)

    def check(self, got, q, window=0, sinks=0, skip=()):
        """Every element of every row within the bound above; returns the worst ratio."""
        d, group, worst = self.dim, self.qheads // self.kvheads, 0.0
        for s in range(len(self.news)):
            a, b = int(self.starts[s]), int(self.starts[s + 1])
            if s in skip or a == b:
                continue
            k, there = self.held(s, 0)
            v, _ = self.held(s, 1)
            n = int(self.lengths[s])
            at = (n - (b - a) + np.arange(b - a))[:, None]
            j = np.arange(n)[None]
            seen = (j <= at) & there[None]
            if window:
                seen &= (j > at - window) | (j < sinks)
            k, v = np.where(there[None, :, None], k, 0), np.where(there[None, :, None], v, 0)
            for h in range(self.qheads):
                x = q[a:b, h * d:(h + 1) * d].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    t = np.where(seen, x @ np.where(seen.any(0)[:, None], k[h // group], 0).T / np.sqrt(d), -np.inf)
                    big = np.where(seen, np.maximum(np.abs(x), np.abs(x).max(1, keepdims=True, initial=0) / 16) @ np.abs(np.where(seen.any(0)[:, None], k[h // group], 0)).T / np.sqrt(d), 0)
                m = t.max(1, keepdims=True, initial=-np.inf)
                p = np.where(seen, np.exp(t - np.where(np.isfinite(m), m, 0)), 0)
                total = p.sum(1, keepdims=True)
                p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
                vv = np.where(seen.any(0)[:, None], v[h // group], 0)
                exact, mass = p @ vv, p @ np.abs(vv)
                tol = 2.0**-23 * (64 * big.max(1, initial=0) + 128 + seen.sum(1) / 8)[:, None] * mass
                tol = tol + 2.0**-36 * seen.sum(1)[:, None] * np.abs(vv).max(initial=0)
                off = np.abs(got[a:b, h * d:(h + 1) * d] - exact)
                assert np.all(np.isfinite(got[a:b, h * d:(h + 1) * d])), (s, h)
                assert np.all(off <= tol), (s, h, float((off - tol).max()), np.argwhere(off > tol)[:4].tolist())
                worst = max(worst, float((off / np.maximum(tol, 1e-300)).max(initial=0)))
        return worst

    def free(self):
        for p in self.live:
            cm.lib().gpu_free(p)
        self.live = []


QWEN, GROUP4, MHA64, MQA, ONE, ODD64 = (12, 2, 128), (8, 2, 128), (4, 4, 64), (8, 1, 128), (1, 1, 128), (14, 2, 64)
GROUP5, GROUP3 = (15, 3, 128), (6, 2, 64)
KINDS = pytest.mark.parametrize("kind", [BF16, BYTES])

# (heads, page, new rows of each sequence, lengths)
SHAPES = [
    (QWEN, 16, [1], [1]), (QWEN, 16, [1], [2]), (QWEN, 16, [1, 1, 1], [15, 16, 17]), (QWEN, 64, [1] * 5, [300, 31, 64, 129, 1]),
    (MQA, 1, [1, 1], [33, 5]), (MHA64, 3, [1, 1], [100, 64]), (ODD64, 24, [1, 1, 1], [255, 256, 257]),
    (ONE, 100, [1], [1000]), (QWEN, 128, [1], [5000]), (GROUP4, 48, [2, 1], [77, 400]), (QWEN, 7, [2, 2], [130, 2]),
    (QWEN, 16, [3, 5, 1], [90, 5, 4]), (MHA64, 16, [16, 17, 15], [16, 40, 700]), (QWEN, 32, [21, 22], [21, 300]),
    (QWEN, 64, [43], [43]), (QWEN, 64, [42, 43, 44], [128, 129, 130]), (GROUP4, 24, [31, 32, 33, 64], [31, 128, 333, 64]),
    (MQA, 128, [100], [1500]), (ODD64, 48, [150, 1, 40], [150, 900, 1024]), (ONE, 256, [130, 257], [130, 600]),
    (QWEN, 50, [0, 4, 0, 60, 0], [9, 40, 0, 61, 200]),
    (QWEN, 16, [5, 6, 10, 11], [400, 36, 129, 65]), (GROUP5, 16, [1, 2, 3, 6, 7], [19, 300, 64, 6, 1025]), (GROUP5, 33, [51, 52, 1], [51, 90, 33]),
    (GROUP3, 64, [5, 6, 10, 11], [640, 129, 10, 65]), (GROUP3, 10, [85, 86, 171], [85, 400, 1111]),
]


@KINDS
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}p{s[1]}n{s[2]}l{s[3]}".replace(" ", ""))
def test_attention_matches_float64(kind, shape):
    heads, page, news, lengths = shape
    p = Pool(kind, heads, page, news, lengths, seed=len(lengths) + sum(lengths))
    q = p.queries()
    p.check(p.attend(q), q)
    assert p.flags() == 0
    p.free()


@KINDS
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 0), (100, 4), (128, 64), (129, 200), (700, 1), (10000, 4)])
@pytest.mark.parametrize("shape", [(QWEN, 16, [1, 1, 1], [700, 129, 3]), (GROUP4, 24, [6, 9], [300, 9]),
                                   (MHA64, 48, [70, 200, 1], [70, 777, 1300])], ids=["one", "few", "chunk"])
def test_window_and_first_rows(kind, window, sinks, shape):
    p = Pool(kind, *shape, seed=window + sinks)
    q = p.queries()
    p.check(p.attend(q, window, sinks), q, window, sinks)
    assert p.flags() == 0
    p.free()


@KINDS
@pytest.mark.parametrize("heads,most", [(QWEN, 1), (MHA64, 3), (GROUP5, 40)])
def test_many_sequences(kind, heads, most):
    """More sequences than one launch of the decode kernel counts, empty ones among them, and (40) both
    kernels of a call at once."""
    rng, count = np.random.default_rng(most), 300 if most < 40 else 140
    news = rng.integers(0, most + 1, count)
    lengths = np.maximum(news, rng.integers(0, 90, count))
    p = Pool(kind, heads, 16, news, lengths, seed=most)
    q = p.queries()
    p.check(p.attend(q), q)
    p.check(p.attend(q, 20, 3), q, 20, 3)
    assert p.flags() == 0
    p.free()


@KINDS
def test_no_status_word(kind):
    L = cm.lib()
    for news, lengths in (([2], [40]), ([60], [90])):
        p = Pool(kind, QWEN, 16, news, lengths, seed=6)
        p.table[0, 1] = p.pages
        p.put()
        q, g = p.queries(), L.gpu_open()
        dq, out = upload(q), upload(np.full_like(q, SENTINEL))
        assert L.gpu_paged_attention(g, out, q.shape[1], dq, q.shape[1], p.cache, p.batch, 12, 0, 0, None) == 0
        p.check(download(out, q.shape), q)
        for x in (dq, out):
            L.gpu_free(x)
        L.gpu_close(g)
        p.free()


@KINDS
def test_long_cache_with_few_rows(kind):
    p = Pool(kind, QWEN, 64, [1, 2, 1], [20011, 9000, 1], seed=5)
    q = p.queries(1.5)
    p.check(p.attend(q), q)
    p.free()


@KINDS
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-4, 12.0])
def test_query_sizes(kind, scale):
    """Equal scores, scores that vanish, and scores so far apart that one row takes nearly all the weight."""
    for news, lengths in (([1, 3], [200, 70]), ([140], [333])):
        p = Pool(kind, QWEN, 32, news, lengths, seed=3)
        q = p.queries(scale)
        q[0, :128] = 0
        p.check(p.attend(q), q)
        p.free()


@KINDS
def test_rows_of_unlike_size(kind):
    """K and V rows whose sizes differ by many powers of two, zero rows among them."""
    for news, lengths in (([1, 3], [200, 70]), ([140], [333])):
        p = Pool(kind, QWEN, 32, news, lengths, seed=4, spread=2.0)
        if kind == BYTES:
            p.host[0][:, 0, 3], p.host[1][:, 1, 5] = 0, 0
            p.scales[0][:, 0, 3], p.scales[1][:, 1, 5] = 1, 1
        else:
            p.host[0][:, 0, 3], p.host[1][:, 1, 5] = 0, 0x8000
        p.put()
        q = p.queries(0.3)
        p.check(p.attend(q), q)
        p.free()


@KINDS
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("what", ["non-finite", "huge"])
@pytest.mark.parametrize("news,lengths", [([1, 1], [37, 80]), ([4, 3], [50, 20]), ([90, 33], [130, 33])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (11, 2)])
def test_what_nothing_sees_may_hold_anything(kind, news, lengths, window, sinks, what, page):
    """NaN and infinities, or numbers far larger than any other, in free pages, behind a sequence's last row and
    before every window, and freed pages there (their entries may also name a page of such rows)."""
    p = Pool(kind, QWEN, page, news, lengths, seed=9)
    plain = Pool(kind, QWEN, page, news, lengths, seed=9)
    used = np.zeros((p.pages, page), bool)
    for s, n in enumerate(lengths):
        low = max(0, n - news[s] - window + 1) if window else 0
        for j in range(n):
            if j >= low or j < sinks:
                used[p.table[s, j // page], j % page] = True
    free = int(np.argwhere(~used.any(1))[0, 0])
    for s, n in enumerate(lengths):
        low = max(0, n - news[s] - window + 1) if window else 0
        if window:
            for k in range(-(-sinks // page), low // page):
                p.table[s, k] = [-1, 2**31 - 1, p.pages, free][(s + k) % 4]
    hide = ~used[:, None, :]
    if kind == BYTES:
        for kk, bad in ((0, np.nan), (1, np.inf)) if what == "non-finite" else ((0, 1e30), (1, 1e30)):
            p.scales[kk][np.broadcast_to(hide, p.scales[kk].shape)] = bad
    else:
        for kk, bad in ((0, 0x7FC0), (1, 0xFF80)) if what == "non-finite" else ((0, 0x7149), (1, 0xF149)):
            p.host[kk][np.broadcast_to(hide, p.host[kk].shape[:3])] = bad
    p.put()
    q = p.queries()
    plain.check(p.attend(q, window, sinks), q, window, sinks)
    assert p.flags() == 0
    p.free()
    plain.free()


@KINDS
def test_a_non_finite_row_touches_only_queries_that_see_it(kind):
    """Row 40 of a 64-row chunk holds NaN: the queries before it are right."""
    for news, lengths in (([64], [64]), ([5], [43])):
        p = Pool(kind, QWEN, 16, news, lengths, seed=21)
        for kk in (0, 1):
            if kind == BYTES:
                p.scales[kk][p.table[0, 40 // 16], :, 40 % 16] = np.nan
            else:
                p.host[kk][p.table[0, 40 // 16], :, 40 % 16, 5] = 0x7FC0
        p.put()
        q = p.queries()
        got = p.attend(q)
        first = lengths[0] - news[0]
        keep = 40 - first
        small = Pool(kind, QWEN, 16, [keep], [40], seed=21)
        small.table, small.host, small.scales, small.pages, small.stride = p.table, p.host, p.scales, p.pages, p.stride
        small.check(got[:keep], q)
        # The window of a later query has left the row.
        p.lengths[:] = lengths
        got = p.attend(q, 3, 0)
        if first + news[0] > 43:
            assert np.all(np.isfinite(got[43 - first:]))
        p.free()
        small.free()


@KINDS
def test_a_non_finite_query_touches_only_its_own_row(kind):
    for news, lengths in (([3], [60]), ([50], [60])):
        p = Pool(kind, QWEN, 16, news, lengths, seed=22)
        q = p.queries()
        clean = q.copy()
        q[1, 5], q[2, 130] = np.nan, np.inf
        got = p.attend(q)
        assert not np.all(np.isfinite(got[1, :128]))
        got[1, :128] = p.attend(clean)[1, :128]
        got[2, 128:256] = p.attend(clean)[2, 128:256]
        p.check(got, clean)
        p.free()


@KINDS
@pytest.mark.parametrize("news,lengths", [([4, 2], [2, 0]), ([60, 20], [21, 0]), ([1, 1], [0, 3])])
def test_queries_that_see_nothing_get_zeros(kind, news, lengths):
    p = Pool(kind, QWEN, 16, news, lengths, seed=11)
    q = p.queries()
    for _ in range(20):  # nothing of the queries' own staging may show, whichever warp is first
        got = p.attend(q)
        for s, (n, length) in enumerate(zip(news, lengths)):
            a = p.starts[s]
            assert np.all(got[a:a + max(0, n - length)] == 0)
    p.check(got, q)
    assert p.flags() == 0
    p.free()


@KINDS
@pytest.mark.parametrize("news,lengths", [([1, 2], [50, 70]), ([30, 50], [50, 70])])
def test_rows_of_no_sequence_are_left_alone(kind, news, lengths):
    """Rows before the first sequence and behind the last, and strides wider than a row."""
    p = Pool(kind, QWEN, 16, news, lengths, seed=12, gap=2)
    n = p.rows + 3
    p.batch.rows = n
    q = (p.rng.standard_normal((n, p.qheads * p.dim))).astype(np.float32)
    got = p.attend(q, pad=20, rows=n)
    assert np.all(got[:2] == SENTINEL) and np.all(got[p.rows:] == SENTINEL)
    p.check(got, q)
    p.free()


@KINDS
@pytest.mark.parametrize("news,lengths", [([1, 1], [90, 40]), ([50, 40], [90, 40])])
def test_bad_pages_are_reported_and_seen_by_nobody(kind, news, lengths):
    p = Pool(kind, QWEN, 16, news, lengths, seed=13)
    p.table[0, 2], p.table[1, 0], p.table[1, 1] = -1, p.pages, 2**31 - 1
    p.put()
    q = p.queries()
    got = p.attend(q)
    assert p.flags() == 2
    p.check(got, q)
    p.free()


@KINDS
@pytest.mark.parametrize("count", [1, 40])
def test_bad_extents_leave_the_sequence_out(kind, count):
    p = Pool(kind, QWEN, 16, [count] * 3, [60, 70, 80], seed=14)
    q = p.queries()
    for what in ("length", "table", "start", "order"):
        starts, lengths = p.starts.copy(), p.lengths.astype(np.int32)
        if what == "length":
            lengths[1] = 81
        elif what == "table":
            lengths[1] = -1
        elif what == "start":
            starts[3] = p.rows + 1
        else:
            starts[1] = starts[2] + 1
        L = cm.lib()
        L.gpu_write(p.live[3], ptr(starts), starts.nbytes)
        L.gpu_write(p.live[4], ptr(lengths), lengths.nbytes)
        L.gpu_zero(p.status, 4)
        got = p.attend(q)
        assert p.flags() == 4, what
        bad = {"length": [1], "table": [1], "start": [2], "order": [0, 1]}[what]
        for s in bad:
            rows = got[p.starts[s]:p.starts[s + 1]]
            assert np.all(rows == SENTINEL), what
        p.check(got, q, skip=bad)
    p.free()


@KINDS
def test_sequences_share_pages(kind):
    """Two sequences on one prefix's pages."""
    table = np.array([[4, 1, 0, -1], [4, 1, 2, -1]], np.int32)
    p = Pool(kind, QWEN, 16, [1, 12], [40, 47], seed=15, table=table)
    q = p.queries()
    p.check(p.attend(q), q)
    p.free()


@KINDS
def test_the_same_bits_every_time_and_handles_reused(kind):
    """Large, small, large on one handle: its scratch grows and is used again."""
    L = cm.lib()
    g = L.gpu_open()
    big, small = Pool(kind, QWEN, 32, [1, 5, 70], [4000, 900, 800], seed=16), Pool(kind, MHA64, 16, [1], [33], seed=17)
    qb, qs = big.queries(), small.queries()
    first = [big.attend(qb, gpu=g), small.attend(qs, gpu=g)]
    for _ in range(3):
        assert np.array_equal(big.attend(qb, gpu=g), first[0])
        assert np.array_equal(small.attend(qs, gpu=g), first[1])
    big.check(first[0], qb)
    small.check(first[1], qs)
    # A sequence's result does not depend on the handle.
    assert np.array_equal(big.attend(qb), first[0])
    L.gpu_close(g)
    big.free()
    small.free()


# ---------------------------------------------------------------- append and read back
def encode(x):
    """The byte codec in NumPy single precision."""
    m = np.abs(x).max(-1)
    scale = np.where(m > 0, m / np.float32(127), np.float32(1)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = (x / scale[..., None]).astype(np.float32)
    y = np.where(scale[..., None] > 0, y, 0)
    return np.clip(np.trunc(y + np.where(y < 0, -0.5, 0.5)), -127, 127).astype(np.int8), scale


def store(p, k, v, stride=None):
    L = cm.lib()
    dk, dv = upload(k), upload(v)
    assert L.gpu_paged_append(p.cache, p.batch, dk, dv, stride or p.kvheads * p.dim, p.status) == 0
    L.gpu_sync()
    for x in (dk, dv):
        L.gpu_free(x)


def read_back(p, pad=0, rows=None):
    L = cm.lib()
    n, width = rows or max(p.rows, 1), p.kvheads * p.dim
    outs = [upload(np.full((n, width + pad), SENTINEL, np.float32)) for _ in range(2)]
    assert L.gpu_paged_read(p.cache, p.batch, outs[0], outs[1], width + pad, p.status) == 0
    got = [download(x, (n, width + pad)) for x in outs]
    for x in outs:
        L.gpu_free(x)
    assert all(np.all(g[:, width:] == SENTINEL) for g in got)
    return [g[:, :width] for g in got]


@KINDS
@pytest.mark.parametrize("heads,page,news,lengths", [
    (QWEN, 16, [1], [1]), (QWEN, 64, [1] * 7, [1, 64, 65, 300, 2, 63, 128]), (MHA64, 3, [10, 0, 1], [40, 5, 1]),
    (ODD64, 24, [33, 70, 1], [33, 500, 24]), (MQA, 1, [9], [9]), (GROUP4, 100, [300, 5], [777, 5]), (ONE, 65536, [20], [33])])
def test_append_and_read_back(kind, heads, page, news, lengths):
    p = Pool(kind, heads, page, news, lengths, seed=31)
    x = [(p.rng.standard_normal((p.rows, p.kvheads, p.dim)) * np.exp(p.rng.standard_normal((p.rows, p.kvheads, 1)))).astype(np.float32)
         for _ in range(2)]
    x[0][0, 0] = 0  # a zero row
    x[1][-1, -1, :] = np.float32(1e-44)  # a row whose scale underflows
    x[0][-1, -1, 3] = np.float32(3.0e38)
    if p.dim == 64:
        x[1][0, 0] = np.arange(64) - 31.5  # halves: rounded away from zero after the division
    store(p, *x)
    pool, scales = p.get()
    want, wscales = [h.copy() for h in p.host], p.scales.copy()
    for s in range(len(news)):
        for i in range(news[s]):
            j = lengths[s] - news[s] + i
            at = (p.table[s, j // page], slice(None), j % page)
            for kk in (0, 1):
                row = x[kk][p.starts[s] + i]
                if kind == BYTES:
                    want[kk][at], wscales[kk][at] = encode(row)
                else:
                    want[kk][at] = bf16(row)
    for kk in (0, 1):  # every other row of the pool is as it was
        assert np.array_equal(pool[kk], want[kk])
    assert np.array_equal(scales, wscales)
    assert p.flags() == 0
    p.host, p.scales = want, wscales
    got = read_back(p)
    for kk in (0, 1):
        for s in range(len(news)):
            v, _ = p.held(s, kk)
            new = v[:, lengths[s] - news[s]:].transpose(1, 0, 2).reshape(news[s], p.kvheads * p.dim)
            assert np.array_equal(got[kk][p.starts[s]:p.starts[s + 1]], new.astype(np.float32))
    p.free()


def test_codes_near_halves():
    """Quotients at, just below and just above halves are rounded as the division says: every element of
    4096 rows against single-precision NumPy."""
    p = Pool(BYTES, (1, 1, 128), 64, [4096], [4096], seed=35)
    rng = p.rng
    m = np.exp(rng.standard_normal((4096, 1)) * 4).astype(np.float32)
    scale = (m / np.float32(127)).astype(np.float32)
    half = (rng.integers(-127, 127, (4096, 128)) + 0.5).astype(np.float32)
    x = (half * scale).astype(np.float32)
    side = rng.integers(0, 3, x.shape)  # the product itself, or its neighbour on either side
    x = np.nextafter(x, np.where(side == 0, x, np.where(side == 1, np.float32(np.inf), np.float32(-np.inf))))
    assert np.all(np.isfinite(x))
    x = np.clip(x, -m, m).astype(np.float32)
    x[:, 0] = m[:, 0]
    x = x.reshape(4096, 1, 128)
    store(p, x, -x)
    (codes, vcodes), scales = p.get()
    want, ws = encode(x)
    at = p.table[0][np.arange(4096) // 64]
    assert np.array_equal(codes[at, :, np.arange(4096) % 64], want)
    assert np.array_equal(vcodes[at, :, np.arange(4096) % 64], -want)
    assert np.array_equal(scales[0][at, :, np.arange(4096) % 64], ws)
    p.free()


def test_append_gives_the_ring_codec_s_bits():
    """The same codes and scales as gpu_encode_current."""
    L = cm.lib()
    p = Pool(BYTES, QWEN, 16, [5], [21], seed=32)
    x = [p.rng.standard_normal((5, 2, 128)).astype(np.float32) for _ in range(2)]
    store(p, *x)
    pool, scales = p.get()
    codes, sc, bad = upload(np.zeros(2 * 2 * 5 * 128, np.int8)), upload(np.zeros(4 * 5, np.float32)), upload(np.zeros(4, np.int32))
    for i in range(5):
        k, v = upload(x[0][i]), upload(x[1][i])
        assert L.gpu_encode_current(codes, codes + 2 * 5 * 128, sc, k, v, 5, i, bad) == 0
        L.gpu_free(k)
        L.gpu_free(v)
    ring, rscales = download(codes, (2, 2, 5, 128), np.int8), download(sc, (2, 2, 5))
    for i in range(5):
        page, row = p.table[0, (16 + i) // 16], (16 + i) % 16
        for kk in (0, 1):
            assert np.array_equal(pool[kk][page, :, row], ring[kk][:, i])
            assert np.array_equal(scales[kk][page, :, row], rscales[kk][:, i])
    for x in (codes, sc, bad):
        L.gpu_free(x)
    p.free()


@KINDS
def test_append_from_a_fused_projection_and_non_finite_rows(kind):
    """K and V inside rows of queries, keys and values; rows with NaN or infinity are stored as zeros and reported."""
    L = cm.lib()
    p = Pool(kind, QWEN, 16, [3, 2], [40, 18], seed=33)
    width = 16 * 128
    x = p.rng.standard_normal((5, width)).astype(np.float32)
    x[1, 12 * 128 + 7], x[4, 15 * 128] = np.nan, -np.inf
    dx = upload(x)
    assert L.gpu_paged_append(p.cache, p.batch, dx + 12 * 512, dx + 14 * 512, width, p.status) == 0
    got = read_back(p, pad=4)
    assert p.flags() == 1
    x[1, 12 * 128:13 * 128], x[4, 15 * 128:] = 0, 0
    for kk in (0, 1):
        new = x[:, (12 + 2 * kk) * 128:(14 + 2 * kk) * 128].reshape(5, 2, 128)
        if kind == BYTES:
            c, s = encode(new)
            new = c.astype(np.float32) * s[..., None]
        else:
            new = widen(bf16(new))
        assert np.array_equal(got[kk].reshape(5, 2, 128), new)
    L.gpu_free(dx)
    p.free()


@KINDS
def test_append_and_read_without_pages_or_places(kind):
    """Rows at negative places and rows without a page are skipped; bad extents leave a sequence out; others are right."""
    p = Pool(kind, MHA64, 16, [6, 4, 3], [4, 20, 33], seed=34)
    p.table[1, 1] = p.pages
    p.table[2, 2] = -1
    p.put()
    x = [p.rng.standard_normal((p.rows, 4, 64)).astype(np.float32) for _ in range(2)]
    before = p.get()
    store(p, *x)
    assert p.flags() == 2
    after = p.get()
    # Sequence 0's places 0 to 3; sequence 2's 30 and 31 (32 has no page).
    touched = {(int(p.table[0, 0]), j) for j in range(4)} | {(int(p.table[2, 1]), j) for j in (14, 15)}
    for kk in (0, 1):
        changed = {tuple(int(c) for c in t) for t in np.argwhere((before[0][kk] != after[0][kk]).any((1, 3)))}
        assert changed == touched
    p.host, p.scales = after
    got = read_back(p, rows=p.rows + 2)
    for kk in (0, 1):
        assert np.all(got[kk][:2] == 0) and np.all(got[kk][6:10] == 0) and np.all(got[kk][12] == 0)
        assert np.all(got[kk][p.rows:] == SENTINEL)
        v = p.values(kk)
        assert np.array_equal(got[kk][2].reshape(4, 64), v[p.table[0, 0], :, 0].astype(np.float32))
        assert np.array_equal(got[kk][11].reshape(4, 64), v[p.table[2, 1], :, 15].astype(np.float32))
    lengths = np.array([4, 99, 33], np.int32)
    cm.lib().gpu_write(p.live[4], ptr(lengths), 12)
    cm.lib().gpu_zero(p.status, 4)
    got = read_back(p)
    assert p.flags() == 6 and np.all(got[0][6:10] == SENTINEL)
    p.free()


@KINDS
def test_a_decoding_program(kind):
    """A prompt in two chunks, then single tokens, three sequences of their own lengths: each call appends and
    attends, all queued on the library's stream, and every output is the one over the rows stored so far."""
    L = cm.lib()
    heads, page, width = QWEN, 16, 16 * 128
    lengths, plan = [0, 0, 0], [[40, 1, 17], [9, 30, 1], [1, 1, 1], [1, 1, 1], [1, 0, 1], [1, 1, 1]]
    final = [sum(step[s] for step in plan) for s in range(3)]
    p = Pool(kind, heads, page, [0, 0, 0], final, seed=41)
    g, rng, outs, held = L.gpu_open(), p.rng, [], []
    for news in plan:
        lengths = [a + b for a, b in zip(lengths, news)]
        starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        x = rng.standard_normal((int(starts[-1]), width)).astype(np.float32)
        dx, out = upload(x), upload(np.full((x.shape[0], 12 * 128), SENTINEL, np.float32))
        ds, dl = upload(starts), upload(np.array(lengths, np.int32))
        batch = cm.PagedBatch(3, x.shape[0], max(news), max(lengths), ds, dl, p.live[5], p.stride)
        assert L.gpu_paged_append(p.cache, batch, dx + 12 * 512, dx + 14 * 512, width, p.status) == 0
        assert L.gpu_paged_attention(g, out, 12 * 128, dx, width, p.cache, batch, 12, 0, 0, p.status) == 0
        outs.append((x, out, starts, list(lengths), news))
        held += [dx, out, ds, dl]
    p.host, p.scales = p.get()
    for x, out, starts, lens, news in outs:
        step = Pool(kind, heads, page, news, lens, seed=41, table=p.table)
        step.host, step.scales, step.pages, step.stride = p.host, p.scales, p.pages, p.stride
        step.check(download(out, (x.shape[0], 12 * 128)), x[:, :12 * 128])
        step.free()
    assert p.flags() == 0
    for x in held:
        L.gpu_free(x)
    L.gpu_close(g)
    p.free()
