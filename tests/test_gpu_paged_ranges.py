"""GPU tests of the paged K/V cache at the ends of its ranges: batches of several launches, values of unlike
size, long sums, small queries, loose maxima. The pool, its float64 oracle and its bound are
tests/test_gpu_paged.py's unless a test states its own."""
import time

import numpy as np
import pytest

import cmachine_b200 as cm
from test_gpu_paged import (BF16, BYTES, KINDS, MHA64, QWEN, SENTINEL, Pool, bf16, encode, read_back, store,
                            upload, widen)

pytestmark = pytest.mark.gpu


@KINDS
def test_many_launches_beside_chunks_give_the_same_bits(kind):
    """Chunks, and so many short sequences that the decode kernel takes four launches beside them: every launch
    leaves its counters and partials to the next. Long and short sequences alternate, so row tiles are cut."""
    rng = np.random.default_rng(7)
    news = np.where(np.arange(400) % 50 == 7, 70, rng.integers(0, 3, 400))
    lengths = np.maximum(news, np.where(np.arange(400) % 9 == 0, 900, rng.integers(0, 60, 400)))
    p = Pool(kind, MHA64, 16, news, lengths, seed=8)
    p.values = [p.values(0), p.values(1)].__getitem__  # once, not for each sequence
    q, g = p.queries(), cm.lib().gpu_open()
    first = p.attend(q, gpu=g)
    p.check(first, q)
    for _ in range(30):
        assert np.array_equal(p.attend(q, gpu=g), first)
    assert p.flags() == 0
    cm.lib().gpu_close(g)
    p.free()


def check_by_query(p, got, q, window=0, sinks=0):
    """Every element against float64, by a bound that takes nothing from rows the query does not see and little from
    rows that hardly count for it. With e_j = exp(t_j) off by a factor 1 + d_j, the result sum e v / sum e is off
    by at most

        sum_j p_j |d_j| |v_j| + (sum_j p_j |d_j|) (sum_j p_j |v_j|),   |d_j| <= 2^-23 (32 S_j + 4 S_a + 64 + n / 16),

    S_j = sum_c max(|q_c|, |q|max / 16) |k_jc| / sqrt(dim) and a the row of the largest score: a score is off by 24 S_j
    and the subtraction of a reference near t_a by S_j + S_a (both roundings), the rest is exp2, a 22-bit weight, its
    scale and the sums' (as in the bound of tests/test_gpu_paged.py). Weights carried as FP16 halves are multiples of
    2^-24, off by 2^-25 at most, where rows whose sizes differ by no more than 2^8 share a scale that brings the largest
    weight times size to 2^11 or more: 2^-25 / 2^(11 - 8) = 2^-28 of the size of the row that counts most, twice that
    for the part of a size above its power of two."""
    d, group = p.dim, p.qheads // p.kvheads
    for s in range(len(p.news)):
        a, b = int(p.starts[s]), int(p.starts[s + 1])
        if a == b:
            continue
        (k, there), (v, _) = p.held(s, 0), p.held(s, 1)
        n = int(p.lengths[s])
        at, j = (n - (b - a) + np.arange(b - a))[:, None], np.arange(n)[None]
        seen = (j <= at) & there[None]
        if window:
            seen &= (j > at - window) | (j < sinks)
        for h in range(p.qheads):
            x = q[a:b, h * d:(h + 1) * d].astype(np.float64)
            kk, vv = k[h // group], v[h // group]
            t = np.where(seen, x @ kk.T / np.sqrt(d), -np.inf)
            size = np.maximum(np.abs(x), np.abs(x).max(1, keepdims=True) / 16) @ np.abs(kk).T / np.sqrt(d)
            w = np.exp(t - t.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            top = np.take_along_axis(size, t.argmax(1)[:, None], 1)
            count = seen.sum(1, keepdims=True)
            wd = w * 2.0**-23 * (32 * size + 4 * top + 64 + count / 16)
            tol = wd @ np.abs(vv) + wd.sum(1, keepdims=True) * (w @ np.abs(vv))
            tol = tol + count * 2.0**-27 * (w * np.abs(vv).max(1)[None]).max(1, keepdims=True)
            off = np.abs(got[a:b, h * d:(h + 1) * d] - w @ vv)
            assert np.all(off <= tol), (s, h, float((off / tol).max()), np.argwhere(off > tol)[:4].tolist())


@KINDS
@pytest.mark.parametrize("power", [10, 30, 60])
@pytest.mark.parametrize("news,lengths,place,window,sinks", [
    ([64], [64], 40, 0, 0), ([64], [64], 40, 9, 2), ([3, 200], [3, 700], 650, 0, 0), ([200], [300], 3, 0, 0),
    ([5], [43], 41, 0, 0), ([5], [43], 41, 2, 0), ([2, 5], [40, 2000], 1997, 0, 0), ([5], [300], 2, 0, 0), ([5], [300], 297, 0, 4)])
def test_a_huge_row_counts_only_where_it_is_seen(kind, power, news, lengths, place, window, sinks):
    """A row whose V is 2^power times the others', in the middle of a chunk and of a short run: the queries before it
    and those whose window has left it are as right as without it."""
    p = Pool(kind, QWEN, 16, news, lengths, seed=power + place)
    s = len(news) - 1
    at = (p.table[s, place // 16], slice(None), place % 16)
    if kind == BYTES:
        p.scales[1][at] *= np.float32(2.0**power)
    else:
        p.host[1][at] = np.where(p.host[1][at] & 0x7F80, p.host[1][at] + (power << 7), 0)
    p.put()
    q = p.queries()
    check_by_query(p, p.attend(q, window, sinks), q, window, sinks)
    assert p.flags() == 0
    p.free()


@KINDS
@pytest.mark.parametrize("power", [30, 60])
@pytest.mark.parametrize("small", [False, True])
@pytest.mark.parametrize("news,lengths,places", [([64], [64], [0]), ([64], [200], [150]), ([200], [900], [5, 300, 640]),
                                                 ([5], [43], [0]), ([5], [300], [17, 150]), ([1], [3000], [0, 1600])])
def test_a_huge_row_with_no_weight(kind, power, small, news, lengths, places):
    """Rows whose V is 2^power times the others' and whose weight vanishes for every query that sees them (small: the
    other way round, rows of 2^-power that take all the weight of a query)."""
    p = Pool(kind, QWEN, 16, news, lengths, seed=power + places[0])
    q = (p.queries() * 0.1 + np.float32(0.5 if not small else 0.1)).astype(np.float32)
    for place in places:
        at = (p.table[0, place // 16], slice(None), place % 16)
        if kind == BYTES:
            p.host[0][at] = 127 if small else -127
            p.scales[0][at] = np.float32((60 if small else 40) / 127)
            p.scales[1][at] *= np.float32(2.0**(-power if small else power))
        else:
            p.host[0][at] = 0x4270 if small else 0xC220  # 60, -40
            p.host[1][at] = np.where(p.host[1][at] & 0x7F80, (p.host[1][at].astype(int) + ((-power if small else power) << 7)).astype(np.uint16), 0)
    p.put()
    check_by_query(p, p.attend(q), q)
    p.free()


@KINDS
@pytest.mark.parametrize("heads,new", [((4, 4, 64), 1), ((8, 4, 64), 5), ((8, 4, 64), 10)], ids=["8", "16", "32"])
def test_long_sums(kind, heads, new):
    """262,144 rows of positive values, in so many sequences (all on the same pages) that most are not split: a warp
    sums up to K = 2048 steps of 16 rows. Added in FP32 to nearest, K sums err by about sqrt(K) / 4 units of 2^-24
    (each by up to half a unit of a partial sum, with either sign): 2 sqrt(K) is eight times that, and 32 covers a
    step's products, the warps' merge and the division. Weights are off by 2^-23 (32 S + 8), S as in check_by_query, in
    numerator and denominator. An adder that truncates every step is off by 2e-4 here, all to one side."""
    length, page, seqs = 262144, 256, 80
    p = Pool(kind, heads, page, [new], [length], seed=3, extra=0)
    size = np.exp(p.rng.standard_normal((p.pages, p.kvheads, page)) * 0.3).astype(np.float32)
    value = p.rng.integers(64, 128, p.host[1].shape)
    if kind == BYTES:
        p.host[1], p.scales[1] = value.astype(np.int8), size / 64
    else:
        p.host[1] = bf16((value / 64).astype(np.float32) * size[..., None])
    q = np.tile(p.queries(0.02)[None], (seqs, 1, 1)).reshape(seqs * new, -1)
    p.news, p.lengths = np.full(seqs, new), np.full(seqs, length)
    p.table = np.tile(p.table, (seqs, 1))
    p.starts = (np.arange(seqs + 1) * new).astype(np.int32)
    p.rows = seqs * new
    p.put()
    got = p.attend(q).reshape(seqs, new, p.qheads, p.dim)
    assert p.flags() == 0
    p.free()
    pages, group = p.table[0, :p.pages], p.qheads // p.kvheads
    k, v = (p.values(kk)[pages].transpose(1, 0, 2, 3).reshape(p.kvheads, length, p.dim) for kk in (0, 1))
    for i in range(new):
        n = length - (new - 1 - i)
        for h in range(p.qheads):
            x = q[i, h * p.dim:(h + 1) * p.dim].astype(np.float64)
            w = np.exp(k[h // group, :n] @ x / 8)
            exact = (w @ v[h // group, :n]) / w.sum()
            s = float((np.abs(k[h // group]) @ np.maximum(np.abs(x), np.abs(x).max() / 16)).max() / 8)
            off = np.abs(got[:, i, h] / exact - 1).max()
            assert off <= (2 * np.sqrt(n / 128) + 32) * 2.0**-24 + 2 * 2.0**-23 * (32 * s + 8), (i, h, float(off))


@KINDS
@pytest.mark.parametrize("news,lengths", [([1, 3], [60, 33]), ([90], [100])])
@pytest.mark.parametrize("q_size,k_size", [(1e-31, 1e30), (1.5e-34, 1e32), (2e-35, 1e32), (1e-42, 1e30), (1e29, 1e-31)])
def test_small_queries_against_large_rows(kind, news, lengths, q_size, k_size):
    """Queries and cached rows at opposite ends of FP32, whose products are ordinary numbers."""
    p = Pool(kind, QWEN, 16, news, lengths, seed=2)
    if kind == BYTES:
        p.scales[0] *= np.float32(k_size)
    else:
        p.host[0] = bf16(widen(p.host[0]) * np.float32(k_size))
    p.put()
    q = p.queries(q_size)
    check_by_query(p, p.attend(q), q)
    p.free()


@KINDS
def test_rows_at_the_top_of_fp32(kind):
    """In BF16 values from 2^128 - 2^119 on round to infinity, and FP32's largest number over 127 times 127 does: such a
    row is stored as zeros and reported, as one of infinities is; any other finite one is an ordinary one."""
    p = Pool(kind, QWEN, 16, [4], [20], seed=33)
    x = [p.rng.standard_normal((4, 2, 128)).astype(np.float32) for _ in range(2)]
    edge = np.float32(2.0**128 - 2.0**119)
    x[0][1, 0, 5], x[1][0, 1, 127] = edge, -np.finfo(np.float32).max
    x[1][2, 1, 5] = np.nextafter(edge, np.float32(0))
    store(p, *x)
    assert p.flags() == 1
    x[1][0, 1] = 0
    if kind == BF16:
        x[0][1, 0] = 0
    got = read_back(p)
    for kk in (0, 1):
        if kind == BYTES:
            codes, scale = encode(x[kk])
            want = codes.astype(np.float32) * scale[..., None]
        else:
            want = widen(bf16(x[kk]))
        assert np.all(np.isfinite(want)) and np.array_equal(got[kk].reshape(4, 2, 128), want)
    p.free()


@pytest.mark.parametrize("news,lengths", [([32, 20, 1, 0, 7], [300, 20, 65, 9, 1000]), ([300], [900]), ([1, 200], [400, 333])])
def test_a_table_for_very_long_sequences(news, lengths):
    """max_length is an upper bound: tables of 2^30 places for short sequences, whose steps would pass 2^31, are
    taken in launches of some KV heads each."""
    p = Pool(BYTES, (16, 16, 64), 4096, news, lengths, seed=6, extra=0)
    table = np.full((len(news), 2**18), -1, np.int32)
    table[:, :p.stride] = p.table
    p.table, p.stride = table, table.shape[1]
    p.put()
    p.batch.max_length = 2**30
    q = p.queries()
    p.check(p.attend(q), q)
    assert p.flags() == 0
    p.free()


@KINDS
@pytest.mark.parametrize("count", [7, 512, 1300])
def test_chunks_among_many_sequences(kind, count):
    """Chunks at the first, last and other places among single tokens and sequences without rows, more of them than
    a CTA's threads; one chunk's extents do not fit. Loose maxima and buffers change no result beyond the bound."""
    rng = np.random.default_rng(count)
    news, lengths = rng.integers(0, 2, count), rng.integers(1, 40, count)
    chunks = sorted({0, 3, count // 2, min(511, count - 1), min(512, count - 1), count - 1})
    for i, s in enumerate(chunks):
        news[s], lengths[s] = 60 + 41 * i, 70 + 300 * i
    p = Pool(kind, MHA64, 16, news, lengths, seed=count)
    p.values = [p.values(0), p.values(1)].__getitem__  # once, not for each sequence
    q = p.queries()
    p.check(p.attend(q), q)
    assert p.flags() == 0
    p.batch.max_new, p.batch.rows = 5000, p.rows + 4000
    more = np.zeros((p.rows + 4000, q.shape[1]), np.float32)
    more[:p.rows] = q
    got = p.attend(more, rows=p.rows + 4000)
    p.check(got, q)
    assert np.all(got[p.rows:] == SENTINEL) and p.flags() == 0
    bad = p.lengths.astype(np.int32)
    bad[chunks[2]] = p.stride * 16 + 1
    cm.lib().gpu_write(p.live[4], cm.ptr(bad), bad.nbytes)
    got = p.attend(q)
    assert p.flags() == 4 and np.all(got[p.starts[chunks[2]]:p.starts[chunks[2] + 1]] == SENTINEL)
    p.check(got, q, skip=[chunks[2]])
    p.free()


@KINDS
@pytest.mark.parametrize("starve", [1, 2])
@pytest.mark.parametrize("news,lengths", [([60], [90]), ([200], [2000]), ([300, 1, 40], [1000, 700, 40])])
def test_waits_that_run_out_are_reported(kind, starve, news, lengths):
    """A first tile that is never ready: every wait behind it runs out after 20 ms, the call comes to its end with
    status 8, and the next one is right."""
    L = cm.lib()
    p = Pool(kind, QWEN, 16, news, lengths, seed=51)
    q, g = p.queries(), L.gpu_open()
    dq, out = upload(q), upload(q)
    try:
        assert L.qwen_b200_wait_limit(20_000_000) == 0
        begin = time.perf_counter()
        assert L.qwen_b200_paged_check(g, out, q.shape[1], dq, q.shape[1], p.cache, p.batch, 12, 0, 0, p.status, starve) == 0
        assert p.flags() == 8
        assert 0.015 <= time.perf_counter() - begin <= 1
        L.gpu_zero(p.status, 4)
        p.check(p.attend(q, gpu=g), q)
        assert p.flags() == 0
    finally:
        assert L.qwen_b200_wait_limit(0) == 0
        for x in (dq, out):
            L.gpu_free(x)
        L.gpu_close(g)
        p.free()


@pytest.mark.parametrize("new", [1, 2, 5, 10])
def test_scores_of_one_sign(new):
    """BF16 rows, queries with full mantissas, all products of one score positive: row 0's score S is a sum of 128
    products in three parts, row 1's one product near it, and no other row counts, so the output tanh((s0 - s1) / 2)
    shows the score. Tensor cores truncate: at most 2^-23 of the sum so far a step, 8 steps of 16 dims, and the sum is
    9/16 of S on average: 4.5. Smaller parts add 2^-8 of that; the factors and the difference round four times, by
    half a unit each, some up and some down: below 6 units of 2^-23 S on average."""
    p = Pool(BF16, QWEN, 16, [new], [new + 2], seed=new)
    d, page = p.dim, p.table[0, 0]
    k = bf16(p.rng.uniform(0.5, 1, (p.kvheads, d)) * 11.0)
    p.host[0][:] = (k ^ 0x8000)[None, :, None]
    p.host[0][page, :, 0] = k
    one = np.zeros((p.kvheads, d), np.float32)
    one[:, 0] = widen(k).sum(1)
    p.host[0][page, :, 1] = bf16(one)
    p.host[1][:] = 0
    p.host[1][page, :, 0], p.host[1][page, :, 1] = 0x3F80, 0xBF80
    p.put()
    q = (1.5 + p.rng.uniform(0, 2.0**-8, (new, p.qheads * d))).astype(np.float32)
    got = p.attend(q).reshape(new, p.qheads, d)
    worst = []
    for h in range(p.qheads):
        kk = widen(p.host[0][page, h // (p.qheads // p.kvheads)]).astype(np.float64)
        s = q.reshape(new, p.qheads, d)[:, h].astype(np.float64) @ kk[:2].T / np.sqrt(d)
        out = np.tanh((s[:, 0] - s[:, 1]) / 2)
        assert np.all(np.abs(s[:, 0] - s[:, 1]) < 3)
        worst.append(np.abs(got[:, h, 0] - out) * 2 / (1 - out**2) / s[:, 0])
    assert np.mean(worst) <= 6 * 2.0**-23, np.mean(worst) * 2**23
    p.free()


@KINDS
@pytest.mark.parametrize("power", [30, 60])
@pytest.mark.parametrize("news,length,places", [(4, 600, [598]), (4, 600, [300, 598]), (2, 700, [0, 699]), (12, 500, [493])])
def test_a_huge_row_late_in_a_warp_s_steps(kind, power, news, length, places):
    """So many sequences that no segment is split: a warp meets the huge row after steps of ordinary ones, whose sums
    it must neither lose nor count as huge."""
    p = Pool(kind, (16, 8, 64), 16, [news] * 40, [length] * 40, seed=power + news)
    for s in range(40):
        for place in places:
            at = (p.table[s, place // 16], slice(None), place % 16)
            if kind == BYTES:
                p.scales[1][at] *= np.float32(2.0**power)
            else:
                p.host[1][at] = np.where(p.host[1][at] & 0x7F80, p.host[1][at] + (power << 7), 0)
    p.put()
    p.values = [p.values(0), p.values(1)].__getitem__  # once, not for each sequence
    q = p.queries()
    check_by_query(p, p.attend(q), q)
    assert p.flags() == 0
    p.free()
