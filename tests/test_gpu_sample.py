"""GPU tests of gpu_sample (include/gpu.h) against float64.

Tokens and counts are exact: the kernel's weights are off by 2^-30 of themselves or 2^-44 of the largest, far less than
the distance of any uniform number here from a border of its row (a token whose border is nearer is none of the
kernel's: the oracle says where that is and the test's inputs have no such row). A log share is a 64-bit value rounded
to FP32, of weights that far off: 2^-24 |x| + 2^-29.
"""
import numpy as np
import pytest

import cmachine_b200 as cm
from test_gpu_paged import download, upload

pytestmark = pytest.mark.gpu

PARAMS = np.dtype([("temperature", "f4"), ("top_k", "i4"), ("top_p", "f4"), ("min_p", "f4")])
OFF = (1.0, 0, 1.0, 0.0)
INF = np.inf
LOW = float(np.finfo(np.float32).min)


def draw(logits, params, uniforms, pad=0, shared=False, rows=None, status=True, partial=False):
    """(ids, kept, logprobs, status bits) of gpu_sample; rows `pad` floats apart with NaN between."""
    L = cm.lib()
    n, vocab = rows or logits.shape[0], logits.shape[1]
    wide = np.full((logits.shape[0], vocab + pad), np.nan, np.float32)
    wide[:, :vocab] = logits
    p = np.array([tuple(x) for x in params], PARAMS)
    up = [upload(wide), upload(p.view(np.int32)), upload(np.asarray(uniforms, np.float32)), upload(np.zeros(1, np.int32)),
          upload(np.full(n + 1, -9, np.int32)), upload(np.full(n + 1, -9, np.int32)), upload(np.full(n + 1, -9, np.float32))]
    g = L.gpu_open()
    assert L.gpu_sample(g, up[4], None if partial else up[6], None if partial else up[5], up[0], 0 if shared else vocab + pad, n, vocab,
                        up[1], up[2], up[3] if status else None) == 0
    ids, kept = (download(up[i], n + 1, np.int32) for i in (4, 5))
    logprobs, bits = download(up[6], n + 1), int(download(up[3], 1, np.int32)[0])
    for x in up:
        L.gpu_free(x)
    L.gpu_close(g)
    assert ids[n] == kept[n] == logprobs[n] == -9
    return ids[:n], kept[:n], logprobs[:n], bits


def exact(l, p, u):
    """(id, kept, logprob, distance of u from the nearest border that decides, as a share of the whole)."""
    t, k, share, least = (float(np.float32(p[0])), int(p[1]), float(np.float32(p[2])), float(np.float32(p[3])))
    if t == 0:
        return int(np.argmax(l)), 1, 0.0, 1.0
    x = l.astype(np.float64)
    with np.errstate(over="ignore"):
        x = (x - x.max()) / t
    order = np.argsort(-l.astype(np.float64), kind="stable")[:int((l > -INF).sum())]
    if k > 0:
        order = order[:k]
    w, room = np.exp(x[order]), 1.0
    n = len(order)
    if share < 1:
        c = np.cumsum(w)
        edge = c[-1] * share
        n = max(1, int(np.searchsorted(c, edge)) + 1)
        room = min(room, np.abs(c - edge).min() / c[-1])
        n = min(n, len(order))
    if least > 0:
        n = min(n, int((x[order] >= np.log(least)).sum()))
    order = np.sort(order[:n])
    c = np.cumsum(np.exp(x[order]))
    edge = float(np.float32(u)) * c[-1]
    at = min(len(c) - 1, int(np.searchsorted(c, edge, side="right")))
    if edge:
        room = min(room, np.abs(c - edge).min() / c[-1])
    return int(order[at]), len(order), float(x[order[at]] - np.log(c[-1])), room


def check(logits, params, uniforms, **kw):
    ids, kept, logprobs, bits = draw(logits, params, uniforms, **kw)
    assert bits == 0
    for r in range(len(uniforms)):
        i, n, lp, room = exact(logits[0 if kw.get("shared") else r], params[r], uniforms[r])
        # Ties of whole numbers are borders that both sides form exactly.
        assert room == 0 or room > 2.0**-40, "a border of the test's own making"
        assert (ids[r], kept[r]) == (i, n), (r, params[r], uniforms[r])
        assert abs(logprobs[r] - lp) <= 2.0**-24 * abs(lp) + 2.0**-29, (r, logprobs[r], lp)


def logits_of(rng, rows, vocab, spread=2.5, coarse=False):
    x = (rng.standard_normal((rows, vocab)) * spread).astype(np.float32)
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 4
    if coarse:
        x = np.round(x * 8) / 8
    return x.astype(np.float32)


SETTINGS = [OFF, (0.7, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 1000, 1.0, 0.0), (1.5, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (0.9, 3, 0.5, 0.3),
            (1.0, 1, 1.0, 0.0), (2.0, 0, 0.999, 0.0), (0.05, 0, 0.99, 0.0), (50.0, 0, 0.5, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0),
            (1.0, 2**31 - 1, 0.3, 0.0), (1.0, -5, 2.0, -1.0), (0.8, 500, 0.9, 0.001)]


@pytest.mark.parametrize("coarse", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 32, 33, 1023, 1025, 2048, 5000, 50257, 151936])
def test_tokens_match_float64(vocab, coarse):
    rng = np.random.default_rng(vocab + coarse)
    rows = len(SETTINGS) * (1 if vocab > 10000 else 3)
    logits = logits_of(rng, rows, vocab, coarse=coarse)
    check(logits, [SETTINGS[r % len(SETTINGS)] for r in range(rows)], rng.random(rows).astype(np.float32), pad=int(rng.integers(0, 4)))


def test_the_largest_vocabulary():
    rng = np.random.default_rng(1)
    logits = logits_of(rng, 6, 524288)
    check(logits, [SETTINGS[r] for r in (0, 1, 2, 4, 8, 15)], rng.random(6).astype(np.float32), pad=1)


@pytest.mark.parametrize("rows", [1, 7, 300])
def test_batches(rows):
    rng = np.random.default_rng(rows)
    check(logits_of(rng, rows, 30000), [SETTINGS[(r * 5) % len(SETTINGS)] for r in range(rows)], rng.random(rows).astype(np.float32))


def test_masked_tokens():
    """Minus infinity, and FP32's lowest number, in most places; one token left; the first and last of the row."""
    rng = np.random.default_rng(3)
    vocab = 40000
    for fill in (-INF, LOW, -1e9):
        logits = np.full((8, vocab), fill, np.float32)
        for r in range(8):
            at = rng.choice(vocab, [1, 2, 5, 40, 700, 3, 1, 20][r], replace=False)
            logits[r, at] = rng.standard_normal(len(at)) * 2
        logits[5, [0, vocab - 1]] = 1.0
        for s in ((1.0, 0, 1.0, 0.0), (0.8, 0, 0.9, 0.0), (1.0, 30, 0.95, 0.01), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.2)):
            check(logits, [s] * 8, rng.random(8).astype(np.float32))


def test_equal_logits():
    """All equal: every border is a border between equal tokens, which go to the lower id."""
    for vocab in (1, 5, 64, 4096, 100000):
        logits = np.full((6, vocab), -3.25, np.float32)
        check(logits, [OFF, (1.0, 17, 1.0, 0.0), (0.3, 0, 0.3, 0.0), (1.0, 40, 0.6, 0.0), (1.0, 0, 0.7, 0.9), (0.0, 0, 1.0, 0.0)],
              np.array([0.3, 0.9, 0.77, 0.1, 0.55, 0.5], np.float32))
    # Two sizes only: the cut falls among one of them.
    logits = np.zeros((4, 9000), np.float32)
    logits[:, ::3] = 1.0
    check(logits, [(1.0, 10, 1.0, 0.0), (1.0, 3500, 1.0, 0.0), (1.0, 0, 0.33, 0.0), (1.0, 3500, 0.93, 0.0)],
          np.array([0.31, 0.97, 0.99, 0.96], np.float32))


@pytest.mark.parametrize("scale", [1e38, 1e30, 1e-30, 1e-38, 1e-42])
def test_logits_of_any_size(scale):
    """Spreads that leave FP32's range, and that are subnormal numbers; temperatures to match."""
    rng = np.random.default_rng(4)
    logits = np.clip(rng.standard_normal((6, 20000)), -3, 3).astype(np.float64) * scale
    logits = logits.astype(np.float32)
    t = float(np.float32(scale))
    if t:
        check(logits, [(t, 0, 1.0, 0.0), (t, 100, 1.0, 0.0), (t, 0, 0.8, 0.0), (1.0, 50, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (t, 0, 1.0, 0.1)],
              rng.random(6).astype(np.float32))


@pytest.mark.parametrize("vocab", [700, 30000, 151936, 400000])
def test_ranges_of_every_width(vocab):
    """Rows that are narrow and wide against their temperature, far from zero, with tokens masked by large numbers."""
    rng = np.random.default_rng(vocab)
    rows = []
    for t in (1.0, 0.6):
        for spread, at in ((0.02, 0), (0.3, -40), (1.5, 15), (6.0, 0), (9.0, 300), (30.0, 0), (2.0, 3900), (2.0, 5000), (2.0, -60000)):
            x = (rng.standard_normal(vocab) * spread + at).astype(np.float32)
            for fill in (None, -1e4, -3000.0, LOW):
                y = x.copy()
                if fill is not None:
                    y[rng.random(vocab) < 0.4] = fill
                rows.append((y, t))
    settings = [(0, 0.9), (50, 1.0), (0, 0.5), (5000, 0.97)]
    for i in range(0, len(rows), 36):
        part = rows[i:i + 36]
        check(np.stack([x for x, _ in part]), [(t, *settings[(i + j + j // 4) % 4], 0.0) for j, (_, t) in enumerate(part)],
              rng.random(len(part)).astype(np.float32), pad=i % 4)


@pytest.mark.parametrize("value", [0.0, 5.0, -4096.0, 1e10, -1e30, 3e38])
def test_one_value_of_any_size(value):
    logits = np.full((4, 5000), value, np.float32)
    check(logits, [(1.0, 0, 0.9, 0.0), (1e-3, 100, 1.0, 0.0), (1e30, 100, 0.3, 0.0), (1e-38, 0, 0.7, 0.5)], np.array([0.3, 0.9, 0.77, 0.1], np.float32))


def test_logits_that_halve():
    """Values that fall by powers of two: each pass over the range cuts off the few largest."""
    x = (2.0 ** -np.arange(240)).astype(np.float32) * np.float32(2.0**100)
    logits = np.concatenate([x, -x, [0.0]])[None].repeat(4, 0).astype(np.float32)
    rng = np.random.default_rng(5)
    logits = logits[:, rng.permutation(logits.shape[1])]
    check(logits, [(2.0**100, 0, 0.9, 0.0), (2.0**100, 300, 1.0, 0.0), (2.0**100, 240, 0.99, 0.0), (1.0, 200, 1.0, 0.0)],
          np.array([0.2, 0.6, 0.9, 0.4], np.float32))


def test_ends_of_the_uniform_range():
    rng = np.random.default_rng(6)
    logits = logits_of(rng, 4, 3000)
    last = np.float32(1 - 2.0**-24)
    ids, kept, _, bits = draw(logits, [OFF, OFF, (1.0, 20, 1.0, 0.0), (1.0, 20, 1.0, 0.0)], np.array([0, last, 0, last], np.float32))
    assert bits == 0
    top = [np.sort(np.argsort(-logits[r], kind="stable")[:20]) for r in (2, 3)]
    assert ids[0] == 0 and ids[1] >= 2990 and ids[2] == top[0][0] and ids[3] == top[1][-1] and kept.tolist() == [3000, 3000, 20, 20]
    # Small uniforms as subnormal numbers.
    assert draw(logits[:1], [OFF], np.array([1e-44], np.float32))[0][0] == 0


def test_one_row_for_all_draws():
    """Stride 0: draws at even distances over one row of logits have every token as often as its weight says, one more or less."""
    rng = np.random.default_rng(7)
    logits, n = logits_of(rng, 1, 700), 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    for s in (OFF, (0.8, 100, 0.9, 0.01)):
        ids, kept, _, bits = draw(logits, [s] * n, u, shared=True, rows=n)
        assert bits == 0 and len(set(kept.tolist())) == 1
        x = logits[0].astype(np.float64) / s[0]
        keep = np.argsort(-logits[0], kind="stable")[:int(kept[0])]
        w = np.zeros(700)
        w[keep] = np.exp(x[keep] - x.max())
        assert np.all(np.abs(np.bincount(ids, minlength=700) - n * w / w.sum()) <= 1.001)
        assert np.all(np.diff(ids) >= 0)


def test_rows_without_a_token_are_reported():
    rng = np.random.default_rng(8)
    logits = logits_of(rng, 12, 5000)
    logits[1, 4321] = np.nan
    logits[2, 17] = INF
    logits[3] = -INF
    p = [OFF] * 12
    p[4], p[5], p[6], p[7], p[8] = (-1.0, 0, 1, 0), (np.nan, 0, 1, 0), (INF, 0, 1, 0), (1.0, 0, np.nan, 0), (1.0, 0, 1.0, 1.5)
    u = rng.random(12).astype(np.float32)
    u[9], u[10] = 1.0, np.nan
    ids, kept, logprobs, bits = draw(logits, p, u)
    assert bits == 7
    for r in range(1, 11):
        assert (ids[r], kept[r], logprobs[r]) == (-1, 0, 0), r
    for r in (0, 11):
        assert (ids[r], kept[r]) == exact(logits[r], OFF, u[r])[:2]
    for row, bit in ((1, 1), (2, 1), (3, 2), (4, 4), (8, 4), (9, 4)):
        assert draw(logits[row:row + 1], [p[row]], u[row:row + 1])[3] == bit
    assert draw(logits, p, u, status=False)[0].tolist() == ids.tolist()
    assert draw(logits, p, u, partial=True)[0].tolist() == ids.tolist()
    # Greedy rows report the same.
    assert draw(logits[1:4], [(0.0, 0, 1.0, 0.0)] * 3, [0.1] * 3)[0].tolist() == [-1, -1, -1]


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(9)
    logits, u = logits_of(rng, 40, 151936, coarse=True), rng.random(40).astype(np.float32)
    p = [SETTINGS[r % len(SETTINGS)] for r in range(40)]
    a = draw(logits, p, u)
    for _ in range(2):
        b = draw(logits, p, u, pad=3)
        assert all(np.array_equal(x, y) for x, y in zip(a[:3], b[:3]))


def test_greedy_agrees_with_top2():
    L = cm.lib()
    rng = np.random.default_rng(10)
    logits = logits_of(rng, 1, 151936, coarse=True)
    g, d = L.gpu_open(), upload(logits)
    top = L.gpu_top2(g, d, 151936)
    assert draw(logits, [(0.0, 0, 1.0, 0.0)], [0.9])[0][0] == top.first
    L.gpu_free(d)
    L.gpu_close(g)
