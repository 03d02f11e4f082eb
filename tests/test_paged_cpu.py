"""The paged K/V cache without a GPU: the index arithmetic its kernels share
(csrc/paged_index.h, built for the host) against plain Python, and the calls
that the entry points refuse before they launch anything."""
import ctypes
from ctypes import POINTER, c_int, c_int64, c_void_p
from pathlib import Path

import numpy as np
import pytest

import cmachine_b200 as cm

ROOT = Path(__file__).resolve().parent.parent


def index_lib():
    L = ctypes.CDLL(str(ROOT / "oracle" / "libpaged_cpu.so"))
    L.paged_cpu_slot.restype = c_int64
    L.paged_cpu_slot.argtypes = [c_int, c_int, c_int, POINTER(c_int), c_int, c_int, c_int, c_int]
    return L


def test_division_by_the_page_size():
    L = index_lib()
    rng = np.random.default_rng(1)
    top = 2**31 - 1
    for page in [*range(1, 70), 100, 127, 128, 129, 255, 256, 257, 1000, 4095, 4096, 65535, 65536]:
        xs = {0, 1, page - 1, page, page + 1, top, top - 1, top // page * page, top // page * page - 1}
        xs |= {int(x) for x in rng.integers(0, top, 60)} | {int(k) * page - 1 for k in rng.integers(1, top // page + 1, 20)}
        for x in xs:
            assert L.paged_cpu_div(page, x) == x // page, (page, x)


def test_extents_that_do_not_fit_leave_no_rows():
    L = index_lib()
    out = (c_int * 3)()
    rows, max_new, max_length, stride, page = 40, 16, 100, 5, 16

    def extent(start, end, length):
        return L.paged_cpu_extent(rows, max_new, max_length, stride, page, start, end, length, out), tuple(out)

    assert extent(0, 16, 16) == (0, (0, 16, 16))
    assert extent(40, 40, 0) == (0, (40, 0, 0))
    assert extent(24, 40, 3) == (0, (24, 16, 3))  # more rows than the sequence has: places below zero
    assert extent(5, 9, 80) == (0, (5, 4, 80))  # the table's last row
    for bad in [(-1, 3, 5), (4, 3, 5), (30, 41, 50), (0, 17, 20), (0, 4, -1), (0, 4, 81), (0, 4, 101),
                (-2**31, 2**31 - 1, 5), (0, 1, 2**31 - 1)]:
        assert extent(*bad) == (4, (0, 0, 0)), bad


def test_rows_stay_inside_the_pool():
    L = index_lib()
    rng = np.random.default_rng(2)
    for page in (1, 3, 16, 24, 100):
        pages, heads, stride = 7, 3, 4
        table = rng.permutation(np.array([0, 1, 2, 3, 4, 5, 6, 7, -1, -2**31, 2**31 - 1, 5], np.int32))
        t = (c_int * 12)(*[int(x) for x in table])
        seen = {}
        for s in range(3):
            for j in range(stride * page):
                for h in range(heads):
                    got = L.paged_cpu_slot(pages, page, heads, t, stride, s, j, h)
                    page_id = int(table[s * stride + j // page])
                    if 0 <= page_id < pages:
                        assert got == (page_id * heads + h) * page + j % page
                        assert 0 <= got < pages * heads * page
                        seen.setdefault((page_id, j % page, h), got)
                    else:
                        assert got == -1
        assert len(set(seen.values())) == len(seen)


def test_row_offsets_pass_32_bits():
    L = index_lib()
    table = (c_int * 2)(2**20, 2**20 + 5)
    assert L.paged_cpu_slot(2**20 + 6, 256, 8, table, 2, 0, 300, 7) == ((2**20 + 5) * 8 + 7) * 256 + 44
    assert L.paged_cpu_slot(2**20 + 5, 256, 8, table, 2, 0, 300, 7) == -1


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 5), (1, 0), (1, 1), (7, 0), (7, 3), (7, 40), (16, 16), (33, 4), (200, 4),
                                          (2**31 - 1, 0), (1, 2**31 - 1), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("shift", [0, 2, 4, 7])
def test_tiles_cover_what_the_queries_see(window, sinks, shift):
    """Every tile that holds a visible row is listed once, in order, and no tile
    lies behind the last query."""
    L = index_lib()
    most = 200
    out = (c_int * most)()
    for first in (-9, -1, 0, 1, 5, 16, 31, 77, 150):
        for count in (1, 2, 17, 40):
            last = first + count - 1
            n = L.paged_cpu_tiles(first, last, window, sinks, shift, out, most)
            tiles = list(out[:n])
            assert n <= most and tiles == sorted(set(tiles))
            need = set()
            for at in range(max(first, 0), last + 1):
                for j in range(at + 1):
                    sees = window == 0 or j > at - window or j < sinks
                    assert bool(L.paged_cpu_sees(at, j, window, sinks)) == sees
                    if sees:
                        need.add(j >> shift)
                assert not L.paged_cpu_sees(at, at + 1, window, sinks)
            assert need <= set(tiles)
            assert all(0 <= t <= max(last, 0) >> shift for t in tiles)
            if shift == 0 and count == 1:
                assert need == set(tiles)


# ---------------------------------------------------------------- refusals
def good():
    """Descriptors that pass every check; their addresses are never followed here."""
    a = 1 << 20
    cache = cm.PagedCache(3, 8, 16, 2, 128, a, a, a)
    batch = cm.PagedBatch(2, 4, 4, 64, a, a, a, 4)
    return cache, batch, a


def calls(cache, batch, a, qheads=12, window=0, sinks=0, stride=12 * 128, q=None, out=None, gpu=1 << 20):
    L = cm.lib()
    return [L.gpu_paged_append(cache, batch, q or a, a, stride, None), L.gpu_paged_read(cache, batch, out or a, a, stride, None),
            L.gpu_paged_attention(gpu, out or a, stride, q or a, stride, cache, batch, qheads, window, sinks, None)]


@pytest.mark.parametrize("field,value", [
    ("kind", 1), ("kind", 0), ("kind", 4), ("pages", 0), ("pages", -1), ("page", 0), ("page", 65537), ("page", -16),
    ("kvheads", 0), ("kvheads", 1025), ("dim", 32), ("dim", 96), ("dim", 256), ("dim", 0), ("keys", None), ("values", None),
    ("keys", (1 << 20) + 8), ("values", (1 << 20) + 2), ("scales", None), ("scales", (1 << 20) + 2)])
def test_bad_caches_are_refused(field, value, capfd):
    cache, batch, a = good()
    setattr(cache, field, value)
    assert calls(cache, batch, a) == [-1, -1, -1]
    assert capfd.readouterr().err.count("gpu_paged_") == 3


@pytest.mark.parametrize("field,value", [
    ("sequences", -1), ("sequences", 65536), ("rows", -1), ("max_new", -1), ("max_length", -1), ("max_length", (1 << 30) + 1), ("starts", None),
    ("lengths", None), ("table", None), ("table_stride", 0), ("starts", (1 << 20) + 2), ("table", (1 << 20) + 1)])
def test_bad_batches_are_refused(field, value):
    cache, batch, a = good()
    setattr(batch, field, value)
    assert calls(cache, batch, a) == [-1, -1, -1]


def test_bad_row_buffers_are_refused():
    cache, batch, a = good()
    assert calls(cache, batch, a, stride=127) == [-1, -1, -1]
    assert calls(cache, batch, a, stride=12 * 128 + 2) == [-1, -1, -1]
    assert calls(cache, batch, a, stride=-1536) == [-1, -1, -1]
    assert cm.lib().gpu_paged_attention(a, a, 512, a, 1536, cache, batch, 12, 0, 0, None) == -1  # not the query heads
    assert calls(cache, batch, a, q=a + 4, out=a + 8) == [-1, -1, -1]
    batch.rows = batch.max_new = 2**31 - 1
    assert calls(cache, batch, a) == [-1, -1, -1]


def test_bad_heads_and_masks_are_refused():
    cache, batch, a = good()
    L = cm.lib()
    for kw in ({"qheads": 0}, {"qheads": 3}, {"qheads": 18}, {"qheads": -2}, {"window": -1}, {"sinks": -1}, {"gpu": None}):
        kw = {"qheads": 12, "window": 0, "sinks": 0, "gpu": 1 << 20, **kw}
        assert L.gpu_paged_attention(kw["gpu"], a, 18 * 128, a, 18 * 128, cache, batch, kw["qheads"], kw["window"],
                                     kw["sinks"], None) == -1, kw
    assert L.gpu_paged_append(None, batch, a, a, 1536, None) == -1
    assert L.gpu_paged_read(cache, None, a, a, 1536, None) == -1


@pytest.mark.parametrize("field", ["sequences", "rows", "max_new"])
def test_an_empty_batch_launches_nothing(field):
    cache, batch, a = good()
    setattr(batch, field, 0)
    assert calls(cache, batch, a) == [0, 0, 0]
