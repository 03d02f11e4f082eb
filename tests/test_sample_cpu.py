"""The bins in which the sampling counts a row's logits (csrc/sample_bins.h, built for the host), without a GPU: where the
counts of the first pass are taken, every bin's is the number of tokens that lie in it."""
import ctypes
from ctypes import c_float, c_int, c_void_p
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
BINS, SLOTS, REACH = 4096, 8192, 2.0**19
INF = np.inf


def bins_lib():
    L = ctypes.CDLL(str(ROOT / "oracle" / "libsample_cpu.so"))
    L.sample_cpu_slots.argtypes = [c_void_p, c_int, c_float, c_void_p, c_void_p]
    L.sample_cpu_bins.argtypes = [c_void_p, c_int, c_float, c_float, c_int, c_void_p]
    L.sample_cpu_bins.restype = None
    return L


def counted(L, row, t):
    """(do the slots' counts hold, those counts, the tokens of each bin)."""
    row = np.ascontiguousarray(row, np.float32)
    a, b = np.zeros(BINS, np.int32), np.zeros(BINS, np.int32)
    hold = L.sample_cpu_slots(row.ctypes.data, len(row), t, a.ctypes.data, b.ctypes.data)
    assert hold in (0, 1)
    return bool(hold), a, b


def test_logits_at_the_floor_are_in_the_last_bin():
    """Ten logits next above the least that is counted, and a hundred thousand at it, which are not."""
    L = bins_lib()
    for t in (1.0, 0.01, 37.5, 2.0**-20, 2.0**20):
        floor = np.float32(-REACH / 128 * t)
        row = np.full(100010, floor, np.float32)
        row[:10] = np.nextafter(floor, np.float32(0))
        hold, a, b = counted(L, row, t)
        assert not hold or np.array_equal(a, b), t


@pytest.mark.parametrize("t", [1.0, 0.6, 0.01, 37.5, 1e-6, 1e6, 1e-30, 1e30])
@pytest.mark.parametrize("above", [0.0, 1e-3, 0.1, 1.0, 6.0, 20.0, 31.0, 31.9, 32.0, 32.1, 33.0, 40.0, 64.0, 100.0])
def test_rows_over_the_floor(t, above):
    """The largest logit `above` temperatures above the floor; tokens on both sides of it, and far below."""
    L = bins_lib()
    rng = np.random.default_rng(int(above * 1000))
    floor = -REACH / 128 * t
    for low in (0.0, 0.5, 20.0, 5000.0):
        with np.errstate(over="ignore"):
            row = (floor + t * np.concatenate([above * rng.random(1500), -low * rng.random(1500)])).astype(np.float32)
        row[0] = floor + above * t
        row[1000:1010] = floor
        row = row[np.isfinite(row)]
        hold, a, b = counted(L, row, t)
        assert not hold or np.array_equal(a, b), low
        # Bins of the row's own cost two more passes. They are needed where the floor is less than the 4096 bins, 32
        # temperatures, below the largest, and where what is counted spans the 8192 slots, 64 temperatures.
        assert hold or not 33 <= above < 63


def test_rows_of_every_place_and_width():
    L = bins_lib()
    rng = np.random.default_rng(1)
    held = 0
    for _ in range(1500):
        t = np.float32(2.0 ** rng.uniform(-126, 120))
        with np.errstate(over="ignore"):
            row = (rng.uniform(-1, 1) * 10 ** rng.uniform(-2, 4) * float(t) + rng.standard_normal(800) * 10 ** rng.uniform(-6, 5) * float(t)).astype(np.float32)
        row[rng.random(800) < rng.choice([0, 0.5])] = rng.choice([-INF, -3e38, -1e4, 0.0])
        row = row[np.isfinite(row) | (row == -INF)]
        hold, a, b = counted(L, row, t)
        assert not hold or np.array_equal(a, b), t
        held += hold
    assert held > 300


def test_usual_rows_are_counted_in_one_pass():
    L = bins_lib()
    rng = np.random.default_rng(2)
    for t in (0.05, 0.7, 1.0, 2.0):
        for at in (-60.0, 0.0, 40.0):
            row = (rng.standard_normal(5000) * 3 * min(t, 1.0) + at * t).astype(np.float32)
            hold, a, b = counted(L, row, t)
            assert hold and np.array_equal(a, b) and a[:8].sum() >= 1


@pytest.mark.parametrize("bins", [1024, 4096])
def test_bins_over_a_range_do_not_fall(bins):
    """Every logit has one of the bins, larger ones none that is higher; the least of the range, and what lies below, not the
    last but one's successor unless it lies outside."""
    L = bins_lib()
    rng = np.random.default_rng(3)
    for _ in range(400):
        x = np.sort((rng.standard_normal(300) * 10.0 ** rng.uniform(-44, 38)).astype(np.float64) + rng.choice([0, 1e-3, 50, -1e30]))
        x = np.clip(x, -3.4e38, 3.4e38).astype(np.float32)
        out = np.zeros(300, np.int32)
        for start in (0, 100):
            L.sample_cpu_bins(x.ctypes.data, 300, float(x[start]), float(x[-1]), bins, out.ctypes.data)
            assert out[-1] == 0 and np.all(np.diff(out) <= 0) and out.max() < bins
            assert np.all(out[start:] <= bins - 2)
