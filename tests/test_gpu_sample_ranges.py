"""GPU tests of gpu_sample on rows whose logits lie on both sides of the least that the first pass counts, 4096 temperatures
below zero (csrc/sample_bins.h); tests/test_sample_cpu.py counts such rows on the host. Tolerances are test_gpu_sample.py's."""
import numpy as np
import pytest

from test_gpu_sample import check

pytestmark = pytest.mark.gpu

# (top_k, top_p, min_p): lists that hold a whole top-k, cuts among thousands, and sums.
CUTS = [(5, 1.0, 0.0), (2000, 1.0, 0.0), (2500, 1.0, 0.0), (40, 0.9, 0.0), (2500, 0.95, 0.0), (0, 0.9, 0.0), (0, 0.999, 0.01), (1, 1.0, 0.0)]
TEMPERATURES = [1.0, 0.01, 37.5, 2.0**-20, 2.0**20]


def floor_of(t):
    return np.float32(-4096.0 * t)


@pytest.mark.parametrize("vocab", [4000, 100010, 400000])
@pytest.mark.parametrize("t", TEMPERATURES)
def test_few_logits_next_above_the_floor(t, vocab):
    """Ten logits next above it, all others at it."""
    rng = np.random.default_rng(1)
    row = np.full(vocab, floor_of(t), np.float32)
    row[rng.choice(vocab, 10, replace=False)] = np.nextafter(floor_of(t), np.float32(0))
    n = len(CUTS)
    check(np.tile(row, (n, 1)), [(t, *c) for c in CUTS], rng.random(n).astype(np.float32), pad=1)


@pytest.mark.parametrize("rows", [1, 3, 12])
@pytest.mark.parametrize("t", TEMPERATURES)
def test_thousands_of_logits_on_both_sides(t, rows):
    """The largest logit 0 to 40 temperatures above the floor, so that the floor lies in the bins or next below them; rows
    in one call and in many, so that a row has up to 16 CTAs."""
    rng = np.random.default_rng(rows)
    logits, settings = [], []
    for above in (1e-3, 0.5, 6.0, 14.0, 31.5, 32.0, 33.0, 40.0):
        for low in (0.0, 1e-3, 14.0, 3000.0):
            x = np.concatenate([above * rng.random(3000), -low * rng.random(3000)])
            x[0] = above
            x[2900:3100] = 0
            logits.append((-4096.0 * t + t * x).astype(np.float32)[rng.permutation(6000)])
            settings.append((t, *CUTS[len(settings) % len(CUTS)]))
            logits.append(logits[-1])
            settings.append((t, *CUTS[(len(settings) + 3) % len(CUTS)]))
    for i in range(0, len(logits), rows):
        part = slice(i, i + rows)
        check(np.stack(logits[part]), settings[part], rng.random(len(settings[part])).astype(np.float32), pad=i % 4)


def test_many_rows_of_one_cta():
    rng = np.random.default_rng(3)
    logits, settings = [], []
    for r in range(330):
        t = TEMPERATURES[r % len(TEMPERATURES)]
        x = np.concatenate([rng.uniform(0, 35) * rng.random(2500), -20 * rng.random(2500)])
        logits.append((-4096.0 * t + t * x).astype(np.float32))
        settings.append((t, *CUTS[r % len(CUTS)]))
    check(np.stack(logits), settings, rng.random(330).astype(np.float32))
