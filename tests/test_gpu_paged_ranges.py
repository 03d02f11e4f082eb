"""GPU tests of the paged K/V cache at the ends of its ranges: batches of several launches, values of unlike
size, long sums, small queries, loose maxima. The pool, its float64 oracle and its bound are
tests/test_gpu_paged.py's unless a test states its own."""
import numpy as np
import pytest

import cmachine_b200 as cm
from test_gpu_paged import KINDS, MHA64, Pool

pytestmark = pytest.mark.gpu


@KINDS
def test_many_launches_beside_chunks_give_the_same_bits(kind):
    """Chunks, and so many short sequences that the decode kernel takes four launches beside them: every launch
    leaves its counters and partials to the next. Long and short sequences alternate, so row tiles are cut."""
    rng = np.random.default_rng(7)
    news = np.where(np.arange(400) % 50 == 7, 70, rng.integers(0, 3, 400))
    lengths = np.maximum(news, np.where(np.arange(400) % 9 == 0, 900, rng.integers(0, 60, 400)))
    p = Pool(kind, MHA64, 16, news, lengths, seed=8)
    q, g = p.queries(), cm.lib().gpu_open()
    first = p.attend(q, gpu=g)
    p.check(first, q)
    for _ in range(30):
        assert np.array_equal(p.attend(q, gpu=g), first)
    assert p.flags() == 0
    cm.lib().gpu_close(g)
    p.free()
