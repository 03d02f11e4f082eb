"""How chunks of a paged batch are shared out (csrc/paged_index.h, built for the host): bounds of a batch's row
tiles that the host launches for, the splits taken for what there is; and a call that is refused."""
import ctypes
from ctypes import c_int, c_int64
from pathlib import Path

import numpy as np
import pytest

import cmachine_b200 as cm

ROOT = Path(__file__).resolve().parent.parent
TILE, SMS = 256, 148


def plan_lib():
    L = ctypes.CDLL(str(ROOT / "oracle" / "libpaged_cpu.so"))
    for f in (L.paged_cpu_tile_bound, L.paged_cpu_tile_guess):
        f.restype, f.argtypes = c_int64, [c_int] * 6
    L.paged_cpu_splits.restype, L.paged_cpu_splits.argtypes = c_int, [c_int64, c_int, c_int, c_int64, c_int]
    return L


def live_tiles(news, group, few):
    return sum(-(-n * group // TILE) for n in news if n > few)


def test_the_bound_holds_every_row_tile():
    L = plan_lib()
    rng = np.random.default_rng(1)
    for _ in range(4000):
        group, few = int(rng.integers(1, 9)), int(rng.integers(0, 65))
        count = int(rng.integers(1, 80))
        news = [int(n) for n in np.exp(rng.uniform(0, np.log(rng.integers(2, 5000)), count)).astype(int) - rng.integers(0, 2, count)]
        if rng.random() < 0.3:  # as many tiles for their rows as can be
            news = [few + 1] * count
        loose = int(rng.integers(0, 3)) * int(rng.integers(0, 1000))
        rows, most = sum(news) + loose, min(max(news) + loose, sum(news) + loose)
        bound = L.paged_cpu_tile_bound(count, rows, most, group, few, TILE)
        assert live_tiles(news, group, few) <= bound
        assert (bound >= 1 or most <= few) and L.paged_cpu_tile_guess(count, rows, most, group, few, TILE) <= bound


def test_bounds_of_the_largest_sizes():
    L = plan_lib()
    top = 2**31 - 1
    assert L.paged_cpu_tile_bound(65535, top, top, 8, 0, TILE) == top * 8 // TILE + 65535
    assert L.paged_cpu_tile_bound(65535, top, 1, 8, 0, TILE) == 65535
    assert L.paged_cpu_tile_bound(1, top, top, 1, 0, TILE) == -(-top // TILE)


@pytest.mark.parametrize("tokens", [0, 63, 255])
@pytest.mark.parametrize("loose", [False, True])
def test_a_chunk_is_split_as_far_beside_single_tokens_as_alone(tokens, loose):
    """512 new rows over 4609 (12 query heads, 2 KV heads): 24 items, which fill the SMs when split in six. Single
    tokens beside them, or a caller whose buffers and max_new are far larger than its batch, change nothing, and the
    CTAs launched for the batch leave room for the splits."""
    L = plan_lib()
    kvheads, group, few = 2, 6, 0 if tokens == 0 else 5
    rows, most = (8192, 8192) if loose else (512 + tokens, 512)
    items, tiles = kvheads * live_tiles([512] + [1] * tokens, group, few), 37
    assert items == 24
    guess = kvheads * L.paged_cpu_tile_guess(tokens + 1, rows, most, group, few, TILE)
    bound = kvheads * L.paged_cpu_tile_bound(tokens + 1, rows, most, group, few, TILE)
    grid = max(bound, guess * L.paged_cpu_splits(guess, tiles, SMS, 8 * SMS, 32))
    splits = L.paged_cpu_splits(items, tiles, SMS, min(grid, 8 * SMS), 32)
    assert 5 <= splits <= 6 and items * splits <= SMS
    assert loose or grid <= 2 * SMS  # few CTAs that find nothing to do


def test_splits_are_the_fewest_that_are_nearly_the_best():
    L = plan_lib()
    rng = np.random.default_rng(2)

    def cost(items, k, tiles):
        return -(-items * k // SMS) * (tiles / k + 3) + 2 * (k > 1)

    for _ in range(3000):
        items, tiles = int(np.exp(rng.uniform(0, 8))), int(np.exp(rng.uniform(0, 9)))
        room, most = int(np.exp(rng.uniform(0, 8))), int(rng.integers(1, 33))
        k = L.paged_cpu_splits(items, tiles, SMS, room, most)
        allowed = [1] + [x for x in range(2, most + 1) if 2 * x <= tiles and items * x <= room]
        assert k in allowed
        best = min(cost(items, x, tiles) for x in allowed)
        assert cost(items, k, tiles) <= 1.0301 * best
        assert all(cost(items, x, tiles) > 1.0299 * best for x in allowed if x < k)


def test_a_status_word_out_of_step_is_refused(capfd):
    """The kernels OR into it: an address that is no multiple of four would fault."""
    L, a = cm.lib(), 1 << 20
    cache, batch = cm.PagedCache(3, 8, 16, 2, 128, a, a, a), cm.PagedBatch(2, 4, 4, 64, a, a, a, 4)
    for off in (1, 2, 3):
        assert L.gpu_paged_append(cache, batch, a, a, 256, a + off) == -1
        assert L.gpu_paged_read(cache, batch, a, a, 256, a + off) == -1
        assert L.gpu_paged_attention(a, a, 1536, a, 1536, cache, batch, 12, 0, 0, a + off) == -1
        assert L.qwen_b200_paged_check(a, a, 1536, a, 1536, cache, batch, 12, 0, 0, a + off, 0) == -1
    assert L.qwen_b200_paged_check(a, a, 1536, a, 1536, cache, batch, 12, 0, 0, None, 3) == -1
    assert capfd.readouterr().err.count("status is 4-byte aligned") == 12
