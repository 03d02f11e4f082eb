"""The serving step's operators without a GPU: the calls that their entry points refuse before they launch anything."""
import pytest

import cmachine_b200 as cm

A = 1 << 20  # an address that is never followed here
INF, NAN = float("inf"), float("nan")


def good(kind=3):
    cache = cm.PagedCache(kind, 8, 16, 2, 128, A, A, A)
    batch = cm.PagedBatch(2, 4, 4, 64, A, A, A, 4)
    return cache, batch


def rotate(cache, batch, turn=None, q_out=A, out_stride=1536, q=A, k=A, v=A, stride=1536, qheads=12, status=None, **turned):
    t = {"qnorm": A, "knorm": A, "eps": 1e-6, "theta": 1e6, "rotary": 128, **turned}
    turn = cm.HeadRotation(**t) if turn is None else turn
    return cm.lib().gpu_paged_rotate_append(cache, batch, turn, q_out, out_stride, q, k, v, stride, qheads, status)


def sparse(cache, batch, gpu=A, out=A, out_stride=1536, q=A, q_stride=1536, bounds=A, qheads=12, blocks=8, first=1, recent=2,
           selected=None, status=None):
    return cm.lib().gpu_paged_sparse_attention(gpu, out, out_stride, q, q_stride, cache, batch, bounds, qheads, blocks, first,
                                               recent, selected, status)


def bounds(cache, batch, bounds=A, status=None):
    return cm.lib().gpu_paged_bounds(cache, batch, bounds, status)


def sample(gpu=A, ids=A, logprobs=A, kept=A, logits=A, stride=100, rows=2, vocab=100, params=A, uniforms=A, status=None):
    return cm.lib().gpu_sample(gpu, ids, logprobs, kept, logits, stride, rows, vocab, params, uniforms, status)


@pytest.mark.parametrize("field,value", [
    ("kind", 1), ("pages", 0), ("page", 0), ("page", 65537), ("kvheads", 0), ("kvheads", 1025), ("dim", 96), ("keys", None),
    ("values", A + 8), ("scales", None), ("scales", A + 2)])
def test_bad_caches_are_refused(field, value, capfd):
    cache, batch = good()
    setattr(cache, field, value)
    assert [rotate(cache, batch), bounds(cache, batch), sparse(cache, batch)] == [-1, -1, -1]
    err = capfd.readouterr().err
    assert all(name in err for name in ("gpu_paged_rotate_append:", "gpu_paged_bounds:", "gpu_paged_sparse_attention:"))


@pytest.mark.parametrize("field,value", [
    ("sequences", -1), ("sequences", 65536), ("rows", -1), ("max_new", -1), ("max_length", -1), ("max_length", (1 << 30) + 1),
    ("starts", None), ("lengths", None), ("table", None), ("table_stride", 0), ("starts", A + 2), ("table", A + 1)])
def test_bad_batches_are_refused(field, value):
    cache, batch = good()
    setattr(batch, field, value)
    assert [rotate(cache, batch), bounds(cache, batch), sparse(cache, batch)] == [-1, -1, -1]


@pytest.mark.parametrize("field", ["sequences", "rows", "max_new"])
def test_an_empty_batch_launches_nothing(field):
    cache, batch = good()
    setattr(batch, field, 0)
    assert [rotate(cache, batch), bounds(cache, batch), sparse(cache, batch)] == [0, 0, 0]


@pytest.mark.parametrize("kw", [
    {"rotary": 130}, {"rotary": -4}, {"rotary": 6}, {"rotary": 132}, {"eps": -1e-6}, {"eps": NAN}, {"eps": INF}, {"theta": 0.0},
    {"theta": -1.0}, {"theta": NAN}, {"theta": INF}, {"qnorm": A + 4}, {"knorm": A + 2}, {"qheads": 0}, {"qheads": 3}, {"qheads": 18},
    {"qheads": -2}, {"stride": 1534}, {"stride": 127}, {"stride": -1536}, {"out_stride": 1532}, {"out_stride": 512}, {"q": A + 4},
    {"k": A + 8}, {"v": None}, {"q_out": None}, {"q_out": A + 4}, {"status": A + 2},
    {"out_stride": 1540}])  # q_out is q: with another stride it would meet rows that are still to be read
def test_bad_rotations_are_refused(kw):
    assert rotate(*good(), **kw) == -1


def test_a_missing_rotation_is_refused():
    cache, batch = good()
    assert cm.lib().gpu_paged_rotate_append(cache, batch, None, A, 1536, A, A, A, 1536, 12, None) == -1
    assert cm.lib().gpu_paged_rotate_append(None, batch, cm.HeadRotation(), A, 1536, A, A, A, 1536, 12, None) == -1


@pytest.mark.parametrize("kw", [{"bounds": None}, {"bounds": A + 8}, {"status": A + 1}])
def test_bad_bounds_are_refused(kw):
    assert bounds(*good(), **kw) == -1
    assert sparse(*good(), **kw) == -1


@pytest.mark.parametrize("kw", [
    {"gpu": None}, {"qheads": 0}, {"qheads": 3}, {"qheads": 18}, {"blocks": 0}, {"blocks": 2}, {"blocks": 8193}, {"blocks": -1},
    {"first": -1}, {"recent": 0}, {"recent": -1}, {"first": 2**31 - 1, "recent": 2**31 - 1}, {"selected": A + 2}, {"q": A + 4},
    {"out": None}, {"out_stride": 1532}, {"q_stride": 1530}])
def test_bad_choices_are_refused(kw):
    assert sparse(*good(), **kw) == -1


@pytest.mark.parametrize("kw", [
    {"gpu": None}, {"ids": None}, {"logits": None}, {"params": None}, {"uniforms": None}, {"rows": -1}, {"rows": (1 << 24) + 1},
    {"vocab": 0}, {"vocab": -1}, {"vocab": 524289, "stride": 524289}, {"stride": 99}, {"stride": -100}, {"ids": A + 2},
    {"logits": A + 1}, {"params": A + 2}, {"uniforms": A + 3}, {"logprobs": A + 2}, {"kept": A + 1}, {"status": A + 2}])
def test_bad_samples_are_refused(kw, capfd):
    assert sample(**kw) == -1
    assert "gpu_sample:" in capfd.readouterr().err


def test_no_rows_launch_nothing():
    assert sample(rows=0) == 0
