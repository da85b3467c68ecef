"""paged_attention against the formula in 64 bits, and exactly where the sums are exact."""

import math
from importlib import import_module

import numpy as np
import pytest

import paged_oracle as po
from decode_step_oracle import to_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


TYPES = {"f32": (False, False), "mixed": (False, True), "bf16": (True, True), "wide": (True, False)}  # (queries, cache) in bfloat16


def run(dev, q, cache, lengths, rows, heads, types, window=0, sinks=0, scale=None, max_rows=None, max_keys=None, ldq=None,
        ldo=None, stream=None, workspace=None, pad_rows=0, table=None, fill=7.0, expect_err=0):
    """out [rows, heads, d] of packed queries q [rows, heads, d]; the buffers are wider and longer than the rows."""
    q_bf16, c_bf16 = TYPES[types]
    total, d = len(q), cache.k_cache.shape[3]
    width = heads * d
    ldq, ldo = ldq or width, ldo or width
    qh = np.zeros((total + pad_rows, ldq), np.float32)
    qh[:total, :width] = q.reshape(total, width)
    out = dev.DeviceArray.from_host(np.full((total + pad_rows, ldo), fill, np.float32))
    err = dev.DeviceArray.zeros(1, np.int32)
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    up = dev.DeviceArray.from_host
    dev.paged_attention(up(to_bf16(qh)[0] if q_bf16 else qh), up(cache.k_cache), up(cache.v_cache),
                        up(cache.table if table is None else table), up(np.array(lengths, np.int32)), up(cu), out, heads=heads,
                        max_rows=max_rows or max(max(rows), 1), max_keys=max_keys or max(max(lengths), 1),
                        scale=scale or 1.0 / math.sqrt(d), window=window, sinks=sinks, bf16=q_bf16, cache_bf16=c_bf16,
                        workspace=workspace, err=err, stream=stream)
    dev.synchronize()
    got = out.host()
    assert err.host()[0] == expect_err
    assert (got[total:] == fill).all() and (got[:, width:] == fill).all()  # nothing else is written
    return got[:total, :width].reshape(total, heads, d)


def queries(rng, rows, heads, d, types, size=1.5):
    q = (size * rng.standard_normal((sum(rows), heads, d))).astype(np.float32)
    return to_bf16(q)[1] if TYPES[types][0] else q


def check(got, q, cache, lengths, rows, window=0, sinks=0, scale=None):
    at = 0
    for b, n in enumerate(rows):
        if n:
            want, bound = po.attention(q[at:at + n], cache.k[b], cache.v[b], lengths[b], window, sinks,
                                       scale or 1.0 / math.sqrt(q.shape[2]))
            off = np.abs(got[at:at + n] - want)
            worst = np.unravel_index(np.argmax(off - bound), off.shape)
            assert (off <= bound).all(), (b, worst, got[at:at + n][worst], want[worst], bound[worst])
        at += n


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("heads, kv_heads, d", [(8, 8, 64), (8, 8, 48), (16, 2, 128), (5, 1, 64), (6, 2, 48), (33, 1, 64)])
def test_against_the_formula(dev, types, heads, kv_heads, d):
    rng = np.random.default_rng(heads * d + kv_heads)
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 130, 300]
    rows = [1, 2, 1, 3, 1, 1, 5, 1, 2, 1]
    cache = po.Cache(rng, lengths, kv_heads, d, 16, TYPES[types][1])
    q = queries(rng, rows, heads, d, types)
    check(run(dev, q, cache, lengths, rows, heads, types), q, cache, lengths, rows)


@pytest.mark.parametrize("page", [8, 16, 64, 1024])
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (7, 1), (100, 4), (64, 70), (5000, 3)])
def test_windows_and_sinks(dev, page, window, sinks):
    rng = np.random.default_rng(page + window)
    lengths, rows = [1, 9, 64, 65, 129, 700], [1, 2, 1, 7, 3, 2]
    for types, d in (("f32", 48), ("bf16", 64)):
        cache = po.Cache(rng, lengths, 2, d, page, TYPES[types][1])
        q = queries(rng, rows, 4, d, types)
        got = run(dev, q, cache, lengths, rows, 4, types, window=window, sinks=sinks)
        check(got, q, cache, lengths, rows, window, sinks)


def mean_of_visible(cache, lengths, rows, heads, window=0, sinks=0):
    """Zero queries: every visible key weighs 1, whole values add up exactly, and one division rounds."""
    out = []
    for b, n in enumerate(rows):
        for i in range(n):
            see = po.visible(lengths[b], n, i, window, sinks)
            total = cache.v[b][see].astype(np.float64).sum(axis=0)
            mean = (total / max(len(see), 1)).astype(np.float32)
            out.append(np.repeat(mean, heads // mean.shape[0], axis=0))
    return np.array(out)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("lengths, rows, heads, kv_heads, d, page, window, sinks", [
    ([5000], [1], 8, 8, 64, 16, 0, 0),
    ([70001], [1], 2, 1, 128, 32, 0, 0),
    ([4097, 1, 100, 2048], [4, 1, 9, 2], 4, 2, 48, 8, 0, 0),
    ([9000, 31, 4000], [3, 1, 2], 8, 1, 64, 16, 1000, 5),
    ([20000, 3], [1, 2], 4, 4, 64, 256, 4097, 64),
    ([300, 64, 77], [64, 64, 33], 8, 2, 64, 16, 0, 0),
    ([1 + b for b in range(200)], [1] * 200, 8, 8, 48, 16, 0, 0),
])
def test_every_visible_key_once(dev, types, lengths, rows, heads, kv_heads, d, page, window, sinks):
    rng = np.random.default_rng(len(lengths) + d)
    cache = po.Cache(rng, lengths, kv_heads, d, page, TYPES[types][1], values="whole")
    q = np.zeros((sum(rows), heads, d), np.float32)
    got = run(dev, q, cache, lengths, rows, heads, types, window=window, sinks=sinks)
    assert np.array_equal(got, mean_of_visible(cache, lengths, rows, heads, window, sinks))


@pytest.mark.parametrize("types", list(TYPES))
def test_rows_before_the_first_key_are_zero(dev, types):
    rng = np.random.default_rng(3)
    lengths, rows = [0, 2, 5], [2, 5, 1]  # positions -2 .. -1, -3 .. 1, 4
    cache = po.Cache(rng, lengths, 2, 64, 16, TYPES[types][1])
    q = queries(rng, rows, 4, 64, types)
    got = run(dev, q, cache, lengths, rows, 4, types)
    assert not got[:5].any()
    check(got, q, cache, lengths, rows)


@pytest.mark.parametrize("types", list(TYPES))
def test_no_rows_and_padding(dev, types):
    """Requests without rows, rows behind the last request, wide strides, bounds above what there is."""
    rng = np.random.default_rng(4)
    lengths, rows = [40, 0, 33, 18], [0, 0, 2, 1]
    cache = po.Cache(rng, lengths, 2, 48, 16, TYPES[types][1], width=9)
    q = queries(rng, rows, 4, 48, types)
    got = run(dev, q, cache, lengths, rows, 4, types, ldq=4 * 48 + 24, ldo=4 * 48 + 4, pad_rows=3, max_rows=17, max_keys=131072)
    check(got, q, cache, lengths, rows)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("stale", [math.nan, math.inf, -math.inf])
def test_slots_out_of_sight_change_nothing(dev, types, stale):
    """Past a request's last key, and between sinks and window, the cache holds NaN and infinities; tables name no
    page where nothing is seen."""
    rng = np.random.default_rng(5)
    lengths, rows, window, sinks = [70, 33, 900], [1, 4, 3], 40, 3
    cache = po.Cache(rng, lengths, 2, 64, 16, TYPES[types][1], stale=stale)
    table = cache.table.copy()
    bad = np.uint16(0x7FC0) if TYPES[types][1] else np.float32(stale)
    for b, (n, m) in enumerate(zip(lengths, rows)):
        low = n - m - window + 1
        for j in range(sinks, max(sinks, low)):
            page = cache.table[b, j // 16]
            cache.k_cache[page, :, j % 16] = bad
            cache.v_cache[page, :, :, j % 16] = bad
        for j in range(table.shape[1]):
            if j * 16 >= n or (j * 16 >= sinks and (j + 1) * 16 <= low):
                table[b, j] = -1
    q = queries(rng, rows, 4, 64, types)
    got = run(dev, q, cache, lengths, rows, 4, types, window=window, sinks=sinks, table=table)
    check(got, q, cache, lengths, rows, window, sinks)


@pytest.mark.parametrize("types", list(TYPES))
def test_large_scores(dev, types):
    """One key far ahead, all keys far below zero, scores that overflow exp on the way."""
    rng = np.random.default_rng(6)
    lengths, rows = [200, 200, 200], [1, 1, 2]
    cache = po.Cache(rng, lengths, 1, 64, 16, TYPES[types][1])
    q = queries(rng, rows, 2, 64, types, size=30.0)
    check(run(dev, q, cache, lengths, rows, 2, types, scale=0.5), q, cache, lengths, rows, scale=0.5)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("heads, kv_heads, d, rows", [(8, 8, 64, 1), (8, 2, 128, 3), (8, 8, 48, 1), (24, 1, 128, 1)])
def test_workspace_is_as_large_as_it_says(dev, types, heads, kv_heads, d, rows):
    """A call writes nothing past the bytes it asks for (a long cache in shares of all workgroups), and gives what it
    gives with library scratch."""
    rng = np.random.default_rng(d)
    lengths, rows = [9000, 4000, 2], [rows] * 3
    q_bf16, c_bf16 = TYPES[types]
    cache = po.Cache(rng, lengths, kv_heads, d, 16, c_bf16)
    q = queries(rng, rows, heads, d, types)
    need = dev.paged_attention_workspace(3, max(rows), max(lengths), heads, kv_heads, d, bf16=q_bf16, cache_bf16=c_bf16)
    assert need > 0
    whole = dev.DeviceArray.from_host(np.full(need + 4096, 0x5A, np.uint8))

    class Part:
        ptr, nbytes = whole.ptr, need

    got = run(dev, q, cache, lengths, rows, heads, types, workspace=Part)
    after = whole.host()
    assert (after[need:] == 0x5A).all() and (after[:need] != 0x5A).any()
    assert np.array_equal(got, run(dev, q, cache, lengths, rows, heads, types))


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("d, length", [(48, 40), (64, 300), (128, 5000)])
def test_rows_that_do_not_see_infinities_and_nan(dev, types, d, length):
    """NaN and infinities in the last row's key and value, among the tile that the rows before it see a part of: their
    results are the finite ones, and the last row's what the formula makes of them."""
    rng = np.random.default_rng(d)
    q_bf16, c_bf16 = TYPES[types]
    lengths, rows = [length, 33], [3, 1]
    for where, bad in (("v", math.nan), ("v", math.inf), ("k", math.nan), ("k", -math.inf)):
        cache = po.Cache(rng, lengths, 2, d, 16, c_bf16)
        q = queries(rng, rows, 4, d, types)
        j = length - 1
        page, place = cache.table[0, j // 16], j % 16
        value = to_bf16(np.float32([bad]))[0][0] if c_bf16 else np.float32(bad)
        if where == "v":
            cache.v_cache[page, 0, 5, place] = value
        else:
            cache.k_cache[page, 0, place, 5] = value
        got = run(dev, q, cache, lengths, rows, 4, types)
        sees = got[2].copy()
        got[2, :2] = 0  # of the first key head's queries, which see it: below
        part = q.copy()
        want, bound = po.attention(part[:3], cache.k[0], cache.v[0], length, scale=1.0 / math.sqrt(d))
        want[2, :2] = 0
        assert (np.abs(got[:3] - want) <= bound).all(), (where, bad)
        check(got[3:], q[3:], type("C", (), dict(k=cache.k[1:], v=cache.v[1:])), lengths[1:], rows[1:])
        if where == "v":  # one value of the weighted sum
            assert np.isnan(sees[:2, 5]).all() if math.isnan(bad) else (sees[:2, 5] == bad).all()
            others = np.arange(d) != 5
            full, bound = po.attention(part[:3], cache.k[0], cache.v[0], length, scale=1.0 / math.sqrt(d))
            assert (np.abs(sees[:2] - full[2, :2]) <= bound[2, :2])[:, others].all()
        elif math.isnan(bad):
            assert np.isnan(sees[:2]).all()
        else:  # a score of one infinity: all weight on its key (not a number), or none
            for h in range(2):
                if part[2, h, 5] < 0:
                    assert np.isnan(sees[h]).all()
                else:
                    k = cache.k[0].copy()
                    w = np.exp((k[:-1, 0].astype(np.float64) @ part[2, h].astype(np.float64)) / math.sqrt(d))
                    np.testing.assert_allclose(sees[h], (w @ cache.v[0][:-1, 0]) / w.sum(), rtol=0, atol=1e-4)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_queries_that_are_not_numbers(dev, types, bad):
    """A row whose query holds a NaN or an infinity is NaN in that head alone, whatever lies beside it."""
    rng = np.random.default_rng(21)
    lengths, rows = [700, 33], [3, 2]
    cache = po.Cache(rng, lengths, 2, 64, 16, TYPES[types][1])
    q = queries(rng, rows, 4, 64, types)
    wrong = q.copy()
    wrong[1, 2, 7], wrong[3, 0, 63] = bad, bad
    cache.v_cache[cache.table[0, 699 // 16], 1, 3, 699 % 16] = 0x7FC0 if TYPES[types][1] else math.nan  # row 2's own value
    got = run(dev, wrong, cache, lengths, rows, 4, types)
    assert np.isnan(got[1, 2]).all() and np.isnan(got[3, 0]).all() and np.isnan(got[2, 2:, 3]).all()
    for b, at in ((0, 0), (1, 3)):
        want, bound = po.attention(q[at:at + rows[b]], cache.k[b], cache.v[b], lengths[b], scale=1.0 / math.sqrt(64))
        off = np.abs(got[at:at + rows[b]] - want)
        fine = np.isfinite(got[at:at + rows[b]])
        assert (off[fine] <= bound[fine]).all()
    assert np.isnan(got).sum() == 64 + 64 + 2
