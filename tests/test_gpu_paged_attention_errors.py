"""What paged_attention does with requests and pages that cannot be taken: err is set, such requests' rows stay as they
were, keys on pages out of range count as unseen, and the rest of the call is right.  Each on a call whose sequences are a
workgroup's each, and on one that is cut into shares and joined."""

import math
from importlib import import_module

import numpy as np
import pytest

import paged_oracle as po
from decode_step_oracle import to_bf16
from test_gpu_paged_attention import TYPES, queries

pytestmark = pytest.mark.gpu

FILL = 7.0
LONG = {"whole": 200, "split": 9000}  # keys of the longest request, and the call's max_keys


@pytest.fixture(scope="module")
def dev(pkg):
    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


def call(dev, q, cache, lengths, cu, heads, types, max_rows, max_keys, table=None, window=0, sinks=0):
    """(out [rows, heads, d], err) of any cu_rows."""
    q_bf16, c_bf16 = TYPES[types]
    rows, d = len(q), q.shape[2]
    need = dev.paged_attention_workspace(len(lengths), max_rows, max_keys, heads, cache.k_cache.shape[1], d, window, sinks, q_bf16,
                                         c_bf16)
    assert (need > 0) == (max_keys >= 4096)  # else the call is not the one that is meant
    qh = q.reshape(rows, heads * d)
    up = dev.DeviceArray.from_host
    out, err = up(np.full((rows, heads * d), FILL, np.float32)), dev.DeviceArray.zeros(1, np.int32)
    dev.paged_attention(up(to_bf16(qh)[0] if q_bf16 else qh), up(cache.k_cache), up(cache.v_cache),
                        up(cache.table if table is None else table), up(np.array(lengths, np.int32)), up(np.array(cu, np.int32)),
                        out, heads=heads, max_rows=max_rows, max_keys=max_keys, scale=1.0 / math.sqrt(d), window=window,
                        sinks=sinks, bf16=q_bf16, cache_bf16=c_bf16, err=err)
    dev.synchronize()
    return out.host().reshape(rows, heads, d), int(err.host()[0])


def expect(q, k, v, length, keep, window=0, sinks=0):
    """The formula for one request's rows over its visible keys that `keep` [length] names; rows that see none: zeros."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(len(q)):
        see = [j for j in po.visible(length, len(q), i, window, sinks) if keep[j]]
        if see:
            o, b = po.attention(q[i:i + 1], k[see], v[see], len(see), scale=1.0 / math.sqrt(q.shape[2]))
            out[i], bound[i] = o[0], b[0]
    return out, bound


def check(got, q, cache, lengths, cu, good, keep=None, window=0, sinks=0):
    left = np.ones(len(q), bool)
    for b in good:
        at = slice(cu[b], cu[b + 1])
        keys = np.ones(lengths[b], bool) if keep is None else keep[b]
        want, bound = expect(q[at], cache.k[b], cache.v[b], lengths[b], keys, window, sinks)
        assert (np.abs(got[at] - want) <= bound).all(), b
        left[at] = False
    assert (got[left] == FILL).all()  # no request's, or one's that cannot be taken


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("form", list(LONG))
@pytest.mark.parametrize("what", ["max_rows", "max_keys", "table", "negative length", "rows before", "rows behind", "descending"])
def test_requests_that_cannot_be_taken(dev, types, form, what):
    rng = np.random.default_rng(len(what))
    long, heads, kv_heads, d = LONG[form], 4, 2, 64
    lengths, rows = [40, 33, long, 70], [2, 3, 1, 2]
    cache = po.Cache(rng, lengths, kv_heads, d, 16, TYPES[types][1])
    cu, given, bad, max_rows, max_keys = [0, 2, 5, 6, 8], list(lengths), {0}, 3, long
    if what == "max_rows":
        max_rows, bad = 2, {1}
    elif what == "max_keys":
        given[0] = long + 1
        cache.table = np.pad(cache.table, ((0, 0), (0, 1)), constant_values=-1)
    elif what == "table":
        given[0] = max_keys = 16 * cache.table.shape[1] + 1
    elif what == "negative length":
        given[0] = -1
    elif what == "rows before":
        cu[0] = -1
    elif what == "rows behind":
        cu[4], bad = 9, {3}
    else:  # the first has too many rows, the second ends before it begins
        cu, bad = [0, 6, 5, 6, 8], {0, 1}
    q = queries(rng, rows, heads, d, types)
    got, err = call(dev, q, cache, given, cu, heads, types, max_rows, max_keys)
    assert err == 1
    check(got, q, cache, lengths, cu, set(range(4)) - bad)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("form", list(LONG))
@pytest.mark.parametrize("page_no", [-1, -2 ** 31, 2 ** 31 - 1, "pages"])
def test_pages_out_of_range_count_as_unseen(dev, types, form, page_no):
    """One page in the middle of a long sequence, and many next to each other (of whole shares)."""
    rng = np.random.default_rng(31)
    long, heads, kv_heads, d, page = LONG[form], 4, 2, 64, 16
    lengths, cu = [long, 45, 60], [0, 2, 3, 5]
    cache = po.Cache(rng, lengths, kv_heads, d, page, TYPES[types][1])
    q = queries(rng, [2, 1, 2], heads, d, types)
    number = len(cache.k_cache) if page_no == "pages" else page_no
    last = (long - 1) // page
    for bad in ([last // 2], range(last // 4, last // 4 + last // 2), [last]):
        table, keep = cache.table.copy(), [np.ones(n, bool) for n in lengths]
        for j in bad:
            table[0, j] = number
            keep[0][j * page:(j + 1) * page] = False
        got, err = call(dev, q, cache, lengths, cu, heads, types, 2, long, table=table)
        assert err == 1
        check(got, q, cache, lengths, cu, range(3), keep)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("heads, kv_heads, d", [(4, 2, 64), (33, 1, 48), (8, 1, 128)])
@pytest.mark.parametrize("form, window, sinks", [("whole", 0, 0), ("split", 0, 0), ("whole", 9000, 0), ("split", 9000, 0),
                                                 ("split", 8000, 70), ("whole", 40, 0), ("whole", 40, 20)])
def test_rows_that_are_left_without_a_key_are_zero(dev, types, form, heads, kv_heads, d, window, sinks):
    """A row all of whose visible keys lie on pages out of range sees no key: zeros, as before the first key.  Beside it
    rows that see one page, and other requests."""
    rng = np.random.default_rng(32)
    long, page = LONG[form], 16
    lengths, cu = [long, 45, 70], [0, 2, 3, 6]
    cache = po.Cache(rng, lengths, kv_heads, d, page, TYPES[types][1])
    q = queries(rng, [2, 1, 3], heads, d, types)
    for some in ((), (1,), ((long - 1) // page,)):  # pages of the first request that stay
        table, keep = cache.table.copy(), [np.ones(n, bool) for n in lengths]
        table[0], table[2] = -1, len(cache.k_cache)
        keep[0][:] = keep[2][:] = False
        for j in some:
            table[0, j] = cache.table[0, j]
            keep[0][j * page:(j + 1) * page] = True
        got, err = call(dev, q, cache, lengths, cu, heads, types, 3, long, table=table, window=window, sinks=sinks)
        assert err == 1
        assert not got[3:].any()
        check(got, q, cache, lengths, cu, range(3), keep, window, sinks)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("form", list(LONG))
def test_rows_whose_scores_are_all_infinitely_low(dev, types, form):
    """Keys of -inf against queries above zero: keys are seen, all weights are 0, and 0 / 0 is not a number."""
    rng = np.random.default_rng(33)
    long, d, page = LONG[form], 64, 16
    lengths, cu = [long, 45], [0, 1, 2]
    cache = po.Cache(rng, lengths, 2, d, page, TYPES[types][1])
    low = np.uint16(0xFF80) if TYPES[types][1] else np.float32(-np.inf)
    cache.k_cache[cache.table[0, :-(-long // page)], 0, :, 3] = low
    q = np.abs(queries(rng, [1, 1], 4, d, types)) + np.float32(0.5)
    q = to_bf16(q)[1] if TYPES[types][0] else q
    table = cache.table.copy()
    for bad in (False, True):
        if bad:
            table[0, 1:(long - 1) // page] = -1  # some unseen, the first and the last page are seen
        got, err = call(dev, q, cache, lengths, cu, 4, types, 1, long, table=table)
        assert err == bad
        assert np.isnan(got[0, :2]).all() and np.isfinite(got[0, 2:]).all() and np.isfinite(got[1]).all()
