"""A row of paged_attention does not depend on what lies beside it, to the bit: not on finite keys and values that it does
not see, and not on the queries of the rows and heads that share its tile."""

import math
from importlib import import_module

import numpy as np
import pytest

import paged_oracle as po
from decode_step_oracle import to_bf16
from test_gpu_paged_attention import TYPES, check, queries, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


def same_bits(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("long", [700, 9000])  # a workgroup's own; cut into shares and joined
@pytest.mark.parametrize("heads, kv_heads, d, n", [(4, 2, 64, 3), (8, 1, 128, 5), (6, 6, 48, 4)])
def test_neighbours_queries(dev, types, long, heads, kv_heads, d, n):
    rng = np.random.default_rng(long + d)
    lengths, rows = [long, 33, 150], [n, n, n]
    cache = po.Cache(rng, lengths, kv_heads, d, 16, TYPES[types][1])
    q = queries(rng, rows, heads, d, types)
    plain = run(dev, q, cache, lengths, rows, heads, types)
    for mine in (0, n // 2):  # of each request's rows; of its heads the first of every key head
        own = np.zeros((sum(rows), heads), bool)
        own[mine::n, ::heads // kv_heads] = True
        for size in (0.0, 16.0, 1024.0):  # powers of two: bfloat16 stays exact
            beside = np.where(own[..., None], q, q * np.float32(size))
            got = run(dev, beside, cache, lengths, rows, heads, types)
            assert same_bits(got[own], plain[own]), (mine, size)
            if size < 1024:
                check(got, beside, cache, lengths, rows)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("long", [700, 9000])
@pytest.mark.parametrize("page, window, sinks", [(16, 0, 0), (8, 0, 0), (64, 0, 0), (16, 300, 5)])
def test_finite_keys_and_values_out_of_sight(dev, types, long, page, window, sinks):
    """The later rows' own keys, keys ahead of a window and slots past the end, of any size."""
    rng = np.random.default_rng(long + page)
    heads, kv_heads, d, n = 4, 2, 64, 6
    lengths, rows = [long, 40, 166], [n, n, n]
    cache = po.Cache(rng, lengths, kv_heads, d, page, TYPES[types][1])
    q = queries(rng, rows, heads, d, types)
    plain = run(dev, q, cache, lengths, rows, heads, types, window=window, sinks=sinks)
    for i in (0, n - 2):
        own = np.zeros(sum(rows), bool)
        own[i::n] = True
        for size in (0.0, 64.0, 2.0 ** 20):
            other = po.Cache(rng, lengths, kv_heads, d, page, TYPES[types][1])
            other.table = cache.table
            other.k_cache, other.v_cache = cache.k_cache.copy(), cache.v_cache.copy()
            for b, length in enumerate(lengths):
                see = set(po.visible(length, n, i, window, sinks).tolist())
                for j in range(-(-length // page) * page):  # whole pages
                    if j in see:
                        continue
                    p, o = cache.table[b, j // page], j % page
                    x = (size * rng.standard_normal((2, kv_heads, d))).astype(np.float32)
                    x = to_bf16(x)[0] if TYPES[types][1] else x
                    other.k_cache[p, :, o], other.v_cache[p, :, :, o] = x[0], x[1]
            got = run(dev, q, other, lengths, rows, heads, types, window=window, sinks=sinks)
            assert same_bits(got[own], plain[own]), (i, size)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_infinities_and_nan_out_of_sight(dev, types, bad):
    """Among the tile that a row sees a part of: the sums may come in another order, within the formula's bounds."""
    rng = np.random.default_rng(41)
    lengths, rows = [9000, 700], [3, 3]
    cache = po.Cache(rng, lengths, 2, 64, 16, TYPES[types][1])
    q = queries(rng, rows, 4, 64, types)
    value = to_bf16(np.float32([bad]))[0][0] if TYPES[types][1] else np.float32(bad)
    for b, length in enumerate(lengths):
        page, place = cache.table[b, (length - 1) // 16], (length - 1) % 16
        cache.k_cache[page, :, place], cache.v_cache[page, :, :, place] = value, value
    got = run(dev, q, cache, lengths, rows, 4, types)
    for b in range(2):
        want, bound = po.attention(q[3 * b:3 * b + 3], cache.k[b], cache.v[b], lengths[b], scale=1.0 / math.sqrt(64))
        assert (np.abs(got[3 * b:3 * b + 2] - want[:2]) <= bound[:2]).all()
