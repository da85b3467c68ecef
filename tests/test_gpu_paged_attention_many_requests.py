"""paged_attention of more requests than a workgroup has threads, cut into shares: each share's beginning is searched for
step by step, 256 requests at a time."""

from importlib import import_module

import numpy as np
import pytest

import paged_oracle as po
from test_gpu_paged_attention import TYPES, check, mean_of_visible, queries, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


def batch(rng, requests, most):
    """Short caches, long ones around the borders of the steps and elsewhere, requests without rows or without keys.  The
    longest takes more work than the whole batch divided by what the chip reads at once and the cost of splitting, which is
    where the kernel cuts sequences."""
    lengths = rng.integers(1, 90, size=requests)
    rows = np.where(rng.random(requests) < 0.1, 0, rng.integers(1, most + 1, size=requests))
    for b in [0, 255, 256, 257, requests - 1, *rng.integers(0, requests, size=5)] + ([511, 512] if requests > 512 else []):
        if b < requests:
            lengths[b], rows[b] = rng.integers(4000, 7000), max(rows[b], 1)
    lengths[requests // 3] = 20000
    rows[requests // 3] = most
    lengths[3], rows[3] = 0, 0
    rows[4] = 0
    return lengths.tolist(), rows.tolist()


def workspace_of(dev, lengths, rows, heads, kv_heads, d, types):
    need = dev.paged_attention_workspace(len(lengths), max(rows), max(lengths), heads, kv_heads, d, bf16=TYPES[types][0],
                                         cache_bf16=TYPES[types][1])
    assert need > 0
    return dev.DeviceArray.from_host(np.full(need, 0x5A, np.uint8))


def was_split(space, requests, kv_heads):
    """The parts come first in the workspace, 8 bytes a sequence (at least) after them."""
    parts = space.host()[:-8 * requests * kv_heads]
    return len(parts) > 0 and (parts != 0x5A).any()


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("requests", [256, 257, 512, 513, 1000])
@pytest.mark.parametrize("kv_heads, group, d, most", [(1, 4, 64, 1), (2, 2, 48, 4)])
def test_every_visible_key_once(dev, types, requests, kv_heads, group, d, most):
    rng = np.random.default_rng(requests)
    lengths, rows = batch(rng, requests, most)
    heads = kv_heads * group
    cache = po.Cache(rng, lengths, kv_heads, d, 16, TYPES[types][1], values="whole")
    q = np.zeros((sum(rows), heads, d), np.float32)
    space = workspace_of(dev, lengths, rows, heads, kv_heads, d, types)
    got = run(dev, q, cache, lengths, rows, heads, types, workspace=space)
    assert was_split(space, requests, kv_heads)
    assert np.array_equal(got, mean_of_visible(cache, lengths, rows, heads))


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("requests", [257, 513])
def test_against_the_formula(dev, types, requests):
    rng = np.random.default_rng(requests + 1)
    lengths, rows = batch(rng, requests, 3)
    cache = po.Cache(rng, lengths, 2, 64, 16, TYPES[types][1])
    q = queries(rng, rows, 4, 64, types)
    space = workspace_of(dev, lengths, rows, 4, 2, 64, types)
    got = run(dev, q, cache, lengths, rows, 4, types, workspace=space)
    assert was_split(space, requests, 2)
    check(got, q, cache, lengths, rows)


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("window, sinks", [(5000, 3), (3000, 200)])
def test_windows(dev, types, window, sinks):
    rng = np.random.default_rng(window)
    lengths, rows = batch(rng, 300, 3)
    cache = po.Cache(rng, lengths, 1, 48, 16, TYPES[types][1], values="whole")
    got = run(dev, np.zeros((sum(rows), 5, 48), np.float32), cache, lengths, rows, 5, types, window=window, sinks=sinks)
    assert np.array_equal(got, mean_of_visible(cache, lengths, rows, 5, window, sinks))


@pytest.mark.parametrize("types", list(TYPES))
def test_two_query_tiles_over_long_caches(dev, types):
    """Several query tiles of a request, each cut: 24 rows of 4 heads to a key head are three of 32 columns."""
    rng = np.random.default_rng(50)
    lengths, rows = [6000, 3000, 24, 50], [24, 9, 24, 17]
    cache = po.Cache(rng, lengths, 2, 64, 16, TYPES[types][1], values="whole")
    space = workspace_of(dev, lengths, rows, 8, 2, 64, types)
    got = run(dev, np.zeros((sum(rows), 8, 64), np.float32), cache, lengths, rows, 8, types, workspace=space)
    assert was_split(space, 4, 2 * 3)
    assert np.array_equal(got, mean_of_visible(cache, lengths, rows, 8))
    cache = po.Cache(rng, lengths, 2, 64, 16, TYPES[types][1])
    q = queries(rng, rows, 8, 64, types)
    check(run(dev, q, cache, lengths, rows, 8, types), q, cache, lengths, rows)
