"""paged_append of many rows: 16 rows a workgroup, values turned by aligned groups of eight slots where rows run on."""

from importlib import import_module

import numpy as np
import pytest

from decode_step_oracle import to_bf16

pytestmark = pytest.mark.gpu

SMALL = 4096  # rows times key heads up to here are a wave's each


@pytest.fixture(scope="module")
def dev(pkg):
    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


def bits(x, bf16):
    return to_bf16(x)[0] if bf16 else x


def slots_of(rng, order, rows, page):
    """(slot of each row, pages).  Every slot at most once."""
    pages = 2 * -(-rows // page) + 6
    whole = pages * page
    if order == "run":  # begins inside a group
        return np.arange(rows) + 13, pages
    if order == "aligned":
        return np.arange(rows) + 16, pages
    if order == "scattered":
        return rng.permutation(whole)[:rows], pages
    if order == "backwards":
        return np.arange(rows)[::-1] + 5, pages
    if order == "groups":  # of eight, each aligned, in any order; their rows begin at any place of a workgroup's
        first = rng.permutation(whole // 8)[:-(-rows // 8) + 1] * 8
        return (first[:, None] + np.arange(8)).ravel()[3:][:rows], pages
    if order == "pages":  # a request's pages, in any order, from inside the first on
        at = rng.permutation(pages)
        s = np.arange(rows) + int(rng.integers(1, page))
        return at[s // page] * page + s % page, pages
    # runs of all lengths, rows left out between and inside them
    slot = np.arange(rows) + 3
    for c in np.sort(rng.integers(0, rows, size=rows // 11)):
        slot[c:] += int(rng.integers(0, 3))
    slot = slot % whole
    slot = np.where(np.arange(rows) < whole, slot, -1)
    first = np.unique(slot, return_index=True)[1]
    twice = np.ones(rows, bool)
    twice[first] = False
    out = rng.random(rows) < (0.3 if order == "holes" else 0.02)
    return np.where(out | twice, -1 - rng.integers(0, 9, size=rows), slot), pages


ORDERS = ["run", "aligned", "scattered", "backwards", "groups", "pages", "mixed", "holes"]


@pytest.mark.parametrize("in_bf16, cache_bf16", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("kv_heads, d, rows, page", [(8, 64, 517, 16), (3, 48, 1399, 8), (128, 128, 33, 32), (2, 48, 2050, 1024),
                                                     (1, 64, 4097, 64), (5, 128, 825, 16)])
@pytest.mark.parametrize("order", ORDERS)
def test_append(dev, in_bf16, cache_bf16, kv_heads, d, rows, page, order):
    rng = np.random.default_rng(rows + ORDERS.index(order))
    assert rows * kv_heads > SMALL and rows % 16 != 0
    slot, pages = slots_of(rng, order, rows, page)
    there = slot >= 0
    assert slot.max() < pages * page and len(set(slot[there].tolist())) == there.sum() and there.sum() > rows // 2
    width = kv_heads * d
    x = rng.standard_normal((rows, 2 * width + 3)).astype(np.float32)  # of their values' alignment only
    x[0, :3], x[-1, width + 2:width + 4] = (np.nan, np.inf, -0.0), (-np.inf, np.nan)
    past = rng.integers(0, rows, size=3)  # slots past the cache: left out, err is set
    given = slot.astype(np.int64)
    given[past] = (pages * page, 2 ** 31 - 1, pages * page + 8)
    there[past] = False
    src, val = bits(x, in_bf16), to_bf16(x)[1] if in_bf16 else x
    dt = np.uint16 if cache_bf16 else np.float32
    up = dev.DeviceArray.from_host
    a = up(src)

    class At:
        def __init__(self, offset):
            self.ptr, self.shape = a.ptr + offset * src.itemsize, src.shape

    for left_out in (False, True):
        s = given if left_out else np.where(there, slot, -1)
        k0, v0 = (rng.integers(1, 100, size=n).astype(dt) for n in ((pages, kv_heads, page, d), (pages, kv_heads, d, page)))
        k, v = k0.copy(), v0.copy()
        p, o = slot[there] // page, slot[there] % page
        k[p, :, o] = bits(val[there, 1:1 + width], cache_bf16).reshape(-1, kv_heads, d)
        v[p, :, :, o] = bits(val[there, width + 2:2 * width + 2], cache_bf16).reshape(-1, kv_heads, d)
        kc, vc, err = up(k0), up(v0), dev.DeviceArray.zeros(1, np.int32)
        dev.paged_append(At(1), At(width + 2), up(s.astype(np.int32)), kc, vc, bf16=in_bf16, cache_bf16=cache_bf16, err=err)
        dev.synchronize()
        for got, want in ((kc.host(), k), (vc.host(), v)):
            assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
        assert err.host()[0] == left_out
