"""paged_plan and paged_append: whole numbers and copies, exactly."""

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


NAMES = ("lengths", "held", "table", "free", "count", "cu", "slot", "request", "position", "served", "err")


def plan(dev, lengths, new, held, page, table, free, count, cap, in_place=False, maps=True, stream=None):
    up = lambda a: dev.DeviceArray.from_host(np.array(a, np.int32))  # noqa: E731
    fill = lambda n: dev.DeviceArray.from_host(np.full(n, 77, np.int32))  # noqa: E731
    n = len(lengths)
    a = dict(lengths=up(lengths), held=up(held), count=up([count]), table=up(table), free=up(free))
    o = {f: a[f] if in_place else fill(a[f].shape) for f in ("lengths", "held", "count")}
    rows = {f: fill(max(cap, 1)) for f in ("slot", "request", "position")}
    cu, served, err = fill(n + 1), fill(1), dev.DeviceArray.zeros(1, np.int32)
    given = {f + "_of_row": rows[f] for f in rows} if maps else {}
    dev.paged_plan(a["lengths"], up(new), page, a["table"], a["held"], a["free"], a["count"], o["lengths"], o["held"], o["count"],
                   cu, served, row_cap=cap, err=err, stream=stream, **given)
    dev.synchronize()
    got = dict(o, table=a["table"], free=a["free"], cu=cu, served=served, err=err, **rows)
    got = {f: got[f].host() for f in NAMES}
    if not maps:
        assert all((got[f] == 77).all() for f in rows)
    return got


def same(got, want, cap, maps=True):
    for f in NAMES:
        if f in ("slot", "request", "position"):
            if maps:
                assert np.array_equal(got[f][:cap], want[f]), f
                assert (got[f][cap:] == 77).all(), f
        else:
            assert np.array_equal(got[f].ravel(), np.ravel(want[f])), (f, got[f], want[f])


def state(rng, requests, page, most, new_most, ended=0.1, spare=None):
    new = rng.integers(0, new_most + 1, size=requests)
    lengths = rng.integers(0, most + 1, size=requests)
    held = -(-lengths // page) + (rng.random(requests) < 0.2)
    new[rng.random(requests) < ended] = rng.choice([-1, -5])
    width = -(-(most + new_most) // page) + 1
    need = int(np.maximum(-(-(lengths + np.maximum(new, 0)) // page) - held, 0).sum())
    pages = int(held.sum()) + (need + 3 if spare is None else spare)
    order = rng.permutation(pages)
    table = np.full((requests, width), -9, np.int64)
    at = 0
    for b in range(requests):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    free = np.full(pages, -8, np.int64)
    free[:pages - at] = order[at:]
    return lengths, new, held, page, table, free, pages - at


@pytest.mark.parametrize("requests, page, most, new_most, cap", [
    (1, 16, 40, 1, 4), (3, 8, 40, 9, 64), (64, 16, 500, 1, 128), (100, 32, 900, 6, 700), (1000, 16, 300, 5, 4096),
    (1025, 64, 100, 3, 4096), (700, 16, 400, 40, 20000), (8192, 8, 30, 2, 20000), (5, 1024, 5000, 2000, 12000), (2, 16, 0, 0, 0),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(dev, requests, page, most, new_most, cap, in_place):
    rng = np.random.default_rng(requests + page)
    args = state(rng, requests, page, most, new_most)
    same(plan(dev, *args, cap, in_place=in_place), po.plan(*args, cap), cap)


@pytest.mark.parametrize("cap, spare, ended, short", [
    (4096, 20, 0.1, True), (300, None, 0.1, True), (0, None, 0.1, True), (5000, 7, 0.1, True),
    (9000, 0, 0.1, False),  # what comes back is enough
    (9001, 0, 0.0, True), (9002, 0, 0.03, True)])
def test_plan_serves_in_order_up_to_the_first_that_does_not_fit(dev, cap, spare, ended, short):
    rng = np.random.default_rng(cap)
    args = state(rng, 400, 16, 300, 30, ended=ended, spare=spare)
    want = po.plan(*args, cap)
    assert (want["served"] < 400) == short and want["err"] == 0
    same(plan(dev, *args, cap), want, cap)
    same(plan(dev, *args, cap, maps=False), want, cap, maps=False)


@pytest.mark.parametrize("where, value", [("lengths", -1), ("lengths", 10000), ("held", -1), ("held", 10 ** 6), ("new", 10 ** 9),
                                          ("count", -1), ("count", 10 ** 6), ("free", -1), ("free", 10 ** 6), ("table", 10 ** 6)])
def test_plan_of_numbers_out_of_range(dev, where, value):
    rng = np.random.default_rng(8)
    lengths, new, held, page, table, free, count = state(rng, 50, 16, 300, 8, ended=0.0)
    new[20:23] = (5, 7, 6)
    if where == "lengths":
        lengths[20] = value
    elif where == "held":
        held[20] = value
    elif where == "new":
        new[20] = value
    elif where == "count":
        count = value
    elif where == "free":
        free[count - 2] = value
    else:
        lengths[20], held[20] = 20, 2
        table[20, 1] = value
    want = po.plan(lengths, new, held, page, table, free, count, 512)
    assert want["err"] == (where != "new")
    same(plan(dev, lengths, new, held, page, table, free, count, 512), want, 512)


def test_plan_of_ended_requests_that_hold_too_much(dev):
    rng = np.random.default_rng(9)
    lengths, new, held, page, table, free, count = state(rng, 30, 16, 300, 3, ended=0.0)
    new[3], new[7], held[7] = -1, -1, -4
    count = len(free) - held[3] + 2  # more come back than there is room for
    free[:count] = np.arange(count)
    want = po.plan(lengths, new, held, page, table, free, count, 512)
    assert want["err"] == 1
    same(plan(dev, lengths, new, held, page, table, free, count, 512), want, 512)


def bits(x, bf16):
    return to_bf16(x)[0] if bf16 else x


@pytest.mark.parametrize("in_bf16, cache_bf16", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("rows, kv_heads, d, page, order", [
    (1, 8, 64, 16, "runs"), (1, 1, 48, 8, "scattered"), (61, 8, 48, 16, "scattered"), (200, 2, 128, 64, "runs"),
    (1000, 3, 64, 8, "runs"), (333, 8, 64, 16, "mixed"), (129, 2, 48, 1024, "mixed"), (70, 1, 128, 32, "backwards")])
def test_append(dev, in_bf16, cache_bf16, rows, kv_heads, d, page, order):
    rng = np.random.default_rng(rows + d)
    pages = -(-rows // page) * 2 + 3
    slots = pages * page
    if order == "runs":
        first = int(rng.integers(0, slots - rows + 1))
        slot = np.arange(first, first + rows)
    elif order == "scattered":
        slot = rng.permutation(slots)[:rows]
    elif order == "backwards":
        slot = np.arange(rows)[::-1] + 5
    else:  # runs of all lengths at places of their own, rows left out between them
        slot = np.arange(rows) + 3
        cuts = np.sort(rng.integers(0, rows, size=12))
        for j, c in enumerate(cuts):
            slot[c:] += 1 + j % 3
        slot[rng.random(rows) < 0.1] = -1 - int(rng.integers(0, 5))
    assert slot.max() < slots and len(set(slot[slot >= 0])) == (slot >= 0).sum()
    width = kv_heads * d
    x = rng.standard_normal((rows, 2 * width + 24)).astype(np.float32)
    x[0, :3], x[-1, width + 8:width + 10] = (np.nan, np.inf, -0.0), (-np.inf, np.nan)
    src = bits(x, in_bf16)
    val = to_bf16(x)[1] if in_bf16 else x
    dt = np.uint16 if cache_bf16 else np.float32
    k0, v0 = (rng.integers(1, 100, size=s).astype(dt) for s in ((pages, kv_heads, page, d), (pages, kv_heads, d, page)))
    k, v = k0.copy(), v0.copy()
    for r in range(rows):
        if slot[r] >= 0:
            p, o = divmod(int(slot[r]), page)
            k[p, :, o] = bits(val[r, :width], cache_bf16).reshape(kv_heads, d)
            v[p, :, :, o] = bits(val[r, width + 8:2 * width + 8], cache_bf16).reshape(kv_heads, d)
    up = dev.DeviceArray.from_host
    a, kc, vc, err = up(src), up(k0), up(v0), dev.DeviceArray.zeros(1, np.int32)

    class At:
        def __init__(self, offset):
            self.ptr, self.shape = a.ptr + offset * src.itemsize, src.shape

    dev.paged_append(At(0), At(width + 8), up(slot.astype(np.int32)), kc, vc, bf16=in_bf16, cache_bf16=cache_bf16, err=err)
    dev.synchronize()
    for got, want in ((kc.host(), k), (vc.host(), v)):
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    assert err.host()[0] == 0


def test_append_of_odd_addresses_and_slots_past_the_cache(dev):
    """Rows at addresses of their values' alignment only; a slot past the last page sets err and stores nothing."""
    rng = np.random.default_rng(10)
    rows, h, d, page, pages = 40, 2, 64, 16, 4
    for in_bf16 in (False, True):
        x = rng.standard_normal((rows, 3 * h * d + 1)).astype(np.float32)
        src = bits(x, in_bf16)
        val = to_bf16(x)[1] if in_bf16 else x
        slot = np.arange(rows).astype(np.int32) + 7
        slot[5], slot[6] = pages * page, 2 ** 31 - 1
        up = dev.DeviceArray.from_host
        a, kc, vc = up(src), dev.DeviceArray.zeros((pages, h, page, d), np.uint16), dev.DeviceArray.zeros((pages, h, d, page), np.uint16)
        err = dev.DeviceArray.zeros(1, np.int32)

        class At:
            def __init__(self, offset):
                self.ptr, self.shape = a.ptr + offset * src.itemsize, src.shape

        dev.paged_append(At(1), At(h * d + 3), up(slot), kc, vc, bf16=in_bf16, cache_bf16=True, err=err)
        dev.synchronize()
        k, v = np.zeros(kc.shape, np.uint16), np.zeros(vc.shape, np.uint16)
        for r in range(rows):
            if slot[r] < pages * page:
                p, o = divmod(int(slot[r]), page)
                k[p, :, o] = to_bf16(val[r, 1:1 + h * d])[0].reshape(h, d)
                v[p, :, :, o] = to_bf16(val[r, h * d + 3:2 * h * d + 3])[0].reshape(h, d)
        assert np.array_equal(kc.host(), k) and np.array_equal(vc.host(), v)
        assert err.host()[0] == 1
