"""A paged cache whose last pages lie past 2^31 values: append stores there, attention reads there."""

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


@pytest.mark.parametrize("kv_heads, d, rows", [(8, 128, 640), (8, 128, 37)])
def test_pages_past_2_to_31_values(dev, kv_heads, d, rows):
    rng = np.random.default_rng(rows)
    page, pages, heads = 16, 140000, 16  # 2.3e9 values a cache, 4.6 GB
    k_cache, v_cache = (dev.DeviceArray(s, np.uint16) for s in ((pages, kv_heads, page, d), (pages, kv_heads, d, page)))
    held = -(-rows // page)
    mine = pages - 1 - rng.permutation(held + 5)[:held]  # the last pages, in any order
    assert int(mine.min()) * kv_heads * d * page > 2 ** 31
    slot = (mine[np.arange(rows) // page] * page + np.arange(rows) % page).astype(np.int32)
    k, v = (rng.standard_normal((rows, kv_heads * d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((3, heads * d)).astype(np.float32)
    up = dev.DeviceArray.from_host
    err = dev.DeviceArray.zeros(1, np.int32)
    dev.paged_append(up(k), up(v), up(slot), k_cache, v_cache, cache_bf16=True, err=err)
    out = dev.DeviceArray.zeros((3, heads * d), np.float32)
    table = np.full((1, held), 0, np.int32)
    table[0] = mine
    dev.paged_attention(up(q), k_cache, v_cache, up(table), up(np.array([rows], np.int32)), up(np.array([0, 3], np.int32)), out,
                        heads=heads, max_rows=3, max_keys=held * page, scale=1.0 / math.sqrt(d), cache_bf16=True, err=err)
    dev.synchronize()
    assert err.host()[0] == 0

    class At:  # one page of a cache
        def __init__(self, cache, p):
            self.ptr, self.nbytes = cache.ptr + int(p) * kv_heads * d * page * 2, kv_heads * d * page * 2

    part = dev.DeviceArray((kv_heads, page, d), np.uint16)
    kb, vb = (to_bf16(x)[0].reshape(rows, kv_heads, d) for x in (k, v))
    for j, p in enumerate(mine):
        n = min(page, rows - j * page)
        dev.copy(part, At(k_cache, p))
        assert np.array_equal(part.host()[:, :n], kb[j * page:j * page + n].transpose(1, 0, 2))
        dev.copy(part, At(v_cache, p))
        got = part.host().reshape(kv_heads, d, page)
        assert np.array_equal(got[:, :, :n], vb[j * page:j * page + n].transpose(1, 2, 0))
    want, bound = po.attention(q.reshape(3, heads, d), to_bf16(k)[1].reshape(rows, kv_heads, d),
                               to_bf16(v)[1].reshape(rows, kv_heads, d), rows, scale=1.0 / math.sqrt(d))
    assert (np.abs(out.host().reshape(3, heads, d) - want) <= bound).all()
