"""verify_drafts where a request that cannot be taken lies over the rows of others: those are verified as without it."""

from importlib import import_module

import numpy as np
import pytest

from test_gpu_verify import case, drawn, mixed, oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


@pytest.mark.parametrize("cu, good", [
    ([0, 3, 6, 3, 12], [0, 1]),       # one that ends before it begins, one of nine rows over the second's
    ([0, 3, 6, 9, 6, 200], [0, 1, 2]),  # past the last row
    ([-3, 9, 6, 9], [2]),             # from before the first row
    ([0, 12, 9, 12], [2]),
])
@pytest.mark.parametrize("v", [700, 5000, 40001])
@pytest.mark.parametrize("drafted", [True, False])
def test_others_are_verified(dev, cu, good, v, drafted):
    rng = np.random.default_rng(v + len(cu))
    rows, requests = 12, len(cu) - 1
    _, logits, small, u, _ = case(rng, v, [rows], 0.5)
    u_draw = rng.random(requests).astype(np.float32)
    settings = mixed(rng, requests)
    settings[0][:] = np.linspace(0.6, 1.4, requests)  # no two alike
    settings[1][:], settings[2][:], settings[3][:] = 0, 1.0, 0.0
    settings[2][::2], settings[1][1::2] = 0.9, 50
    drafts = rng.integers(0, v, size=rows)
    for b in good:
        at = slice(cu[b], cu[b + 1])
        own = tuple(s[b:b + 1] for s in settings)
        drafts[at] = drawn(rng, (small if drafted else logits)[at], [0, cu[b + 1] - cu[b]], own)
    up = dev.DeviceArray.from_host
    space = up(np.full(dev.verify_drafts_workspace(rows, requests, v, drafted), 0xFF, np.uint8))
    token, accepted, err = up(np.full(rows, 77, np.int32)), up(np.full(requests, 77, np.int32)), dev.DeviceArray.zeros(1, np.int32)
    dev.verify_drafts(up(logits), up(drafts.astype(np.int32)), up(np.array(cu, np.int32)), up(u), up(u_draw), token, accepted,
                      max_rows=3, draft_logits=up(small) if drafted else None, temperature=up(settings[0]),
                      top_k=up(settings[1].astype(np.int32)), top_p=up(settings[2]), min_p=up(settings[3]), workspace=space, err=err)
    dev.synchronize()
    assert err.host()[0] == 1
    left, got = np.ones(rows, bool), token.host()
    for b in range(requests):
        if b not in good:
            assert accepted.host()[b] == 0
            continue
        at = slice(cu[b], cu[b + 1])
        want = oracle(logits[at], [0, cu[b + 1] - cu[b]], drafts[at], u[at], u_draw[b:b + 1], tuple(s[b:b + 1] for s in settings),
                      small[at] if drafted else None)
        assert got[at].tolist() == want[0].tolist() and accepted.host()[b] == want[1][0], b
        left[at] = False
    assert (got[left] == 77).all()
