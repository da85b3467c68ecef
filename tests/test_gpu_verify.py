"""verify_drafts against whole masses and 64 bits: accepted drafts and drawn ids are equal."""

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


def run(dev, logits, cu, drafts, u, u_draw, settings, draft_logits=None, draft_row=None, bf16=False, ids=None, max_rows=None,
        workspace=None, stream=None):
    up = dev.DeviceArray.from_host
    token, accepted = (up(np.full(n, 77, np.int32)) for n in (len(drafts), len(cu) - 1))
    err = dev.DeviceArray.zeros(1, np.int32)
    some = lambda a, t: None if a is None else up(np.asarray(a, t))  # noqa: E731
    dev.verify_drafts(up(logits), up(np.asarray(drafts, np.int32)), up(np.asarray(cu, np.int32)), up(np.asarray(u, np.float32)),
                      up(np.asarray(u_draw, np.float32)), token, accepted, max_rows=max_rows,
                      draft_logits=some(draft_logits, logits.dtype), draft_row=some(draft_row, np.int32),
                      temperature=some(settings[0], np.float32), top_k=some(settings[1], np.int32),
                      top_p=some(settings[2], np.float32), min_p=some(settings[3], np.float32), bf16=bf16, ids=ids,
                      workspace=workspace, err=err, stream=stream)
    dev.synchronize()
    return token.host(), accepted.host(), int(err.host()[0])


def oracle(logits, cu, drafts, u, u_draw, settings, small=None):
    """logits, small: fp32 values; small [rows] rows of draft logits, or None."""
    token, accepted = [], []
    get = lambda a, b, none: none if a is None else a[b]  # noqa: E731
    for b in range(len(cu) - 1):
        lo, hi = cu[b], cu[b + 1]
        if hi == lo:
            accepted.append(0)
            continue
        s = (get(settings[0], b, 1.0), get(settings[1], b, 0), get(settings[2], b, 1.0), get(settings[3], b, 0.0))
        t, a = po.verify(logits[lo:hi], drafts[lo:hi - 1], None if small is None else small[lo:hi - 1], s, u[lo:hi], u_draw[b])
        token += t
        accepted.append(a)
    return np.array(token), np.array(accepted)


def mixed(rng, n):
    return (np.where(rng.random(n) < 0.1, 0, rng.uniform(0.5, 1.5, n)).astype(np.float32),
            rng.choice([0, 0, 1, 3, 40, 300], size=n), rng.choice([1.0, 0.9, 0.5, 0.0], size=n).astype(np.float32),
            rng.choice([0.0, 0.0, 0.05, 1.0], size=n).astype(np.float32))


def case(rng, v, counts, noise, spread=2.5):
    cu = np.concatenate([[0], np.cumsum(counts)])
    rows = int(cu[-1])
    logits = (spread * rng.standard_normal((rows, v))).astype(np.float32)
    small = (logits + noise * rng.standard_normal((rows, v))).astype(np.float32)
    return cu, logits, small, rng.random(rows).astype(np.float32), rng.random(len(counts)).astype(np.float32)


def drawn(rng, small, cu, settings):
    """Drafts drawn from the small model's rows under each request's settings."""
    out = np.zeros(len(small), np.int64)
    get = lambda a, b, none: none if a is None else a[b]  # noqa: E731
    for b in range(len(cu) - 1):
        for r in range(cu[b], cu[b + 1]):
            m, total = po.masses(small[r], get(settings[0], b, 1.0), get(settings[1], b, 0), get(settings[2], b, 1.0),
                                 get(settings[3], b, 0.0))
            out[r] = rng.choice(len(m), p=m / total) if total else 0
    return out


@pytest.mark.parametrize("v", [5, 256, 257, 1000, 4096, 4097, 32000, 40001])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("drafted", [True, False])
def test_mixed_settings(dev, v, bf16, drafted):
    rng = np.random.default_rng(v + bf16)
    counts = [1, 2, 5, 3, 0, 4, 1, 9] + [3] * (4 if v > 4096 else 20)
    cu, logits, small, u, u_draw = case(rng, v, counts, 0.7)
    if bf16:
        (logits_in, logits), (small_in, small) = to_bf16(logits), to_bf16(small)
    else:
        logits_in, small_in = logits, small
    settings = mixed(rng, len(counts))
    if drafted:
        drafts = drawn(rng, small, cu, settings)
    else:
        drafts = np.where(rng.random(len(u)) < 0.7, logits.argmax(axis=1), rng.integers(0, v, size=len(u)))
    got = run(dev, logits_in, cu, drafts, u, u_draw, settings, small_in if drafted else None, bf16=bf16)
    want = oracle(logits, cu, drafts, u, u_draw, settings, small if drafted else None)
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0]) and got[2] == 0
    assert v < 256 or 0 < want[1].sum() < len(u) - len(counts)  # some accepted, some not


def test_draft_rows_by_step_and_narrow_ids(dev):
    """Draft logits in blocks of one step for all requests; rows with values past the ids; no settings."""
    rng = np.random.default_rng(2)
    v, wide, counts = 3000, 3040, [4, 2, 1, 5]
    cu, logits, small, u, u_draw = case(rng, wide, counts, 0.5)
    logits[:, v:], small[:, v:] = 50.0, 60.0
    settings = (None,) * 4
    drafts = drawn(rng, small[:, :v], cu, settings)
    blocks = np.full((4 * 4, wide), 9.0, np.float32)
    draft_row = np.full(len(u), -1, np.int64)
    for b, n in enumerate(counts):
        for i in range(n - 1):
            draft_row[cu[b] + i] = i * 4 + b
            blocks[i * 4 + b] = small[cu[b] + i]
    got = run(dev, logits, cu, drafts, u, u_draw, settings, blocks, draft_row, ids=v, max_rows=5)
    want = oracle(logits[:, :v], cu, drafts, u, u_draw, settings, small[:, :v])
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and got[2] == 0


def test_equal_distributions_accept_everything(dev):
    rng = np.random.default_rng(3)
    cu, logits, _, u, u_draw = case(rng, 700, [6] * 30, 0.0)
    settings = mixed(rng, 30)
    drafts = drawn(rng, logits, cu, settings)
    got = run(dev, logits, cu, drafts, u, u_draw, settings, logits)
    want = oracle(logits, cu, drafts, u, u_draw, settings, logits)
    assert (got[1] == 5).all()  # u q < p = q for any u below 1
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_disjoint_distributions_draw_from_the_target(dev):
    rng = np.random.default_rng(4)
    cu, logits, small, u, u_draw = case(rng, 600, [3] * 20, 1.0)
    logits[:, 300:], small[:, :300] = -np.inf, -np.inf
    drafts = drawn(rng, small, cu, (None,) * 4)
    got = run(dev, logits, cu, drafts, u, u_draw, (None,) * 4, small)
    want = oracle(logits, cu, drafts, u, u_draw, (None,) * 4, small)
    assert not got[1].any() and np.array_equal(got[0], want[0])
    assert (got[0].reshape(20, 3)[:, 0] < 300).all() and (got[0].reshape(20, 3)[:, 1:] == -1).all()


def test_infinities_nan_and_rows_of_nothing(dev):
    rng = np.random.default_rng(5)
    v = 500
    cu, logits, small, u, u_draw = case(rng, v, [3] * 12, 0.5)
    logits[0] = -np.inf                       # nothing to accept, id 0
    logits[4, 5:9] = np.nan                   # never drawn
    logits[6, [3, 400]] = np.inf              # those two, evenly
    small[9] = -np.inf                        # q is nowhere: any draft that p has is accepted
    small[12, 17] = np.inf
    logits[15], small[15] = np.nan, np.nan
    settings = (np.full(12, 0.9, np.float32), None, np.full(12, 0.95, np.float32), None)
    drafts = drawn(rng, small, cu, settings)
    drafts[6] = 400
    got = run(dev, logits, cu, drafts, u, u_draw, settings, small)
    want = oracle(logits, cu, drafts, u, u_draw, settings, small)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and got[2] == 0
    assert got[0][0] == 0 and got[1][0] == 0


def test_numbers_out_of_range(dev):
    """A draft, its row, a u or a setting out of range: err, and the rest of the call as it is."""
    rng = np.random.default_rng(6)
    v = 400
    cu, logits, small, u, u_draw = case(rng, v, [4] * 10, 0.3)
    settings = (np.full(10, 0.8, np.float32), np.zeros(10, np.int64), np.ones(10, np.float32), np.zeros(10, np.float32))
    drafts = drawn(rng, small, cu, settings)
    rows = [small[r] for r in range(len(u))]
    draft_row = np.arange(len(u))
    for change in ("draft", "draft_row", "u", "u_draw", "setting"):
        d, r, s, uu, ud, st = drafts.copy(), draft_row.copy(), list(rows), u.copy(), u_draw.copy(), [a.copy() for a in settings]
        if change == "draft":
            d[5], d[13] = -1, v
        elif change == "draft_row":
            r[5], r[13] = -1, len(u)
            s[5] = s[13] = None
        elif change == "u":
            uu[5], uu[13], uu[17] = 1.0, np.nan, -0.5
        elif change == "u_draw":
            ud[1], ud[2] = 1.0, np.nan
        else:
            st[0][1], st[2][2], st[3][3] = -1.0, np.nan, 1.5
        got = run(dev, logits, cu, d, uu, ud, st, small, r)
        want = oracle(logits, cu, d, uu, ud, st, s)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), change
        assert got[2] == 1, change


def test_rows_out_of_range(dev):
    rng = np.random.default_rng(7)
    cu, logits, small, u, u_draw = case(rng, 300, [3, 3, 3], 0.3)
    drafts = drawn(rng, small, cu, (None,) * 4)
    want = oracle(logits, cu, drafts, u, u_draw, (None,) * 4, small)
    got = run(dev, logits, cu, drafts, u, u_draw, (None,) * 4, small, max_rows=2)
    assert (got[0] == 77).all() and not got[1].any() and got[2] == 1
    bad = [0, 3, 9, 12]  # 6 rows, then 3 past the last
    got = run(dev, logits, bad, drafts, u, u_draw, (None,) * 4, small, max_rows=3)
    assert np.array_equal(got[0][:3], want[0][:3]) and (got[0][3:] == 77).all()
    assert got[1].tolist() == [want[1][0], 0, 0] and got[2] == 1


def test_many_requests(dev):
    rng = np.random.default_rng(8)
    counts = rng.integers(0, 4, size=1500)
    cu, logits, small, u, u_draw = case(rng, 64, counts, 0.6)
    settings = mixed(rng, 1500)
    drafts = drawn(rng, small, cu, settings)
    got = run(dev, logits, cu, drafts, u, u_draw, settings, small)
    want = oracle(logits, cu, drafts, u, u_draw, settings, small)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and got[2] == 0


@pytest.mark.parametrize("v, requests, most, drafted", [(5000, 150, 7, True), (5000, 150, 7, False), (33000, 70, 6, True),
                                                         (200, 24, 90, True), (300, 900, 4, False)])
def test_more_rows_than_run_at_once(dev, v, requests, most, drafted):
    """Many workgroups a compute unit, one after the other; some drafts and numbers out of range among them, and requests of
    more than 64 rows."""
    rng = np.random.default_rng(v + most)
    counts = rng.integers(0, most + 1, size=requests)
    counts[rng.integers(0, requests)] = most
    cu, logits, small, u, u_draw = case(rng, v, counts, 0.35)
    settings = mixed(rng, requests)
    if most > 64:
        settings, small, u = (None,) * 4, logits + np.float32(0.01) * small, 0.9 * u  # long runs of accepted drafts
    drafts = drawn(rng, small, cu, settings)
    odd = rng.random(len(u)) < 0.02
    drafts[odd] = rng.choice([-1, v, v + 7], size=int(odd.sum()))
    u = u.copy()
    u[rng.random(len(u)) < 0.02] = 1.0
    for _ in range(2):  # the workspace as the last call left it
        got = run(dev, logits, cu, drafts, u, u_draw, settings, small if drafted else None, max_rows=most)
        want = oracle(logits, cu, drafts, u, u_draw, settings, small if drafted else None)
        assert np.array_equal(got[1], want[1])
        assert np.array_equal(got[0], want[0]) and got[2] == 1
    assert want[1].max() > (3 if drafted else 0)


@pytest.mark.parametrize("v", [3000, 32000, 40001, 131072])
def test_equal_logits(dev, v):
    """Few distinct logits: borders inside long runs of equal ones, bins of more ids than a list holds."""
    rng = np.random.default_rng(v)
    counts = [3, 1, 4, 2, 3, 5]
    cu, logits, small, u, u_draw = case(rng, v, counts, 0.7)
    logits, small = np.round(logits), np.round(small)
    logits[2], logits[3, ::2] = 1.0, -np.inf
    logits[5, 7], small[6, 9] = np.nan, -np.inf
    settings = (np.array([1, 0.7, 1.3, 0.9, 1, 0.5], np.float32), np.array([0, 0, 0, 700, 0, 0]),
                np.array([0.9, 0.5, 1, 0.7, 0.99, 1], np.float32), np.array([0, 0, 0.02, 0, 0.1, 0], np.float32))
    drafts = drawn(rng, small, cu, settings)
    got = run(dev, logits, cu, drafts, u, u_draw, settings, small)
    want = oracle(logits, cu, drafts, u, u_draw, settings, small)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0]) and got[2] == 0
