"""marian_hip_sample_logits and marian_hip_sample_candidates against whole-number running sums."""

import numpy as np
import pytest

import decode_step_oracle as dso
from hip_graph import Graph

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    from importlib import import_module

    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


class At:
    def __init__(self, base, offset, shape):
        self.base, self.ptr, self.shape = base, base.ptr + offset, shape


def settings(rng, rows):
    pick = lambda v, t: rng.choice(np.array(v, t), size=rows)  # noqa: E731
    return dict(temperature=pick([0.0, 0.1, 0.7, 1.0, 1.3, 5.0], np.float32),
                top_k=pick([-1, 0, 0, 1, 2, 3, 40, 1000], np.int32), top_p=pick([0.0, 0.1, 0.5, 0.9, 0.999, 1.0, 1.0, 1.5], np.float32),
                min_p=pick([0.0, 0.0, 0.0, 1e-4, 0.05, 1.0], np.float32))


def draw(dev, logits, u, bf16=False, **f):
    """(token, logprob, err) of the rows of a host array, with sentinels behind them."""
    D = dev.DeviceArray
    rows = len(u)
    token, lp, err = D((rows + 3,), np.int32), D((rows + 3,), np.float32), D.zeros(1, np.int32)
    token.fill_bytes(0x5A)
    lp.fill_bytes(0x5A)
    dl = D.from_host(logits)
    dev.sample_logits(dl, D.from_host(np.asarray(u, np.float32)), token, logprob=lp, err=err, bf16=bf16,
                      **{k: D.from_host(v) for k, v in f.items()})
    dev.synchronize()
    t, p = token.host(), lp.host()
    assert (t[rows:].view(np.uint8) == 0x5A).all() and (p[rows:].view(np.uint8) == 0x5A).all()
    return t[:rows], p[:rows], int(err.host()[0])


def agree(token, lp, values, u, **f):
    for m in range(len(u)):
        mine = {k: v[m] for k, v in f.items()}
        want, want_lp = dso.sample(values[m], u=u[m], **mine)
        assert token[m] == want, (m, mine, u[m], int(token[m]), want)
        # one rounding to fp32, of a value whose masses are within a unit of 2^-44
        assert lp[m] == want_lp or abs(lp[m] - want_lp) <= 2.0 ** -24 * abs(want_lp) + 1e-10, (m, mine, lp[m], want_lp)


KINDS = ["normal", "flat", "two", "bf16", "masked", "peaked", "ramp"]


def values_of(kind, rng, rows, n):
    l = (2.5 * rng.standard_normal((rows, n))).astype(np.float32)
    if kind == "flat":
        l[:] = 1.25
    elif kind == "two":
        l = np.where(rng.random((rows, n)) < 0.3, 0.5, -0.5).astype(np.float32)
    elif kind == "bf16":  # many equal logits
        l = dso.to_bf16(l)[1]
    elif kind == "masked":
        l[rng.random((rows, n)) < 0.9] = -np.inf
        l[:, ::7] = np.nan
    elif kind == "peaked":
        l *= 20
    elif kind == "ramp":
        l = np.broadcast_to(np.linspace(-30, 0, n, dtype=np.float32), (rows, n)).copy()
    return l


SIZES = [1, 2, 3, 4, 5, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 4095, 4096, 4097, 32000, 32767, 32768, 32769, 50001]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", SIZES)
def test_sizes_and_distributions(dev, n, kind):
    print(f"sample n={n} {kind}", flush=True)
    rng = np.random.default_rng(n)
    rows = 64 if n < 5000 else 24
    l = values_of(kind, rng, rows, n)
    u = rng.random(rows).astype(np.float32) * np.float32(0.999999)
    u[0], u[1 % rows] = 0.0, np.float32(1 - 2.0 ** -24)
    f = settings(rng, rows)
    token, lp, err = draw(dev, l, u, **f)
    assert err == 0
    agree(token, lp, l, u, **f)


@pytest.mark.parametrize("n", [100003, 262145, 524288])
def test_large_vocabularies(dev, n):
    print(f"sample n={n}", flush=True)
    rng = np.random.default_rng(n)
    for kind in ("normal", "flat", "bf16"):
        l = values_of(kind, rng, 6, n)
        u = rng.random(6).astype(np.float32)
        f = dict(temperature=np.array([1, 1, 0.8, 1.2, 1, 1], np.float32), top_k=np.array([0, 0, 5000, 0, 300, 0], np.int32),
                 top_p=np.array([1, 0.9, 0.9, 0.99, 1, 1], np.float32), min_p=np.array([0, 0, 0, 0.001, 0, 0.2], np.float32))
        token, lp, err = draw(dev, l, u, **f)
        assert err == 0
        agree(token, lp, l, u, **f)


@pytest.mark.parametrize("n", [7, 1000, 5003, 70001])
def test_bf16_rows_at_odd_addresses(dev, n):
    rng = np.random.default_rng(n)
    rows, ld = 20, n + 3
    bits, v = dso.to_bf16((3 * rng.standard_normal(rows * ld + 1)).astype(np.float32))
    u = rng.random(rows).astype(np.float32)
    f = settings(rng, rows)
    D = dev.DeviceArray
    base, token, lp = D.from_host(bits), D.zeros(rows, np.int32), D.zeros(rows, np.float32)
    dev.sample_logits(At(base, 2, (rows, ld)), D.from_host(u), token, ids=n, logprob=lp, bf16=True,
                      **{k: D.from_host(x) for k, x in f.items()})
    dev.synchronize()
    agree(token.host(), lp.host(), v[1:].reshape(rows, ld)[:, :n], u, **f)


@pytest.mark.parametrize("n, ld, off", [(6, 9, 1), (1001, 1003, 3), (32000, 32001, 2), (40001, 40007, 1)])
def test_fp32_strides_and_addresses(dev, n, ld, off):
    rng = np.random.default_rng(n)
    rows = 16
    l = (3 * rng.standard_normal(rows * ld + off)).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    f = settings(rng, rows)
    D = dev.DeviceArray
    base, token, lp = D.from_host(l), D.zeros(rows, np.int32), D.zeros(rows, np.float32)
    dev.sample_logits(At(base, 4 * off, (rows, ld)), D.from_host(u), token, ids=n, logprob=lp,
                      **{k: D.from_host(x) for k, x in f.items()})
    dev.synchronize()
    agree(token.host(), lp.host(), l[off:].reshape(rows, ld)[:, :n], u, **f)


def test_nothing_to_draw_and_extremes(dev):
    n = 40
    l = np.zeros((9, n), np.float32)
    l[0] = -np.inf
    l[1] = np.nan
    l[2, 5:9] = np.inf
    l[3, 4] = 3e38
    l[4] = -3e38
    l[5, :] = -np.inf
    l[5, 17] = -3.4e38
    l[6] = np.where(np.arange(n) % 2 == 0, 0.0, -0.0)  # equal
    l[7] = np.finfo(np.float32).min
    l[8] = np.linspace(0, 1e-30, n)
    u = np.full(9, 0.6, np.float32)
    for t in (1.0, 1e-30, 1e30, np.inf):
        for k, p, mp in ((0, 1.0, 0.0), (3, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 1.0), (7, 0.3, 0.5)):
            f = dict(temperature=np.full(9, t, np.float32), top_k=np.full(9, k, np.int32),
                     top_p=np.full(9, p, np.float32), min_p=np.full(9, mp, np.float32))
            token, lp, err = draw(dev, l, u, **f)
            assert err == 0
            agree(token, lp, l, u, **f)


def test_borders_of_the_running_mass(dev):
    """Equal masses: u at a multiple of 1 / n begins the next id, the number below it ends the one before."""
    n = 256
    j = np.arange(n)
    edge = (j / n).astype(np.float32)
    below = np.nextafter(edge, np.float32(-1)).clip(0)
    l = np.full((2 * n, n), -2.0, np.float32)
    token, lp, _ = draw(dev, l, np.concatenate([edge, below]))
    assert np.array_equal(token[:n], j)
    # u counts in multiples of 2^-32: below 2^-8 the number under an edge may round down no further than the id before
    assert np.array_equal(token[n:], np.maximum(j - 1, 0))
    assert np.allclose(lp, -np.log(n), rtol=1e-7)


def test_defaults_and_bad_settings(dev):
    rng = np.random.default_rng(0)
    l = rng.standard_normal((5, 300)).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    token, lp, err = draw(dev, l, u)  # every array left out
    assert err == 0
    agree(token, lp, l, u)
    for f, v in (("temperature", -1.0), ("temperature", np.nan), ("top_p", -0.1), ("top_p", np.nan), ("min_p", 1.5),
                 ("min_p", -0.5), ("min_p", np.nan), ("u", 1.0), ("u", -0.1), ("u", np.nan)):
        a = dict(temperature=np.ones(5, np.float32), top_p=np.ones(5, np.float32), min_p=np.zeros(5, np.float32))
        w = u.copy()
        (w if f == "u" else a[f])[2] = v
        token, lp, err = draw(dev, l, w, **a)
        assert err == 1, f
        assert token[2] == np.argmax(l[2]) and lp[2] == 0.0
        rest = [0, 1, 3, 4]
        agree(token[rest], lp[rest], l[rest], u[rest])


def run_candidates(dev, flat, cand, off, most, u, **f):
    D = dev.DeviceArray
    rows = len(off) - 1
    token, lp, err = D.zeros(rows, np.int32), D.zeros(rows, np.float32), D.zeros(1, np.int32)
    dev.sample_candidates(D.from_host(flat), D.from_host(cand), D.from_host(off.astype(np.uint32)), most,
                          D.from_host(u), token, logprob=lp, err=err, **{k: D.from_host(v) for k, v in f.items()})
    dev.synchronize()
    return token.host(), lp.host(), int(err.host()[0])


@pytest.mark.parametrize("most", [1, 5, 1000, 4097, 33000])
def test_candidate_lists(dev, most):
    rng = np.random.default_rng(most)
    rows = 30
    lens = rng.integers(0, most + 1, size=rows)
    lens[3], lens[7] = most, 0
    off = np.concatenate([[0], np.cumsum(lens)])
    total = int(off[-1])
    flat = (2 * rng.standard_normal(total)).astype(np.float32)
    cand = np.cumsum(rng.integers(1, 9, size=total)).astype(np.uint32)
    u = rng.random(rows).astype(np.float32)
    f = settings(rng, rows)
    token, lp, err = run_candidates(dev, flat, cand, off, most, u, **f)
    assert err == 0
    places = np.full(rows, -1)
    for m in range(rows):
        if lens[m] == 0:
            assert token[m] == -1 and lp[m] == -np.inf
        else:
            places[m] = int(np.searchsorted(cand[off[m]:off[m + 1]], token[m]))
            assert cand[off[m] + places[m]] == token[m]
    agree(places, lp, [flat[off[m]:off[m + 1]] for m in range(rows)], u, **f)


def test_bad_candidate_offsets(dev):
    flat = np.zeros(20, np.float32)
    cand = np.arange(100, 120).astype(np.uint32)
    u = np.full(3, 0.99, np.float32)
    token, _, err = run_candidates(dev, flat, cand, np.array([0, 10, 4, 8]), 10, u)
    assert err == 1 and token[0] == 109 and token[1] == -1 and token[2] == 107
    token, _, err = run_candidates(dev, flat, cand, np.array([0, 10, 20, 20]), 8, u)  # lists longer than said
    assert err == 1 and token[0] == 107 and token[1] == 117 and token[2] == -1


def test_same_result_by_itself_and_in_a_batch(dev):
    rng = np.random.default_rng(9)
    l = (2 * rng.standard_normal((40, 9000))).astype(np.float32)
    u = rng.random(40).astype(np.float32)
    f = settings(rng, 40)
    token, lp, _ = draw(dev, l, u, **f)
    again = draw(dev, l, u, **f)
    assert np.array_equal(token, again[0]) and np.array_equal(lp, again[1])
    for m in (0, 17, 39):
        t1, p1, _ = draw(dev, l[m:m + 1], u[m:m + 1], **{k: v[m:m + 1] for k, v in f.items()})
        assert t1[0] == token[m] and p1[0] == lp[m]


def test_captured_graph(pkg, dev):
    rows, n = 8, 32000
    rng = np.random.default_rng(3)
    D = dev.DeviceArray
    p = np.full(rows, 0.9, np.float32)
    dl, du, dp = D.zeros((rows, n), np.float32), D.zeros(rows, np.float32), D.from_host(p)
    token, lp = D.zeros(rows, np.int32), D.zeros(rows, np.float32)
    dev.synchronize()
    stream = dev.Stream()
    graph = Graph(pkg._lib.load(), stream.handle,
                  lambda s: dev.sample_logits(dl, du, token, top_p=dp, logprob=lp, stream=s))
    for _ in range(4):
        l, u = rng.standard_normal((rows, n)).astype(np.float32), rng.random(rows).astype(np.float32)
        dev.copy(dl, D.from_host(l))
        dev.copy(du, D.from_host(u))
        dev.synchronize()
        graph.launch(stream.handle)
        stream.sync()
        agree(token.host(), lp.host(), l, u, top_p=p)
    graph.close()
    stream.close()


@pytest.mark.parametrize("n", [4097, 32000, 40000])
def test_top_k_around_the_threads_of_a_row(dev, n):
    """A top-k too long for the list: on its own up to 1024 ids, with top-p and min-p, ties at the border."""
    print(f"sample top-k n={n}", flush=True)
    rng = np.random.default_rng(n)
    ks = [193, 255, 256, 257, 600, 1000, 1023, 1024, 1025, 2000, n - 1, n]
    for kind in ("normal", "bf16", "two", "flat", "masked"):
        rows = 3 * len(ks)
        l = values_of(kind, rng, rows, n)
        u = rng.random(rows).astype(np.float32)
        f = dict(temperature=np.full(rows, 1.1, np.float32), top_k=np.repeat(ks, 3).astype(np.int32),
                 top_p=np.tile([1, 0.9, 0.6], len(ks)).astype(np.float32), min_p=np.tile([0, 0, 0.02], len(ks)).astype(np.float32))
        token, lp, err = draw(dev, l, u, **f)
        assert err == 0
        agree(token, lp, l, u, **f)
