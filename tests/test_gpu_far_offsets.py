"""The decode-step operators (RMS norm, adapter layer, sampling) on tensors whose offsets pass 32 bits, and on more
rows than a launch has workgroups.  Buffers are zero but for the rows looked at."""

import numpy as np
import pytest

import decode_step_oracle as dso

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    from importlib import import_module

    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


class At:
    """A view of a device buffer: an address past its start, with a shape."""

    def __init__(self, base, offset, shape):
        self.base, self.ptr, self.shape = base, base.ptr + offset, shape


def put(dev, base, at, a):
    """a's bytes at byte `at` of a device buffer."""
    src = dev.DeviceArray.from_host(a)
    assert at + src.nbytes <= base.nbytes
    dst = At(base, at, a.shape)
    dst.nbytes = src.nbytes
    dev.copy(dst, src)


def get(dev, base, at, shape, dtype):
    out = dev.DeviceArray(shape, dtype)
    src = At(base, at, shape)
    src.nbytes = out.nbytes
    assert at + src.nbytes <= base.nbytes
    dev.copy(out, src)
    dev.synchronize()
    return out.host()


def check_norm(s, out, q, a, want):
    assert np.array_equal(s.view(np.uint32), want[0].view(np.uint32))
    assert (np.abs(out - want[1]) <= np.abs(want[1]) * (2.0 ** -24 + 1e-12) + 2.0 ** -150).all()
    want_q, want_a = dso.quantize_rows(out)
    assert np.array_equal(a, want_a) and np.array_equal(q, want_q)


def test_norm_rows_far_apart(dev):
    rows, dim, ld = 5, 515, 1 << 29  # the last row begins at value 2^31
    rng = np.random.default_rng(1)
    x, scale = rng.standard_normal((rows, dim)).astype(np.float32), rng.standard_normal(dim).astype(np.float32)
    D = dev.DeviceArray
    base = D(((rows - 1) * ld + dim,), np.float32)
    for m in range(rows):
        put(dev, base, m * ld * 4, x[m])
    s, out, q, a = D((rows, dim), np.float32), D((rows, dim), np.float32), D((rows, dim), np.int8), D(rows, np.float32)
    dev.residual_rms_norm(At(base, 0, (rows, dim)), None, D.from_host(scale), 1e-6, total=s, out=out, q=q, a=a, ldx=ld)
    dev.synchronize()
    check_norm(s.host(), out.host(), q.host(), a.host(), dso.rms_norm(x, None, scale, 1e-6))


def test_norm_of_more_short_rows_than_workgroups(dev):
    rows, dim = (4 << 20) + 9, 4
    rng = np.random.default_rng(2)
    x, scale = rng.standard_normal((rows, dim)).astype(np.float32), rng.standard_normal(dim).astype(np.float32)
    D = dev.DeviceArray
    out, q, a = D((rows, dim), np.float32), D((rows, dim), np.int8), D(rows, np.float32)
    dev.residual_rms_norm(D.from_host(x), None, D.from_host(scale), 1e-6, out=out, q=q, a=a)
    dev.synchronize()
    check_norm(x, out.host(), q.host(), a.host(), dso.rms_norm(x, None, scale, 1e-6))


def test_norm_of_more_long_rows_than_workgroups(dev):
    rows, dim = (1 << 20) + 5, 1027
    rng = np.random.default_rng(3)
    scale = rng.standard_normal(dim).astype(np.float32)
    D = dev.DeviceArray
    x, q, a = D.zeros((rows, dim), np.uint16), D((rows, dim), np.int8), D(rows, np.float32)
    some = [0, 1, 77, 4, (1 << 20) - 1, 1 << 20, (1 << 20) + 4]
    bits, v = dso.to_bf16(rng.standard_normal((len(some), dim)).astype(np.float32))
    for m, b in zip(some, bits):
        put(dev, x, m * dim * 2, b)
    dev.residual_rms_norm(x, None, D.from_host(scale), 1e-6, q=q, a=a, bf16=True)
    dev.synchronize()
    got_q = np.stack([get(dev, q, m * dim, (dim,), np.int8) for m in some])
    want_q, want_a = dso.quantize_rows(dso.rms_norm(v, None, scale, 1e-6)[1].astype(np.float32))
    got_a = a.host()
    assert np.array_equal(got_q, want_q) and np.array_equal(got_a[some], want_a)
    rest = np.ones(rows, bool)
    rest[some] = False
    assert (got_a[rest] == 1.0).all()
    assert not get(dev, q, ((1 << 20) + 1) * dim, (3, dim), np.int8).any()


@pytest.mark.parametrize("n", [1000, 20000, 40001])
def test_sampling_rows_far_apart(dev, n):
    rows, ld = 9, 1 << 29  # the last row begins at value 2^32
    rng = np.random.default_rng(n)
    bits, v = dso.to_bf16((2 * rng.standard_normal((rows, n))).astype(np.float32))
    u = rng.random(rows).astype(np.float32)
    p = np.full(rows, 0.9, np.float32)
    D = dev.DeviceArray
    base = D(((rows - 1) * ld + n,), np.uint16)
    for m in range(rows):
        put(dev, base, m * ld * 2, bits[m])
    token = D.zeros(rows, np.int32)
    dev.sample_logits(At(base, 0, (rows, ld)), D.from_host(u), token, top_p=D.from_host(p), bf16=True, ids=n)
    dev.synchronize()
    assert token.host().tolist() == [dso.sample(v[m], u=u[m], top_p=p[m])[0] for m in range(rows)]


def test_candidate_lists_far_from_the_start(dev):
    first = (1 << 31) + 5
    lens = np.array([400, 0, 7, 1500])
    off = (first + np.concatenate([[0], np.cumsum(lens)])).astype(np.uint32)
    total = int(lens.sum())
    rng = np.random.default_rng(4)
    logits = rng.standard_normal(total).astype(np.float32)
    cand = np.cumsum(rng.integers(1, 5, size=total)).astype(np.uint32)
    u = rng.random(4).astype(np.float32)
    D = dev.DeviceArray
    dl, dc = D((first + total,), np.float32), D((first + total,), np.uint32)
    put(dev, dl, first * 4, logits)
    put(dev, dc, first * 4, cand)
    token, err = D.zeros(4, np.int32), D.zeros(1, np.int32)
    dev.sample_candidates(dl, dc, D.from_host(off), 1500, D.from_host(u), token, err=err)
    dev.synchronize()
    at = np.concatenate([[0], np.cumsum(lens)])
    want = [-1 if lens[m] == 0 else int(cand[at[m] + dso.sample(logits[at[m]:at[m + 1]], u=u[m])[0]]) for m in range(4)]
    assert err.host()[0] == 0 and token.host().tolist() == want


@pytest.mark.parametrize("M", [3, 40, 400])
def test_adapters_far_into_the_tables(dev, M):
    K, N, R, slots = 256, 300, 8, 1 << 20  # the last slots' weights lie past value 2^31
    used = [0, 1, (1 << 19) + 3, slots - 2, slots - 1]
    rng = np.random.default_rng(M)
    x = rng.standard_normal((M, K)).astype(np.float32)
    w = rng.integers(-127, 128, size=(N, K)).astype(np.int8)
    mult, bias = rng.uniform(500, 1500, size=N).astype(np.float32), rng.standard_normal(N).astype(np.float32)
    a_bits, a = dso.to_bf16((rng.standard_normal((len(used), R, K)) / 16).astype(np.float32))
    b_bits, b = dso.to_bf16(rng.standard_normal((len(used), N, R)).astype(np.float32))
    pick = rng.integers(0, len(used), size=M)
    scale, rank = np.ones(slots, np.float32), np.zeros(slots, np.int32)
    rank[used] = [8, 3, 8, 7, 8]
    D = dev.DeviceArray
    da, db = D((slots, R, K), np.uint16), D((slots, N, R), np.uint16)
    for i, s in enumerate(used):
        put(dev, da, s * R * K * 2, a_bits[i])
        put(dev, db, s * N * R * 2, b_bits[i])
    out, err = D((M, N), np.float32), D.zeros(1, np.int32)
    dev.q8_linear_lora(D.from_host(x), D.from_host(w), D.from_host(mult), D.from_host(bias), da, db, D.from_host(scale),
                       D.from_host(rank), D.from_host(np.array(used)[pick].astype(np.int32)), out, err=err)
    dev.synchronize()
    q, am = dso.quantize_rows(x)
    want, bound = dso.lora(x, q, am, w, mult, bias, a, b, scale[used], rank[used], pick)
    assert err.host()[0] == 0 and (np.abs(out.host() - want) <= bound).all()


def test_adapter_layer_of_very_many_rows(dev):
    M, K, N, R = (1 << 23) + 77, 256, 24, 16  # x passes value 2^31
    some = np.array([0, 5, 31, 32, 1 << 22, (1 << 23) - 1, 1 << 23, M - 33, M - 1])
    rng = np.random.default_rng(5)
    x = rng.standard_normal((len(some), K)).astype(np.float32)
    w = rng.integers(-127, 128, size=(N, K)).astype(np.int8)
    mult, bias = rng.uniform(500, 1500, size=N).astype(np.float32), rng.standard_normal(N).astype(np.float32)
    a_bits, a = dso.to_bf16((rng.standard_normal((3, R, K)) / 16).astype(np.float32))
    b_bits, b = dso.to_bf16(rng.standard_normal((3, N, R)).astype(np.float32))
    slot = np.full(M, 1, np.int32)
    slot[some] = [0, 1, 2, 0, 1, 2, 0, -1, 2]
    scale, rank = np.array([1, -2, 0.5], np.float32), np.array([16, 9, 16], np.int32)
    D = dev.DeviceArray
    dx = D.zeros((M, K), np.float32)
    for m, v in zip(some, x):
        put(dev, dx, int(m) * K * 4, v)
    out, err = D((M, N), np.float32), D.zeros(1, np.int32)
    dev.q8_linear_lora(dx, D.from_host(w), D.from_host(mult), D.from_host(bias), D.from_host(a_bits), D.from_host(b_bits),
                       D.from_host(scale), D.from_host(rank), D.from_host(slot), out, err=err)
    dev.synchronize()
    got = out.host()
    q, am = dso.quantize_rows(x)
    want, bound = dso.lora(x, q, am, w, mult, bias, a, b, scale, rank, slot[some])
    assert err.host()[0] == 0 and (np.abs(got[some] - want) <= bound).all()
    rest = np.ones(M, bool)
    rest[some] = False
    assert (got[rest] == bias).all(), "rows of zeros"
