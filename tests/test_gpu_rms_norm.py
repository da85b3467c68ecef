"""marian_hip_residual_rms_norm against its definition in 64 bits."""

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
    """A view of a device buffer: an address past its start, with a shape."""

    def __init__(self, base, offset, shape):
        self.base, self.ptr, self.shape = base, base.ptr + offset, shape


def check(s, out, q, a, want_s, want_y):
    assert np.array_equal(s.view(np.uint32), want_s.view(np.uint32)), "residual sum"
    # rounded once to fp32, from 64-bit sums whose own error is below 1e-12
    assert (np.abs(out - want_y) <= np.abs(want_y) * (2.0 ** -24 + 1e-12) + 2.0 ** -150).all(), "norm"
    want_q, want_a = dso.quantize_rows(out)
    assert np.array_equal(a, want_a) and np.array_equal(q, want_q), "codes"


def case(rng, rows, dim, ldx, ldr, residual, bf16):
    x = (rng.standard_normal((rows, ldx)) * np.exp(rng.standard_normal(ldx))).astype(np.float32)
    r = rng.standard_normal((rows, ldr)).astype(np.float32) if residual else None
    scale = (1 + 0.2 * rng.standard_normal(dim)).astype(np.float32)
    if bf16:
        xh, x = dso.to_bf16(x)
        rh, r = dso.to_bf16(r) if residual else (None, None)
        return x, r, scale, xh, rh
    return x, r, scale, x, r


DIMS = [1, 2, 3, 4, 5, 63, 64, 65, 255, 256, 257, 384, 512, 513, 1000, 1024, 1025, 2048, 2049, 4096, 4100, 5000, 6001,
        6144, 8192, 8195, 12287, 12289, 16383, 16384]


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("dim", DIMS)
def test_widths(dev, dim, bf16, residual):
    rows = 7
    print(f"rms norm dim={dim} bf16={bf16} residual={residual}", flush=True)
    rng = np.random.default_rng(dim)
    x, r, scale, dx, dr = case(rng, rows, dim, dim, dim, residual, bf16)
    D = dev.DeviceArray
    s, out, q, a = D((rows + 1, dim), np.float32), D((rows + 1, dim), np.float32), D((rows + 1, dim), np.int8), D(rows + 1, np.float32)
    for b in (s, out, q, a):
        b.fill_bytes(0x5A)
    err = D.zeros(1, np.int32)
    dev.residual_rms_norm(D.from_host(dx), D.from_host(dr) if residual else None, D.from_host(scale), 1e-6, total=s,
                          out=out, q=q, a=a, bf16=bf16, err=err)
    dev.synchronize()
    assert err.host()[0] == 0
    want_s, want_y = dso.rms_norm(x, r, scale, 1e-6)
    check(s.host()[:rows], out.host()[:rows], q.host()[:rows], a.host()[:rows], want_s, want_y)
    for b in (s, out, q, a):  # the row behind the last one
        assert (b.host()[rows:].view(np.uint8) == 0x5A).all()


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 64, 1459, 7405])
def test_row_counts(dev, rows):
    rng = np.random.default_rng(rows)
    x, r, scale, dx, dr = case(rng, rows, 512, 512, 512, True, False)
    D = dev.DeviceArray
    s, out, q, a = D.zeros((rows, 512), np.float32), D.zeros((rows, 512), np.float32), D.zeros((rows, 512), np.int8), D.zeros(rows, np.float32)
    dev.residual_rms_norm(D.from_host(dx), D.from_host(dr), D.from_host(scale), 1e-6, total=s, out=out, q=q, a=a)
    dev.synchronize()
    check(s.host(), out.host(), q.host(), a.host(), *dso.rms_norm(x, r, scale, 1e-6))
    q2, a2 = D.zeros((rows, 512), np.int8), D.zeros(rows, np.float32)
    dev.quantize_rows(out, q2, a2)
    dev.synchronize()
    assert np.array_equal(q.host(), q2.host()) and np.array_equal(a.host(), a2.host()), "quantize_rows of out"


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("dim, ldx, ldr, off", [(512, 1536, 520, 0), (512, 515, 513, 1), (100, 101, 100, 3),
                                                (1500, 1504, 2000, 1), (6000, 6004, 6001, 2), (3, 5, 4, 1), (4099, 4101, 4103, 3)])
def test_strides_and_addresses(dev, dim, ldx, ldr, off, bf16):
    rows, size = 9, 2 if bf16 else 4
    rng = np.random.default_rng(dim + off)
    x, r, scale, dx, dr = case(rng, rows + 1, dim, ldx, ldr, True, bf16)
    D = dev.DeviceArray
    bx, br = D.from_host(dx), D.from_host(dr)
    s, out, q, a = D.zeros((rows, dim), np.float32), D.zeros((rows, dim), np.float32), D.zeros((rows, dim), np.int8), D.zeros(rows, np.float32)
    dev.residual_rms_norm(At(bx, off * size, (rows, dim)), At(br, off * size, (rows, dim)), D.from_host(scale), 1e-6,
                          total=s, out=out, q=q, a=a, bf16=bf16, ldx=ldx, ldr=ldr)
    dev.synchronize()
    view = lambda t, ld: np.ascontiguousarray(  # noqa: E731
        np.lib.stride_tricks.as_strided(t.reshape(-1)[off:], (rows, dim), (4 * ld, 4)))
    check(s.host(), out.host(), q.host(), a.host(), *dso.rms_norm(view(x, ldx), view(r, ldr), scale, 1e-6))


@pytest.mark.parametrize("dim", [1, 3, 7, 384, 1001, 2000, 5003, 7997, 10000, 10001])
def test_optional_outputs_and_in_place(dev, dim):
    rows = 33
    rng = np.random.default_rng(dim)
    x, r, scale, _, _ = case(rng, rows, dim, dim, dim, True, False)
    want_s, want_y = dso.rms_norm(x, r, scale, 1e-5)
    D = dev.DeviceArray
    dsc = D.from_host(scale)
    out = D.zeros((rows, dim), np.float32)
    dev.residual_rms_norm(D.from_host(x), D.from_host(r), dsc, 1e-5, out=out)
    q, a = D.zeros((rows, dim), np.int8), D.zeros(rows, np.float32)
    dev.residual_rms_norm(D.from_host(x), D.from_host(r), dsc, 1e-5, q=q, a=a)
    # the residual stream updated in place, the norm over the sublayer's output
    dx, dr, q2, a2 = D.from_host(x), D.from_host(r), D.zeros((rows, dim), np.int8), D.zeros(rows, np.float32)
    dev.residual_rms_norm(dx, dr, dsc, 1e-5, total=dr, out=dx, q=q2, a=a2)
    dev.synchronize()
    check(dr.host(), dx.host(), q2.host(), a2.host(), want_s, want_y)
    assert np.array_equal(out.host(), dx.host()) and np.array_equal(q.host(), q2.host()) and np.array_equal(a.host(), a2.host())


def test_zero_rows_large_values_and_non_finite(dev):
    D = dev.DeviceArray
    dim = 300
    x = np.zeros((6, dim), np.float32)
    x[1] = 3e38   # squares beyond fp32's range
    x[2] = 1e-30  # and below it: eps rules
    x[3, 7] = np.inf
    x[4, 8] = np.nan
    x[5] = np.linspace(-1, 1, dim)
    scale = np.ones(dim, np.float32)
    for rows, bad in (((0, 1, 2, 5), 0), ((3,), 1), ((4,), 1)):
        z = np.ascontiguousarray(x[list(rows)])
        out, q, a = D.zeros(z.shape, np.float32), D.zeros(z.shape, np.int8), D.zeros(len(z), np.float32)
        err = D.zeros(1, np.int32)
        dev.residual_rms_norm(D.from_host(z), None, D.from_host(scale), 1e-6, out=out, q=q, a=a, err=err)
        dev.synchronize()
        assert err.host()[0] == bad
        if not bad:
            s, y = dso.rms_norm(z, None, scale, 1e-6)
            check(s, out.host(), q.host(), a.host(), s, y)
            assert a.host()[0] == 1.0 and not q.host()[0].any()


def test_another_stream_and_a_captured_graph(pkg, dev):
    rows, dim = 100, 512
    rng = np.random.default_rng(8)
    D = dev.DeviceArray
    r, scale = (rng.standard_normal(n).astype(np.float32) for n in ((rows, dim), dim))
    dx, dr, dsc = D.zeros((rows, dim), np.float32), D.from_host(r), D.from_host(scale)
    out, q, a = D.zeros((rows, dim), np.float32), D.zeros((rows, dim), np.int8), D.zeros(rows, np.float32)
    dev.synchronize()
    stream = dev.Stream()
    graph = Graph(pkg._lib.load(), stream.handle,
                  lambda s: dev.residual_rms_norm(dx, dr, dsc, 1e-6, out=out, q=q, a=a, stream=s))
    for _ in range(4):
        x = rng.standard_normal((rows, dim)).astype(np.float32)
        dev.copy(dx, D.from_host(x))
        out.fill_bytes(0)
        dev.synchronize()
        graph.launch(stream.handle)
        stream.sync()
        s, y = dso.rms_norm(x, r, scale, 1e-6)
        check(s, out.host(), q.host(), a.host(), s, y)
    graph.close()
    stream.close()
