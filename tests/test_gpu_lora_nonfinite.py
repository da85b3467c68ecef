"""marian_hip_q8_linear_lora with values that are not finite in a row's own adapter, or in the row: what the definition
gives, in those rows alone."""

import numpy as np
import pytest

import decode_step_oracle as dso
from test_gpu_lora import dev, inputs, run  # noqa: F401 (dev: the fixture)

pytestmark = pytest.mark.gpu

SHAPES = [  # M, K, N, R: one launch, a row at a time (row pieces in registers or not), tiles of 64 and of 128 columns
    (3, 192, 100, 8), (2, 1088, 1030, 16), (40, 192, 100, 16), (40, 704, 1100, 40), (30, 2112, 96, 24),
    (1200, 192, 100, 16), (1200, 320, 130, 32), (1100, 1088, 70, 72), (4100, 128, 1000, 16), (4102, 192, 897, 48),
]


def broken(M, K, N, R):
    """Slot 0 sound, slots 1 to 3 to be broken; x of 8 bits, slot 1's and 2's first rank takes one value of x as it is:
    the lower parts of a split operand are zero."""
    c = inputs(np.random.default_rng(M + K), M, K, N, R, 4)
    c["x"] = dso.to_bf16(c["x"])[1].copy()
    c["rank"][:] = [R, R, 1, R - 1]
    c["slot"] = np.random.default_rng(M).integers(-1, 4, size=M).astype(np.int32)
    c["slot"][:2] = [1, 2]
    c["scale"][:] = [1.5, 1.0, -1.0, 0.5]
    for s in (1, 2):
        c["la"][s, 0] = 0.0
        c["la"][s, 0, 7] = 1.0
        c["la_bits"][s] = dso.to_bf16(c["la"][s])[0]
    return c


def put(c, name, at, value):
    bits, v = dso.to_bf16(np.array([value], np.float32))
    c[name + "_bits"][at] = bits[0]
    c[name][at] = v[0]


def agree(got, c, x, relu):
    q, a = dso.quantize_rows(c["x"])
    with np.errstate(invalid="ignore"):
        want, bound = dso.lora(x, q, a, c["w"], c["mult"], c["bias"], c["la"], c["lb"], c["scale"], c["rank"], c["slot"],
                               relu)
    sound = np.isfinite(bound)  # the rest: not finite, or an infinity that relu took to zero
    assert np.isfinite(want[sound]).all() and (np.abs(got[sound] - want[sound]) <= bound[sound]).all()
    assert not sound.all() and np.array_equal(got[~sound], want[~sound], equal_nan=True)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("M, K, N, R", SHAPES)
def test_nan_in_an_adapter(dev, M, K, N, R, relu):
    print(f"lora NaN M={M} K={K} N={N} R={R} relu={relu}", flush=True)
    c = broken(M, K, N, R)
    put(c, "la", (3, R - 2, K - 3), np.nan)  # A: in the last eight columns
    put(c, "la", (1, R - 1, 5), np.nan)
    put(c, "lb", (2, 3, 0), np.nan)  # B: one output
    got, err = run(dev, c, relu)
    assert err == 0
    agree(got, c, c["x"], relu)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
@pytest.mark.parametrize("M, K, N, R", SHAPES)
def test_infinity_in_an_adapter(dev, M, K, N, R, value, relu):
    print(f"lora infinity M={M} K={K} N={N} R={R} {value} relu={relu}", flush=True)
    c = broken(M, K, N, R)
    put(c, "la", (3, R - 2, K - 3), value)
    put(c, "la", (1, R - 1, 5), value)
    got, err = run(dev, c, relu)
    assert err == 0
    agree(got, c, c["x"], relu)
    c = broken(M, K, N, R)
    put(c, "lb", (1, N - 1, 0), value)
    put(c, "lb", (2, 3, 0), value)
    put(c, "lb", (3, N // 2, R - 2), value)
    got, err = run(dev, c, relu)
    assert err == 0
    agree(got, c, c["x"], relu)


@pytest.mark.parametrize("M, K, N, R", SHAPES)
def test_a_broken_row(dev, M, K, N, R):
    """A row that is not finite, its codes given: its own adapter's product takes it up, no other row does."""
    print(f"lora non-finite rows M={M} K={K} N={N} R={R}", flush=True)
    D = dev.DeviceArray
    c = broken(M, K, N, R)
    x = c["x"].copy()
    x[0, 7], x[1, 7] = np.inf, -np.inf
    if M > 2:
        x[2, 9] = np.nan
    q, a = dso.quantize_rows(c["x"])
    out = D.zeros((M, N), np.float32)
    f = {k: D.from_host(c[k]) for k in ("w", "mult", "bias", "la_bits", "lb_bits", "scale", "rank", "slot")}
    dev.q8_linear_lora(D.from_host(x), f["w"], f["mult"], f["bias"], f["la_bits"], f["lb_bits"], f["scale"], f["rank"],
                       f["slot"], out, xq=D.from_host(q), xa=D.from_host(a))
    dev.synchronize()
    agree(out.host(), c, x, False)
