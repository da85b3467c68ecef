"""marian_hip_q8_linear_lora against the layer and its adapters in 64 bits."""

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


def inputs(rng, M, K, N, R, slots, runs=1):
    c = dict(x=rng.standard_normal((M, K)).astype(np.float32),
             w=rng.integers(-127, 128, size=(N, K)).astype(np.int8),
             mult=rng.uniform(500, 1500, size=N).astype(np.float32), bias=rng.standard_normal(N).astype(np.float32),
             scale=rng.uniform(-2, 2, size=slots).astype(np.float32),
             rank=rng.integers(0, R + 1, size=slots).astype(np.int32))
    c["rank"][0] = R
    c["la_bits"], c["la"] = dso.to_bf16((rng.standard_normal((slots, R, K)) / np.sqrt(K)).astype(np.float32))
    c["lb_bits"], c["lb"] = dso.to_bf16(rng.standard_normal((slots, N, R)).astype(np.float32))
    s = np.repeat(rng.integers(-1, slots, size=-(-M // runs)), runs)[:M]
    c["slot"] = s.astype(np.int32)
    return c


def run(dev, c, relu=False, quantized=True, pad=2, workspace=None):
    D = dev.DeviceArray
    M, N = c["x"].shape[0], c["w"].shape[0]
    out, err = D((M + pad, N), np.float32), D.zeros(1, np.int32)
    out.fill_bytes(0x5A)
    f = {k: D.from_host(c[k]) for k in ("x", "w", "mult", "bias", "la_bits", "lb_bits", "scale", "rank", "slot")}
    q = a = None
    if quantized:
        hq, ha = dso.quantize_rows(c["x"])
        q, a = D.from_host(hq), D.from_host(ha)
    dev.q8_linear_lora(f["x"], f["w"], f["mult"], f["bias"], f["la_bits"], f["lb_bits"], f["scale"], f["rank"],
                       f["slot"], out, relu=relu, xq=q, xa=a, workspace=workspace, err=err)
    dev.synchronize()
    got = out.host()
    assert (got[M:].view(np.uint8) == 0x5A).all(), "rows behind the last one"
    return got[:M], int(err.host()[0])


def check(got, c, relu=False):
    q, a = dso.quantize_rows(c["x"])
    want, bound = dso.lora(c["x"], q, a, c["w"], c["mult"], c["bias"], c["la"], c["lb"], c["scale"], c["rank"],
                           c["slot"], relu)
    off = np.abs(got - want)
    assert (off <= bound).all(), (float((off - bound).max()), np.argwhere(off > bound)[:4].tolist())
    # Rounding errors of sums add up like random steps: about sqrt(K) + sqrt(R) of them; 24-bit operands stay below this
    K, R = c["x"].shape[1], c["la"].shape[1]
    rel = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert rel <= 2.0 ** -24 * (8 + np.sqrt(K) + np.sqrt(R)), rel


SHAPES = [  # M, K, N, R, slots, run length
    (1, 64, 1, 8, 1, 1), (1, 512, 2048, 8, 4, 1), (2, 128, 33, 16, 2, 1), (7, 192, 100, 24, 3, 1),
    (15, 512, 512, 16, 16, 1), (16, 512, 129, 64, 5, 1), (17, 320, 64, 40, 9, 1), (31, 64, 2048, 8, 31, 1),
    (33, 1536, 384, 64, 7, 3), (61, 512, 1536, 16, 64, 1), (64, 2048, 512, 128, 3, 5), (65, 512, 300, 32, 4, 9),
    (127, 704, 1000, 56, 6, 20), (129, 512, 2300, 16, 8, 1), (200, 1536, 384, 64, 24, 1), (256, 512, 2048, 128, 40, 1),
    (257, 384, 1536, 8, 300, 1), (700, 512, 512, 16, 5, 33), (1459, 512, 2048, 16, 32, 25), (2100, 384, 1152, 48, 9, 1),
    (3000, 64, 70, 8, 20, 100),
    # one launch from codes and from rows, on both column widths and row lengths
    (1, 2048, 512, 16, 3, 1), (2, 1536, 2300, 16, 2, 1), (1, 1088, 1025, 32, 2, 1), (4, 640, 1030, 16, 4, 1),
    (8, 512, 1000, 8, 5, 1), (16, 256, 1027, 8, 9, 1),
    # few rows past the registers' row pieces, every group of ranks
    (9, 2560, 300, 128, 4, 1), (40, 2112, 1100, 16, 6, 1), (320, 4096, 96, 24, 30, 1), (18, 960, 2050, 72, 4, 1),
    # many rows: one, two and four tiles of ranks a workgroup, long rows, ranks over several workgroups
    (321, 2048, 520, 64, 4, 40), (340, 1088, 200, 128, 3, 50), (4100, 512, 64, 32, 7, 60), (4099, 64, 128, 64, 3, 1),
    (8200, 192, 96, 64, 6, 100), (8195, 128, 65, 128, 4, 300), (4097, 1152, 70, 128, 5, 90),
    # rows by themselves up to 1024, tiles before and after
    (321, 512, 512, 16, 9, 1), (1024, 512, 512, 16, 20, 1), (1025, 512, 512, 16, 20, 3), (1024, 64, 2300, 8, 7, 2),
    (818, 2048, 512, 16, 5, 4), (1000, 2048, 512, 16, 5, 4),
    # tiles of 128 columns
    (4100, 128, 1000, 16, 6, 70), (4101, 192, 900, 24, 8, 1), (4102, 128, 897, 48, 5, 33),
]


@pytest.mark.parametrize("M, K, N, R, slots, runs", SHAPES)
def test_shapes(dev, M, K, N, R, slots, runs):
    print(f"lora M={M} K={K} N={N} R={R} slots={slots} runs={runs}", flush=True)
    c = inputs(np.random.default_rng(M + N), M, K, N, R, slots, runs)
    relu, quantized = bool(M % 2), bool(N % 3)
    got, err = run(dev, c, relu, quantized)
    assert err == 0
    check(got, c, relu)
    again, _ = run(dev, c, relu, quantized)
    assert np.array_equal(got, again), "the same call twice"


@pytest.mark.parametrize("M", [1, 5, 64, 300, 1500])
def test_without_adapters_it_is_the_shared_layer(dev, M):
    rng = np.random.default_rng(M)
    c = inputs(rng, M, 512, 700, 16, 2)
    c["slot"][:] = -1
    D = dev.DeviceArray
    for relu in (False, True):
        got, err = run(dev, c, relu)
        q, a = dso.quantize_rows(c["x"])
        plain = D.zeros((M, 700), np.float32)
        dev.q8_linear(None, D.from_host(c["w"]), D.from_host(c["mult"]), D.from_host(c["bias"]), None, plain, relu=relu,
                      xq=D.from_host(q), xa=D.from_host(a))
        dev.synchronize()
        assert err == 0 and np.array_equal(got, plain.host())


@pytest.mark.parametrize("M", [3, 40, 300, 1200])
def test_rows_do_not_touch_each_other(dev, M):
    """A broken adapter (infinite, NaN) and unused places of the tables reach no other request's rows."""
    rng = np.random.default_rng(M)
    c = inputs(rng, M, 256, 320, 16, 6)
    c["rank"][:] = [16, 5, 0, 16, 11, 16]
    c["slot"][:3] = [3, 0, 1]
    bad = dso.to_bf16(np.array([np.inf, np.nan], np.float32))[0]
    for name in ("la_bits", "lb_bits"):
        c[name][3] = bad[0] if name == "la_bits" else bad[1]
    for s, r in enumerate(c["rank"]):  # past the rank
        c["la_bits"][s, r:] = bad[1]
        c["lb_bits"][s, :, r:] = bad[0]
    got, err = run(dev, c, pad=5)
    assert err == 0
    good = c["slot"] != 3
    assert not np.isfinite(got[~good]).any()
    part = dict(c, x=c["x"][good], slot=c["slot"][good])
    check(got[good], part)


def test_slots_and_ranks_out_of_range(dev):
    for M in (4, 70, 900):
        c = inputs(np.random.default_rng(M), M, 128, 96, 8, 3)
        c["rank"][:] = [8, 9, -1]
        c["slot"][:4] = [0, 1, 2, 3]
        c["slot"][4:] = 0
        got, err = run(dev, c)
        assert err == 1
        c["slot"][1:4] = -1
        check(got, c)
        got, err = run(dev, c)
        assert err == 0


@pytest.mark.parametrize("M", [5, 100, 800])
def test_large_and_small_values(dev, M):
    """Rows of very different sizes: every bit of x counts, tiny values included."""
    rng = np.random.default_rng(M)
    c = inputs(rng, M, 512, 256, 32, 4)
    c["x"] *= np.exp(rng.uniform(-20, 20, size=(M, 1))).astype(np.float32)
    c["x"][:, ::5] *= np.float32(1e-4)
    got, err = run(dev, c)
    assert err == 0
    q, a = dso.quantize_rows(c["x"])
    want, bound = dso.lora(c["x"], q, a, c["w"], c["mult"], c["bias"], c["la"], c["lb"], c["scale"], c["rank"], c["slot"])
    assert (np.abs(got - want) <= bound).all()


def test_output_over_the_input(dev):
    D = dev.DeviceArray
    for M in (3, 64, 700):
        c = inputs(np.random.default_rng(M), M, 512, 512, 16, 4)
        f = {k: D.from_host(c[k]) for k in ("x", "w", "mult", "bias", "la_bits", "lb_bits", "scale", "rank", "slot")}
        dev.q8_linear_lora(f["x"], f["w"], f["mult"], f["bias"], f["la_bits"], f["lb_bits"], f["scale"], f["rank"],
                           f["slot"], f["x"])
        dev.synchronize()
        check(f["x"].host(), c)


@pytest.mark.parametrize("M", [1, 80, 600])
def test_non_finite_rows_set_err(dev, M):
    c = inputs(np.random.default_rng(M), M, 128, 64, 8, 2)
    c["x"][M // 2, 5] = np.nan
    got, err = run(dev, c, quantized=False)
    assert err == 1
    keep = np.arange(M) != M // 2
    if keep.any():
        check(got[keep], dict(c, x=c["x"][keep], slot=c["slot"][keep]))


def test_workspace_of_the_caller(dev):
    for M, quantized in ((9, True), (9, False), (500, True), (500, False)):
        c = inputs(np.random.default_rng(M), M, 512, 384, 24, 5)
        n = dev.q8_linear_lora_workspace(M, 512, 24, quantized)
        ws = dev.DeviceArray((n + 64,), np.uint8)
        ws.fill_bytes(0x5A)
        ws.nbytes = n
        got, err = run(dev, c, quantized=quantized, workspace=ws)
        assert err == 0
        check(got, c)
        ws.nbytes = n + 64
        assert (ws.host()[n:] == 0x5A).all(), "behind the workspace"


NAMES = ("x", "w", "mult", "bias", "la_bits", "lb_bits", "scale", "rank", "slot")


@pytest.mark.parametrize("M", [6, 90, 400])
def test_streams_and_captured_graphs(pkg, dev, M):
    """Two streams at once on library scratch, then two graphs at once with a workspace each."""
    rng = np.random.default_rng(M)
    D = dev.DeviceArray
    c = inputs(rng, M, 256, 512, 16, 5)
    f = {k: D.from_host(c[k]) for k in NAMES}
    outs = [D.zeros((M, 512), np.float32) for _ in range(2)]
    wss = [D.zeros(dev.q8_linear_lora_workspace(M, 256, 16, False), np.uint8) for _ in range(2)]
    streams = [dev.Stream() for _ in range(2)]
    call = lambda o, ws, s: dev.q8_linear_lora(*(f[k] for k in NAMES), o, workspace=ws, stream=s)  # noqa: E731
    dev.synchronize()
    for o, s in zip(outs, streams):
        call(o, None, s.handle)
    dev.synchronize()
    for o in outs:
        check(o.host(), c)
    graphs = [Graph(pkg._lib.load(), s.handle, lambda h, o=o, ws=ws: call(o, ws, h))
              for o, ws, s in zip(outs, wss, streams)]
    for _ in range(3):
        c["x"] = rng.standard_normal((M, 256)).astype(np.float32)
        dev.copy(f["x"], D.from_host(c["x"]))
        for o in outs:
            o.fill_bytes(0)
        dev.synchronize()
        for g, s in zip(graphs, streams):
            g.launch(s.handle)
        dev.synchronize()
        for o in outs:
            check(o.host(), c)
    for g, s in zip(graphs, streams):
        g.close()
        s.close()


def test_capture_without_a_workspace_is_refused(pkg, dev):
    c = inputs(np.random.default_rng(0), 4, 64, 64, 8, 2)
    D = dev.DeviceArray
    f = {k: D.from_host(c[k]) for k in NAMES}
    out, other = D.zeros((4, 64), np.float32), D.zeros(4, np.float32)
    q = D.zeros((4, 64), np.int8)
    dev.synchronize()
    stream = dev.Stream()

    def call(s):
        dev.quantize_rows(f["x"], q, other, stream=s)
        with pytest.raises(RuntimeError, match="workspace"):
            dev.q8_linear_lora(*(f[k] for k in NAMES), out, stream=s)

    graph = Graph(pkg._lib.load(), stream.handle, call)
    graph.launch(stream.handle)
    stream.sync()
    assert np.array_equal(q.host(), dso.quantize_rows(c["x"])[0]) and not out.host().any()
    graph.close()
    stream.close()
