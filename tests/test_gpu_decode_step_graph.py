"""A decode step of many requests captured into one graph: norm, adapted projections, vocabulary logits, draw.  Every
replay, on inputs of its own and with eager work between, gives the bits of the eager calls."""

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


@pytest.mark.parametrize("M, D, F, V", [(1, 512, 2048, 32000), (37, 384, 1536, 5000), (1100, 512, 2048, 8000)])
def test_captured_step(pkg, dev, M, D, F, V):
    print(f"captured decode step M={M} D={D} F={F} V={V}", flush=True)
    rng = np.random.default_rng(M)
    lib = pkg._lib.load()
    up, new = dev.DeviceArray.from_host, dev.DeviceArray.zeros
    slots, R = 6, 16
    bf16 = lambda *shape: dso.to_bf16((0.05 * rng.standard_normal(shape)).astype(np.float32))[0]  # noqa: E731
    uniform = lambda lo, hi, *shape: up(rng.uniform(lo, hi, size=shape).astype(np.float32))  # noqa: E731
    layers = [dict(w=up(rng.integers(-127, 128, size=(N, K)).astype(np.int8)), mult=uniform(500, 1500, N),
                   bias=uniform(-1, 1, N), lora_a=up(bf16(slots, R, K)), lora_b=up(bf16(slots, N, R)),
                   lora_scale=uniform(0.5, 2, slots), lora_rank=up(rng.integers(1, R + 1, size=slots).astype(np.int32)))
              for K, N in ((D, F), (F, D))]
    emb, emult, ebias = up(rng.integers(-127, 128, size=(V, D)).astype(np.int8)), uniform(2000, 4000, V), uniform(-.1, .1, V)
    gains = [uniform(0.8, 1.2, D) for _ in range(2)]
    settings = dict(temperature=up(rng.choice(np.array([0, 0.7, 1.0], np.float32), size=M)),
                    top_k=up(rng.choice(np.array([0, 5, 50], np.int32), size=M)), top_p=uniform(0.8, 1.1, M),
                    min_p=uniform(0, 0.05, M))
    x, y, slot, u = new((M, D), np.float32), new((M, D), np.float32), new(M, np.int32), new(M, np.float32)
    # the second layer makes its codes itself
    spaces = [new(dev.q8_linear_lora_workspace(M, K, R, has), np.uint8) for K, has in ((D, True), (F, False))]

    def outputs():
        f32 = lambda *shape: new(shape, np.float32)  # noqa: E731
        return dict(first=f32(M, D), h=f32(M, D), q=new((M, D), np.int8), a=f32(M), mid=f32(M, F), back=f32(M, D),
                    q2=new((M, D), np.int8), a2=f32(M), logits=f32(M, V), best=new(M, np.int32), token=new(M, np.int32),
                    lp=f32(M), err=new(1, np.int32))

    def step(o, stream, workspaces):
        dev.residual_rms_norm(x, y, gains[0], 1e-6, total=o["first"], out=o["h"], q=o["q"], a=o["a"], err=o["err"], stream=stream)
        dev.q8_linear_lora(o["h"], slot_of_row=slot, out=o["mid"], relu=True, xq=o["q"], xa=o["a"], err=o["err"],
                           workspace=workspaces[0], stream=stream, **layers[0])
        dev.q8_linear_lora(o["mid"], slot_of_row=slot, out=o["back"], err=o["err"], workspace=workspaces[1], stream=stream,
                           **layers[1])
        dev.residual_rms_norm(o["back"], o["first"], gains[1], 1e-6, q=o["q2"], a=o["a2"], err=o["err"], stream=stream)
        pkg._lib.check(lib.marian_hip_vocab_argmax_noalloc(o["q2"].ptr, o["a2"].ptr, M, D, emb.ptr, emult.ptr, ebias.ptr, V,
                                                           0, o["best"].ptr, o["logits"].ptr, stream), "vocab_argmax_noalloc")
        dev.sample_logits(o["logits"], u, o["token"], logprob=o["lp"], err=o["err"], stream=stream, **settings)

    captured, eager = outputs(), outputs()
    dev.synchronize()
    stream = dev.Stream()
    graph = Graph(lib, stream.handle, lambda s: step(captured, s, spaces))
    drawn = set()
    for _ in range(4):
        for dst, src in ((x, rng.standard_normal((M, D)).astype(np.float32)), (y, rng.standard_normal((M, D)).astype(np.float32)),
                         (slot, rng.integers(-1, slots, size=M).astype(np.int32)), (u, rng.random(M).astype(np.float32))):
            dev.copy(dst, up(src))
        for b in captured.values():
            b.fill_bytes(0)
        dev.synchronize()
        graph.launch(stream.handle)
        stream.sync()
        step(eager, None, (None, None))
        dev.synchronize()
        for name in captured:
            got, want = captured[name].host(), eager[name].host()
            assert np.array_equal(got.view(np.uint8), want.view(np.uint8)), name
        assert captured["err"].host()[0] == 0
        drawn.add(captured["token"].host().tobytes())
    assert len(drawn) > 1  # inputs of its own each time
    graph.close()
    stream.close()
