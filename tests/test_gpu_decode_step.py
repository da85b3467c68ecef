"""One decode step of many requests, as a serving host issues it: norm, adapted projections, vocabulary logits, draw.

Every request has its own adapter and its own sampling settings.  All calls go to one stream with nothing waited for
between them; each result is then checked from the step's own inputs as the device stored them."""

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


@pytest.mark.parametrize("M, D, F, V", [(1, 512, 2048, 32000), (37, 384, 1536, 5000), (150, 512, 2048, 32000)])
def test_decode_step(dev, M, D, F, V):
    print(f"decode step M={M} D={D} F={F} V={V}", flush=True)
    rng = np.random.default_rng(M)
    up = dev.DeviceArray.from_host
    new = dev.DeviceArray.zeros
    slots, R = 6, 16
    slot = rng.integers(-1, slots, size=M).astype(np.int32)
    layer = {}
    for name, K, N in (("up", D, F), ("down", F, D)):
        la, lav = dso.to_bf16((rng.standard_normal((slots, R, K)) / np.sqrt(K)).astype(np.float32))
        lb, lbv = dso.to_bf16((0.2 * rng.standard_normal((slots, N, R))).astype(np.float32))
        layer[name] = dict(w=rng.integers(-127, 128, size=(N, K)).astype(np.int8),
                           mult=rng.uniform(500, 1500, size=N).astype(np.float32),
                           bias=rng.standard_normal(N).astype(np.float32), la=la, lb=lb,
                           scale=rng.uniform(0.5, 2, size=slots).astype(np.float32),
                           rank=rng.integers(1, R + 1, size=slots).astype(np.int32), lav=lav, lbv=lbv)
    emb = rng.integers(-127, 128, size=(V, D)).astype(np.int8)
    emult = rng.uniform(2000, 4000, size=V).astype(np.float32)
    ebias = (0.1 * rng.standard_normal(V)).astype(np.float32)
    gains = [(1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
    x, y = (rng.standard_normal((M, D)).astype(np.float32) for _ in range(2))
    settings = dict(temperature=rng.choice(np.array([0, 0.7, 1.0], np.float32), size=M),
                    top_k=rng.choice(np.array([0, 5, 50], np.int32), size=M),
                    top_p=rng.choice(np.array([1.0, 0.9], np.float32), size=M),
                    min_p=rng.choice(np.array([0.0, 0.05], np.float32), size=M))
    u = rng.random(M).astype(np.float32)

    stream = dev.Stream()
    s = stream.handle
    dx, dy = up(x), up(y)
    h, q, a = new((M, D), np.float32), new((M, D), np.int8), new(M, np.float32)
    mid, back, err = new((M, F), np.float32), new((M, D), np.float32), new(1, np.int32)
    q2, a2 = new((M, D), np.int8), new(M, np.float32)
    logits, best, token, lp = new((M, V), np.float32), new(M, np.int32), new(M, np.int32), new(M, np.float32)
    d = {n: {k: up(v) for k, v in layer[n].items() if k[-1] != "v"} for n in layer}
    dslot, dg = up(slot), [up(g) for g in gains]
    de, dm, db, du = up(emb), up(emult), up(ebias), up(u)
    dset = {k: up(v) for k, v in settings.items()}
    first = new((M, D), np.float32)
    dev.synchronize()

    dev.residual_rms_norm(dx, dy, dg[0], 1e-6, total=first, out=h, q=q, a=a, err=err, stream=s)
    f = d["up"]
    dev.q8_linear_lora(h, f["w"], f["mult"], f["bias"], f["la"], f["lb"], f["scale"], f["rank"], dslot, mid, relu=True,
                       xq=q, xa=a, err=err, stream=s)
    f = d["down"]
    dev.q8_linear_lora(mid, f["w"], f["mult"], f["bias"], f["la"], f["lb"], f["scale"], f["rank"], dslot, back, err=err,
                       stream=s)
    dev.residual_rms_norm(back, first, dg[1], 1e-6, q=q2, a=a2, err=err, stream=s)
    dev.vocab_argmax(q2, a2, de, dm, db, best, logits=logits, stream=s)
    dev.sample_logits(logits, du, token, logprob=lp, err=err, stream=s, **dset)
    stream.sync()
    assert err.host()[0] == 0

    s0, h0 = dso.rms_norm(x, y, gains[0], 1e-6)
    assert np.array_equal(first.host(), s0)
    assert (np.abs(h.host() - h0) <= np.abs(h0) * (2.0 ** -24 + 1e-12)).all()
    hq, ha = dso.quantize_rows(h.host())
    assert np.array_equal(q.host(), hq) and np.array_equal(a.host(), ha)
    for name, rows, out, relu in (("up", h.host(), mid.host(), True), ("down", mid.host(), back.host(), False)):
        f = layer[name]
        rq, ra = dso.quantize_rows(rows)
        want, bound = dso.lora(rows, rq, ra, f["w"], f["mult"], f["bias"], f["lav"], f["lbv"], f["scale"], f["rank"], slot,
                               relu)
        assert (np.abs(out - want) <= bound).all(), name
    _, n2 = dso.rms_norm(back.host(), s0, gains[1], 1e-6)
    # the codes belong to rows that were not stored; one that lies within 2^-23 of a border may be the neighbour
    t = np.float64(127) * n2 / np.abs(n2).max(axis=1, keepdims=True)
    assert (np.abs(q2.host() - t) <= 0.5 + 127 * 2.0 ** -22).all()
    acc = q2.host().astype(np.float64) @ emb.astype(np.float64).T
    want = acc / (a2.host()[:, None].astype(np.float64) * emult) + ebias
    got = logits.host()
    masked = np.zeros(V, bool)
    masked[1], masked[7:39] = True, True
    assert np.isneginf(got[:, masked]).all()
    assert (np.abs(got - want)[:, ~masked] <= 2.0 ** -24 * (4 * np.abs(want - ebias) + np.abs(want))[:, ~masked]).all()
    for m in range(M):
        w, wl = dso.sample(got[m], u=u[m], **{k: v[m] for k, v in settings.items()})
        assert token.host()[m] == w and abs(lp.host()[m] - wl) <= 2.0 ** -24 * abs(wl) + 1e-10
    assert np.array_equal(best.host(), np.argmax(got, axis=1))
    greedy = settings["temperature"] == 0
    assert np.array_equal(token.host()[greedy], best.host()[greedy])
    stream.close()


def test_candidate_step(dev):
    """Shortlisted scoring, then a draw from the lists it scored."""
    rng = np.random.default_rng(4)
    M, K, V = 50, 384, 32000
    q, a = rng.integers(-127, 128, size=(M, K)).astype(np.int8), rng.uniform(20, 60, size=M).astype(np.float32)
    emb, mult = rng.integers(-127, 128, size=(V, K)).astype(np.int8), rng.uniform(2000, 4000, size=V).astype(np.float32)
    bias = rng.standard_normal(V).astype(np.float32)
    lens = rng.integers(1, 1200, size=M)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.uint32)
    cand = np.concatenate([np.sort(rng.permutation(V)[:n]) for n in lens]).astype(np.uint32)
    u, t = rng.random(M).astype(np.float32), np.full(M, 0.8, np.float32)
    up, new = dev.DeviceArray.from_host, dev.DeviceArray.zeros
    best, token, logits = new(M, np.int32), new(M, np.int32), new(int(off[-1]), np.float32)
    dc, do = up(cand), up(off)
    dev.candidate_argmax(up(q), up(a), up(emb), up(mult), up(bias), dc, do, int(lens.max()), best, logits=logits)
    dev.sample_candidates(logits, dc, do, int(lens.max()), up(u), token, temperature=up(t))
    dev.synchronize()
    for m in range(M):
        at, _ = dso.sample(logits.host()[off[m]:off[m + 1]], temperature=0.8, u=u[m])
        assert token.host()[m] == cand[off[m] + at]
