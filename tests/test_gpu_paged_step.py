"""Steps over a paged cache as a server runs them: plan, append, attention, verification of drafts.  Several steps on
one state against the whole numbers and the formulas, and a step captured into one graph, replayed against the eager
calls."""

import math
from importlib import import_module

import numpy as np
import pytest

import paged_oracle as po
from decode_step_oracle import to_bf16
from hip_graph import Graph

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(pkg):
    d = import_module(pkg.__name__ + ".device")
    assert d.device_count() >= 1, "no HIP device visible"
    return d


class Server:
    """The device state of a server's cache, and one step's buffers."""

    def __init__(self, dev, requests, heads, kv_heads, d, page, pages, width, cap, most, v, c_bf16=True, window=0, sinks=0):
        self.dev, self.v, self.heads, self.kv_heads, self.d, self.page, self.cap = dev, v, heads, kv_heads, d, page, cap
        self.most, self.c_bf16, self.window, self.sinks = most, c_bf16, window, sinks
        new = dev.DeviceArray.zeros
        i32 = lambda *n: new(n, np.int32)  # noqa: E731
        f32 = lambda *n: new(n, np.float32)  # noqa: E731
        self.lengths, self.held, self.table, self.count = i32(requests), i32(requests), i32(requests, width), i32(1)
        self.free = dev.DeviceArray.from_host(np.arange(pages, dtype=np.int32)[::-1].copy())
        dev.copy(self.count, dev.DeviceArray.from_host(np.array([pages], np.int32)))
        dt = np.uint16 if c_bf16 else np.float32
        self.k_cache, self.v_cache = new((pages, kv_heads, page, d), dt), new((pages, kv_heads, d, page), dt)
        self.new, self.cu, self.served, self.err = i32(requests), i32(requests + 1), i32(1), i32(1)
        self.slot, self.request, self.position = i32(cap), i32(cap), i32(cap)
        self.q, self.k, self.val = f32(cap, heads * d), f32(cap, kv_heads * d), f32(cap, kv_heads * d)
        self.out = f32(cap, heads * d)
        self.logits, self.drafts, self.u, self.u_draw = f32(cap, v), i32(cap), f32(cap), f32(requests)
        self.small, self.token, self.accepted = f32(cap, v), i32(cap), i32(requests)
        need = dev.paged_attention_workspace(requests, most, width * page, heads, kv_heads, d, window, sinks, cache_bf16=c_bf16)
        self.space = new(max(need, 16), np.uint8) if need else None
        self.verify_space = new(dev.verify_drafts_workspace(cap, requests, v, True), np.uint8)

    def put(self, buf, a):
        full = np.zeros(buf.shape, buf.dtype)
        full[:len(a)] = a
        self.dev.copy(buf, self.dev.DeviceArray.from_host(full))

    def step(self, stream=None, verify=True, own_space=True):
        dev = self.dev
        dev.paged_plan(self.lengths, self.new, self.page, self.table, self.held, self.free, self.count, self.lengths, self.held,
                       self.count, self.cu, self.served, slot_of_row=self.slot, request_of_row=self.request,
                       position_of_row=self.position, err=self.err, stream=stream)
        dev.paged_append(self.k, self.val, self.slot, self.k_cache, self.v_cache, cache_bf16=self.c_bf16, err=self.err, stream=stream)
        dev.paged_attention(self.q, self.k_cache, self.v_cache, self.table, self.lengths, self.cu, self.out, heads=self.heads,
                            max_rows=self.most, max_keys=self.table.shape[1] * self.page, scale=1.0 / math.sqrt(self.d),
                            window=self.window, sinks=self.sinks, cache_bf16=self.c_bf16,
                            workspace=self.space if own_space else None, err=self.err, stream=stream)
        if verify:
            dev.verify_drafts(self.logits, self.drafts, self.cu, self.u, self.u_draw, self.token, self.accepted,
                              max_rows=self.most, draft_logits=self.small, workspace=self.verify_space if own_space else None,
                              err=self.err, stream=stream)


@pytest.mark.parametrize("c_bf16, window, sinks, pages", [(True, 0, 0, 60), (False, 0, 0, 60), (True, 50, 3, 60), (True, 0, 0, 14),
                                                          (False, 20, 1, 14)])
def test_steps_of_a_server(dev, c_bf16, window, sinks, pages):
    """Requests come with prompts, draft, are cut back to what was accepted, end and are replaced, with too few
    pages at times: every step's state, attention and tokens."""
    rng = np.random.default_rng(7 + window)
    n, heads, kv, d, page, width, v = 9, 4, 2, 64, 16, 12, 300
    s = Server(dev, n, heads, kv, d, page, pages, width, 128, 16, v, c_bf16, window, sinks)
    lengths, held, table = np.zeros(n, np.int64), np.zeros(n, np.int64), np.zeros((n, width), np.int64)
    free, count = np.arange(pages)[::-1].copy(), pages
    keys = [(np.zeros((0, kv, d), np.float32),) * 2 for _ in range(n)]
    short = 0
    for step in range(14):
        new = np.where(lengths == 0, rng.integers(1, 17, size=n), rng.integers(1, 6, size=n))
        new[rng.random(n) < (0.3 if step % 4 == 3 else 0.03)] = -1
        rows = int(np.maximum(new, 0).sum())
        q, k, val = (rng.standard_normal((rows, h * d)).astype(np.float32) for h in (heads, kv, kv))
        logits = (2 * rng.standard_normal((rows, v))).astype(np.float32)
        small = (logits + 0.4 * rng.standard_normal((rows, v))).astype(np.float32)
        drafts, u, u_draw = small.argmax(axis=1), rng.random(rows).astype(np.float32), rng.random(n).astype(np.float32)
        for buf, a in ((s.new, new), (s.lengths, lengths), (s.q, q), (s.k, k), (s.val, val), (s.logits, logits), (s.small, small),
                       (s.drafts, drafts), (s.u, u), (s.u_draw, u_draw)):
            s.put(buf, a)
        s.out.fill_bytes(0xFF)
        s.step()
        dev.synchronize()
        want = po.plan(lengths, new, held, page, table, free, count, 128)
        got = dict(lengths=s.lengths, held=s.held, table=s.table, free=s.free, count=s.count, cu=s.cu, slot=s.slot,
                   request=s.request, position=s.position, served=s.served, err=s.err)
        for f in got:
            assert np.array_equal(got[f].host().ravel(), np.ravel(want[f])), (step, f)
        cu, short = want["cu"], short + (want["served"] < n)
        out, token, accepted = s.out.host(), s.token.host(), s.accepted.host()
        assert np.isnan(out[cu[-1]:]).all()
        for b in range(n):
            lo, hi = cu[b], cu[b + 1]
            if new[b] < 0:
                keys[b] = (np.zeros((0, kv, d), np.float32),) * 2
            if lo == hi:
                assert accepted[b] == 0
                continue
            into = (lambda x: to_bf16(x)[1]) if c_bf16 else (lambda x: x)
            keys[b] = tuple(np.concatenate([old, into(x[lo:hi].reshape(-1, kv, d))]) for old, x in zip(keys[b], (k, val)))
            expect, bound = po.attention(q[lo:hi].reshape(-1, heads, d), *keys[b], want["lengths"][b], window, sinks,
                                         1.0 / math.sqrt(d))
            assert (np.abs(out[lo:hi].reshape(-1, heads, d) - expect) <= bound).all(), (step, b)
            t, a = po.verify(logits[lo:hi], drafts[lo:hi - 1], small[lo:hi - 1], (1.0, 0, 1.0, 0.0), u[lo:hi], u_draw[b])
            assert accepted[b] == a and token[lo:hi].tolist() == t, (step, b)
            # the keys of rejected drafts are written over by the next step's
            want["lengths"][b] -= hi - lo - 1 - a
            keys[b] = tuple(x[:want["lengths"][b]] for x in keys[b])
        lengths, held, table, free, count = (want[f] for f in ("lengths", "held", "table", "free", "count"))
    assert pages > 14 or 0 < short < 14  # pages ran out, and came back


@pytest.mark.parametrize("n, heads, kv, d, page, width, v, c_bf16", [
    (1, 8, 8, 64, 16, 8, 3000, True), (13, 8, 2, 128, 32, 140, 5000, True), (40, 8, 8, 48, 16, 300, 400, False)])
def test_captured_step(pkg, dev, n, heads, kv, d, page, width, v, c_bf16):
    print(f"captured paged step n={n} heads={heads} kv={kv} d={d} width={width}", flush=True)
    rng = np.random.default_rng(n)
    lib = pkg._lib.load()
    most, cap, pages = 4, 4 * n + 3, n * width
    make = lambda: Server(dev, n, heads, kv, d, page, pages, width, cap, most, v, c_bf16)  # noqa: E731
    captured, eager = make(), make()
    dev.synchronize()
    stream = dev.Stream()
    graph = Graph(lib, stream.handle, lambda st: captured.step(st))
    state = ("lengths", "held", "table", "free", "count", "k_cache", "v_cache")
    results = state + ("cu", "slot", "request", "position", "served", "out", "token", "accepted", "err")
    seen = set()
    for turn in range(5):
        # caches of many lengths, as after many steps: pages in any order, keys of any kind
        lengths = np.minimum(rng.integers(0, width * page - most, size=n), 6000)
        held = -(-lengths // page)
        order, table = rng.permutation(pages), np.full((n, width), -1, np.int32)
        at = np.concatenate([[0], np.cumsum(held)])
        for b in range(n):
            table[b, :held[b]] = order[at[b]:at[b + 1]]
        new = rng.integers(1, most + 1, size=n)
        if n > 1:
            new[rng.integers(0, n)] = -1
        shape = (pages, kv, page, d)
        cells = rng.standard_normal(4096).astype(np.float32)
        cells = to_bf16(cells)[0] if c_bf16 else cells
        caches = np.resize(np.roll(cells, turn), int(np.prod(shape)))
        free = np.concatenate([order[at[n]:], np.full(at[n], -1)])
        logits = (2 * rng.standard_normal((cap, v))).astype(np.float32)
        small = (logits + 0.4 * rng.standard_normal((cap, v))).astype(np.float32)
        inputs = dict(lengths=lengths, held=held, table=table, free=free, count=[pages - at[n]], new=new,
                      k_cache=caches.reshape(shape), v_cache=caches.reshape(pages, kv, d, page),
                      q=rng.standard_normal((cap, heads * d)), k=rng.standard_normal((cap, kv * d)),
                      val=rng.standard_normal((cap, kv * d)), logits=logits, small=small, drafts=small.argmax(axis=1),
                      u=rng.random(cap), u_draw=rng.random(n))
        for s in (captured, eager):
            for f, a in inputs.items():
                s.put(getattr(s, f), np.asarray(a))
            for f in set(results) - set(inputs):
                getattr(s, f).fill_bytes(0)
        dev.synchronize()
        graph.launch(stream.handle)
        stream.sync()
        eager.step(own_space=False)
        dev.synchronize()
        for f in results:
            a, b = getattr(captured, f).host(), getattr(eager, f).host()
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), (turn, f)
        assert captured.err.host()[0] == 0 and captured.served.host()[0] == n
        seen.add(captured.token.host().tobytes())
    assert len(seen) > 1
    graph.close()
    stream.close()


def test_calls_on_two_streams_at_once(dev):
    """Library scratch is a stream's own: two streams' steps, enqueued before either is waited for."""
    rng = np.random.default_rng(11)
    servers = [Server(dev, 6, 8, 8, 64, 16, 6 * 300, 300, 24, 4, 2000) for _ in range(3)]
    for s in servers:
        lengths = rng.integers(2500, 4700, size=6)
        held = -(-lengths // 16)
        table = np.full((6, 300), -1, np.int32)
        order, at = rng.permutation(1800), np.concatenate([[0], np.cumsum(held)])
        for b in range(6):
            table[b, :held[b]] = order[at[b]:at[b + 1]]
        logits = (2 * rng.standard_normal((24, 2000))).astype(np.float32)
        for f, a in dict(lengths=lengths, held=held, table=table, free=np.concatenate([order[at[6]:], np.full(at[6], -1)]),
                         count=[1800 - at[6]], new=np.full(6, 4), k_cache=np.resize(to_bf16(rng.standard_normal(4001).astype(
                             np.float32))[0], s.k_cache.shape), v_cache=np.resize(to_bf16(rng.standard_normal(4003).astype(
                                 np.float32))[0], s.v_cache.shape), q=rng.standard_normal((24, 512)),
                         k=rng.standard_normal((24, 512)), val=rng.standard_normal((24, 512)), logits=logits,
                         small=logits + 0.3 * rng.standard_normal(logits.shape), drafts=logits.argmax(axis=1), u=rng.random(24),
                         u_draw=rng.random(6)).items():
            s.put(getattr(s, f), np.asarray(a))
    first = [[getattr(s, f).host() for f in ("lengths", "held", "table", "count", "free")] for s in servers]
    dev.synchronize()
    want = []
    for s, start in zip(servers, first):
        s.step()
        dev.synchronize()
        want.append([getattr(s, f).host() for f in ("out", "token", "accepted")])
        for f, a in zip(("lengths", "held", "table", "count", "free"), start):
            s.put(getattr(s, f), a)
        s.out.fill_bytes(0)
    dev.synchronize()
    streams = [dev.Stream() for _ in servers]
    for _ in range(3):
        for s, st in zip(servers, streams):
            s.step(stream=st.handle, own_space=False)
        for st in streams:
            st.sync()
        for s, w, start in zip(servers, want, first):
            for f, a in zip(("out", "token", "accepted"), w):
                assert np.array_equal(getattr(s, f).host(), a), f
            for f, a in zip(("lengths", "held", "table", "count", "free"), start):
                s.put(getattr(s, f), a)
            s.out.fill_bytes(0)
        dev.synchronize()
    for st in streams:
        st.close()
