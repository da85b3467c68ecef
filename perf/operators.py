"""Operators of a decode step that serves many requests at once, as a host calls them.

Three operators, through the functions of marian-edge_amd/device.py on device buffers:

  norm    residual_rms_norm: residual addition, root-mean-square norm, int8 rows with multipliers
  lora    q8_linear_lora: a shared int8 projection with each row's own low-rank adapter
  sample  sample_logits, sample_candidates: temperature, top-k, top-p and min-p per row

Sizes are the repository's own (512- and 384-wide layers, FFN 2048 and 1536, 32000 ids, the packed rows of the 64-
and 256-sentence batches) or generic.  listed() names the cases, draw() gives more of the same ranges, prepare()
builds what a caller holds, run() is one pass (`own`: through the framework, else in elementary torch operations),
exact() the same from the definitions in 64 bits, work() the bytes and operations a pass cannot do without.
"""

from __future__ import annotations

import importlib
import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_ROOT = Path(__file__).resolve().parents[1]
_NAME = "marian_edge_amd"
_DEV = "cuda"
_EPS = 1e-6
_NO_LIMIT = 1 << 30


def _device():
    """marian-edge_amd/device.py (the package directory is not an identifier)."""
    if _NAME not in sys.modules:
        where = _ROOT / "marian-edge_amd"
        spec = importlib.util.spec_from_file_location(_NAME, where / "__init__.py",
                                                      submodule_search_locations=[str(where)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[_NAME] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module(_NAME + ".device")


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # The norm of one decode row: the smallest call, all latency.
        _norm("norm-decode-1", 1, 512),
        # The encoder's rows of the 256-sentence batch, residual stream kept, int8 rows for the next projection.
        _norm("norm-encoder-7405", 7405, 512),
        # A wide layer's rows in bfloat16, a width that is no multiple of 64, no residual.
        _norm("norm-wide-bf16", 6001, 5000, bf16=True, residual=False),
        # One request's row through the FFN's first layer, quantized in the call.
        _lora("lora-decode-1", 1, 512, 2048, 8, 4, "mixed", relu=True, quantized=False),
        # A decode step of 61 requests through the query, key and value projection, an adapter each.
        _lora("lora-decode-61", 61, 512, 1536, 16, 64, "mixed"),
        # The down-projection of the 384-wide graph, 200 active rows, adapters of rank up to 64.
        _lora("lora-decode-200", 200, 1536, 384, 64, 24, "mixed"),
        # The encoder of the 64-sentence batch: 1459 packed rows, an adapter per sentence.
        _lora("lora-encoder-1459", 1459, 512, 2048, 16, 32, "packed", relu=True),
        # A large prompt batch: long runs of rows with one adapter.
        _lora("lora-prompts-16384", 16384, 512, 2048, 32, 16, "packed", relu=True),
        # One sampled token with a nucleus: latency.
        _sample("sample-decode-1", 1, 32000, "nucleus"),
        # A decode step of 64 requests, each with settings of its own.
        _sample("sample-decode-64", 64, 32000, "mixed"),
        # Many rows over a large vocabulary in bfloat16, every setting in use.
        _sample("sample-wide-256", 256, 100003, "mixed", bf16=True),
        # Sampling from lexical-shortlist candidates, ragged lists.
        _sample("sample-candidates-200", 200, 1500, "mixed", ragged=True),
    ]


def _case(name, **fields):
    return dict(fields, name=name) if name else dict(fields)


def _norm(name, rows, dim, bf16=False, residual=True):
    return _case(name, kind="norm", rows=rows, dim=dim, bf16=bf16, residual=residual)


def _lora(name, m, k, n, rank, slots, rows, relu=False, quantized=True):
    return _case(name, kind="lora", m=m, k=k, n=n, rank=rank, slots=slots, rows=rows, relu=relu, quantized=quantized)


def _sample(name, m, v, settings, bf16=False, ragged=False):
    return _case(name, kind="sample", m=m, v=v, settings=settings, bf16=bf16, ragged=ragged)


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "lora", "lora", "sample", "sample"])
    if kind == "norm":
        dim = rng.choice([512, 384, 1024, _log(rng, 33, 8192), _log(rng, 33, 8192)])
        return _norm(None, _log(rng, 1, min(16384, (1 << 25) // dim)), dim, bf16=rng.random() < 0.4,
                     residual=rng.random() < 0.7)
    if kind == "lora":
        k, n = rng.choice([(512, 1536), (512, 512), (512, 2048), (2048, 512), (384, 1152), (384, 384), (384, 1536),
                           (1536, 384), (64 * rng.randint(1, 32), rng.randint(100, 2300))])
        m = _log(rng, 1, 8192)
        return _lora(None, m, k, n, 8 * _log(rng, 1, 8), _log(rng, 1, 64), "packed" if m > 300 else "mixed",
                     relu=rng.random() < 0.3, quantized=rng.random() < 0.7)
    if rng.random() < 0.3:
        return _sample(None, _log(rng, 1, 512), _log(rng, 104, 4000), rng.choice(["nucleus", "mixed", "temperature"]),
                       ragged=True)
    v = rng.choice([32000, 32000, _log(rng, 300, 131072)])
    return _sample(None, _log(rng, 1, min(512, (1 << 24) // v)), v, rng.choice(["nucleus", "mixed", "mixed", "temperature"]),
                   bf16=rng.random() < 0.3)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
class _Buf:
    """A torch tensor on the GPU as the device buffer the op-level functions take."""

    __slots__ = ("t", "ptr", "shape", "dtype")

    def __init__(self, t):
        self.t, self.ptr, self.shape, self.dtype = t, t.data_ptr(), tuple(t.shape), t.dtype


def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=_DEV, dtype=torch.float32)


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device=_DEV, dtype=torch.float32)


def _pick(g, n, values, dtype):
    """n values of a list, uniformly."""
    at = torch.randint(0, len(values), (n,), generator=g, device=_DEV)
    return torch.tensor(values, device=_DEV, dtype=dtype)[at]


def _host(case, salt):
    """What a case's shape fixes (run lengths, list lengths) does not depend on the seed of the inputs."""
    return np.random.Generator(np.random.PCG64([case["m"], salt]))


def _slots_of_rows(case):
    """Slot of each row: one in five rows (packed: sentences) has no adapter, -1."""
    r, m, slots = _host(case, 1), case["m"], case["slots"]
    if case["rows"] == "mixed":  # a decode step: neighbouring rows belong to different requests
        s = r.integers(0, slots, size=m)
        return np.where(r.random(m) < 0.2, -1, s).astype(np.int32)
    lens = np.clip(np.rint(r.lognormal(3.2, 0.6, size=m)), 4, 256).astype(np.int64)  # the packed workload's lengths
    s = np.where(r.random(m) < 0.2, -1, r.integers(0, slots, size=m))
    return np.repeat(s, lens)[:m].astype(np.int32)


def _candidate_offsets(case):
    """Offsets of ragged candidate lists of 1 to case["v"] ids."""
    r = _host(case, 2)
    off = np.zeros(case["m"] + 1, np.int64)
    off[1:] = np.cumsum(np.maximum(1, r.integers(case["v"] // 3, case["v"] + 1, size=case["m"])))
    off[-1] += case["v"] - (off[-1] - off[-2])  # one list has the full length
    return off


def _inputs(case, seed):
    """The call's inputs as torch tensors, from the seed alone."""
    g, kind = _gen(seed), case["kind"]
    if kind == "norm":
        rows, dim = case["rows"], case["dim"]
        dt = torch.bfloat16 if case["bf16"] else torch.float32
        channel = torch.exp(0.5 * _normal(g, dim))  # residual streams have loud channels
        got = dict(x=(_normal(g, rows, dim) * channel).to(dt), scale=1.0 + 0.1 * _normal(g, dim))
        if case["residual"]:
            got["r"] = _normal(g, rows, dim).to(dt)
        return got
    if kind == "lora":
        m, k, n, rank, slots = (case[f] for f in ("m", "k", "n", "rank", "slots"))
        got = dict(x=_normal(g, m, k), w=torch.randint(-127, 128, (n, k), generator=g, device=_DEV, dtype=torch.int8),
                   mult=1.0 / (0.0005 + 0.001 * _uniform(g, n)), bias=0.02 * _normal(g, n),
                   lora_a=(_normal(g, slots, rank, k) / math.sqrt(k)).to(torch.bfloat16),
                   lora_b=(0.3 * _normal(g, slots, n, rank) / math.sqrt(rank)).to(torch.bfloat16),
                   lora_scale=0.5 + 1.5 * _uniform(g, slots),
                   lora_rank=_pick(g, slots, [rank, rank, rank, rank // 2, max(1, rank - 3)], torch.int32),
                   slot=torch.from_numpy(_slots_of_rows(case)).to(_DEV))
        if case["quantized"]:
            got["q"], got["a"] = _quantize_rows(got["x"])
        return got
    m = case["m"]
    if case["ragged"]:
        off = _candidate_offsets(case)
        total = int(off[-1])
        got = dict(logits=2.5 * _normal(g, total), off=torch.from_numpy(off.astype(np.int32)).to(_DEV))
        step = torch.randint(1, 12, (total,), generator=g, device=_DEV)  # ascending ids within a list
        run = torch.cumsum(step, 0)
        got["cand"] = (run - torch.repeat_interleave(run[torch.from_numpy(off[:-1]).to(_DEV)],
                                                     torch.from_numpy(np.diff(off)).to(_DEV))).to(torch.int32)
    else:
        logits = 2.5 * _normal(g, m, case["v"])
        logits[:, 1] = -math.inf  # the generation mask
        logits[:, 7:39] = -math.inf
        got = dict(logits=logits.to(torch.bfloat16 if case["bf16"] else torch.float32))
    few = case["settings"]
    got["temperature"] = 0.6 + 0.7 * _uniform(g, m)
    got["top_k"] = torch.zeros(m, device=_DEV, dtype=torch.int32)
    got["top_p"] = torch.ones(m, device=_DEV)
    got["min_p"] = torch.zeros(m, device=_DEV)
    if few == "nucleus":
        got["top_p"] = 0.8 + 0.19 * _uniform(g, m)
    elif few == "mixed":  # requests choose for themselves; temperature 0 is greedy
        got["temperature"] = torch.where(_uniform(g, m) < 0.05, 0.0, got["temperature"])
        got["top_k"] = _pick(g, m, [0, 0, 0, 1, 20, 40, 50, 200, 1000], torch.int32)
        got["top_p"] = _pick(g, m, [1.0, 1.0, 0.5, 0.9, 0.95, 0.99], torch.float32)
        got["min_p"] = _pick(g, m, [0.0, 0.0, 0.0, 0.02, 0.1], torch.float32)
    got["u"] = _uniform(g, m)
    return got


def prepare(case, seed):
    got, kind = _inputs(case, seed), case["kind"]
    s = {name: _Buf(t) for name, t in got.items()}
    new = lambda shape, dtype: _Buf(torch.zeros(shape, device=_DEV, dtype=dtype))  # noqa: E731
    if kind == "norm":
        shape = (case["rows"], case["dim"])
        s["out"], s["oq"], s["oa"] = new(shape, torch.float32), new(shape, torch.int8), new(shape[:1], torch.float32)
        s["sum"] = new(shape, torch.float32) if case["residual"] else None
    elif kind == "lora":
        s["out"] = new((case["m"], case["n"]), torch.float32)
    else:
        s["token"], s["logprob"] = new(case["m"], torch.int32), new(case["m"], torch.float32)
    s["case"], s["kind"] = dict(case), kind
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)[s["kind"]](s, s["case"])


def _own_norm(s, c):
    _device().residual_rms_norm(s["x"], s.get("r"), s["scale"], _EPS, total=s["sum"], out=s["out"], q=s["oq"], a=s["oa"],
                                bf16=c["bf16"])
    got = dict(out=s["out"].t, a=s["oa"].t, values=torch.div(s["oq"].t, s["oa"].t[:, None]))
    return dict(got, sum=s["sum"].t) if c["residual"] else got


def _own_lora(s, c):
    _device().q8_linear_lora(s["x"], s["w"], s["mult"], s["bias"], s["lora_a"], s["lora_b"], s["lora_scale"],
                             s["lora_rank"], s["slot"], s["out"], relu=c["relu"], xq=s.get("q"), xa=s.get("a"))
    return s["out"].t


def _own_sample(s, c):
    settings = dict(temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                    logprob=s["logprob"])
    if c["ragged"]:
        _device().sample_candidates(s["logits"], s["cand"], s["off"], c["v"], s["u"], s["token"], **settings)
    else:
        _device().sample_logits(s["logits"], s["u"], s["token"], bf16=c["bf16"], **settings)
    return dict(token=s["token"].t, logprob=s["logprob"].t)


def _quantize_rows(y):
    """Row multipliers 127 / max|row| (1 for a zero row) and codes clamp(rne(y a), -127, 127): quotient and product
    rounded once to 32 bits."""
    m = y.abs().amax(dim=1)
    a = torch.where(m > 0, 127.0 / torch.where(m > 0, m, 1.0).double(), 1.0).float()
    return torch.clamp(torch.round(y * a[:, None]), -127, 127).to(torch.int8), a


def _plain_norm(s, c):
    x = s["x"].t.float()
    if c["residual"]:
        x = x + s["r"].t.float()
    # 64 bits: the int8 codes lie next to rounding borders
    d = x.double()
    y = (d / torch.sqrt((d * d).mean(dim=1, keepdim=True) + _EPS) * s["scale"].t.double()).float()
    q, a = _quantize_rows(y)
    got = dict(out=y, a=a, values=torch.div(q, a[:, None]))
    return dict(got, sum=x) if c["residual"] else got


def _plain_lora(s, c):
    x = s["x"].t
    q, a = (s["q"].t, s["a"].t) if c["quantized"] else _quantize_rows(x)
    y = (q.float() @ s["w"].t.float().T) / (a[:, None] * s["mult"].t[None, :]) + s["bias"].t
    slots, rank = c["slots"], c["rank"]
    # Every adapter at once: rows keep the products of their own slot's live ranks.
    live = torch.arange(rank, device=x.device)[None, :] < s["lora_rank"].t[:, None]
    gain = torch.where(live, s["lora_scale"].t[:, None], 0.0)
    mine = s["slot"].t[:, None] == torch.arange(slots, device=x.device)[None, :]
    t = (x @ s["lora_a"].t.float().reshape(slots * rank, -1).T).reshape(-1, slots, rank)
    t = (t * gain * mine[:, :, None]).reshape(-1, slots * rank)
    y = y + t @ s["lora_b"].t.float().transpose(1, 2).reshape(slots * rank, -1)
    return torch.clamp_min(y, 0.0) if c["relu"] else y


def _plain_sample(s, c):
    z = s["logits"].t
    if c["ragged"]:
        off = s["off"].t.long()
        at = off[:-1, None] + torch.arange(c["v"], device=z.device)[None, :]
        inside = at < off[1:, None]
        z = torch.where(inside, z[torch.where(inside, at, 0)], -math.inf)
    z, order = torch.sort(z.float(), dim=1, descending=True, stable=True)
    # 64 bits: a drawn number may lie next to a border of the running sums
    t = s["temperature"].t.double()[:, None]
    greedy = t == 0
    x = (z.double() - z[:, :1].double()) / torch.where(greedy, 1.0, t)
    k = torch.where(s["top_k"].t > 0, s["top_k"].t, _NO_LIMIT)[:, None]
    k = torch.where(greedy, 1, k)
    p = torch.exp(x) * (torch.arange(z.shape[1], device=z.device)[None, :] < k)
    upto = torch.cumsum(p, dim=1)
    p = p * (upto - p < s["top_p"].t.double()[:, None] * upto[:, -1:])
    p = p * (x >= torch.log(s["min_p"].t.double())[:, None])
    by_id = torch.zeros_like(p).scatter_(1, order, p)
    upto = torch.cumsum(by_id, dim=1)
    total = upto[:, -1:]
    at = (upto <= s["u"].t.double()[:, None] * total).sum(dim=1).clamp_max(z.shape[1] - 1)
    chosen = torch.gather(by_id, 1, at[:, None])
    token = s["cand"].t[off[:-1] + at] if c["ragged"] else at.to(torch.int32)
    return dict(token=token, logprob=torch.log(chosen / total)[:, 0].float())


_own = dict(norm=_own_norm, lora=_own_lora, sample=_own_sample)
_plain = dict(norm=_plain_norm, lora=_plain_lora, sample=_plain_sample)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, b = case["rows"] * case["dim"], 2 if case["bf16"] else 4
        return {"bytes": n * (b + 4 + 1 + ((b + 4) if case["residual"] else 0)) + 4 * case["rows"] + 4 * case["dim"],
                "flops": 8 * n}
    if kind == "lora":
        m, k, n, rank = (case[f] for f in ("m", "k", "n", "rank"))
        slot = _slots_of_rows(case)
        used, rows = len(set(slot[slot >= 0].tolist())), int((slot >= 0).sum())
        x = 4 * k + ((k + 4) if case["quantized"] else 0)
        return {"bytes": m * (x + 4 * n + 4) + n * (k + 8) + used * (2 * rank * (k + n) + 8),
                "flops": 2 * m * n * k + 2 * rows * rank * (k + n)}
    n = int(_candidate_offsets(case)[-1]) if case["ragged"] else case["m"] * case["v"]
    return {"bytes": n * (2 if case["bf16"] else 4) + 28 * case["m"], "flops": 12 * n}


# ---------------------------------------------------------------------------
# The same results in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    got, kind = _inputs(case, seed), case["kind"]
    if kind == "norm":
        s = got["x"].double()
        if case["residual"]:
            s = (s + got["r"].double()).float().double()  # the stored residual stream is what is normalized
        rms = torch.linalg.vector_norm(s, dim=1, keepdim=True) / math.sqrt(case["dim"])
        y = s * got["scale"].double() / torch.sqrt(rms * rms + _EPS)
        # The codes belong to the stored 32-bit rows and multipliers.
        y32 = y.float().double()
        m = y32.abs().amax(dim=1, keepdim=True)
        a = torch.where(m > 0, 127.0 / m, torch.ones_like(m)).float().double()
        out = dict(out=y, a=a[:, 0], values=torch.clamp(torch.round((y32 * a).float().double()), -127, 127) / a)
        return dict(out, sum=s) if case["residual"] else out
    if kind == "lora":
        x = got["x"].double()
        if case["quantized"]:
            q, a = got["q"].double(), got["a"].double()[:, None]
        else:
            a = (127.0 / x.abs().amax(dim=1, keepdim=True)).float().double()
            q = torch.clamp(torch.round((x * a).float().double()), -127, 127)
        y = (q @ got["w"].double().T) / a / got["mult"].double() + got["bias"].double()
        slot = got["slot"].cpu().numpy()
        for j in sorted(set(slot[slot >= 0].tolist())):
            rows = torch.from_numpy(np.flatnonzero(slot == j)).to(_DEV)
            r = int(got["lora_rank"][j])
            t = x[rows] @ got["lora_a"][j, :r].double().T
            y[rows] += float(got["lora_scale"][j]) * (t @ got["lora_b"][j, :, :r].double().T)
        return torch.relu(y) if case["relu"] else y
    token, logprob = [], []
    temperature, top_k, top_p, min_p, u = (got[f].cpu().tolist() for f in ("temperature", "top_k", "top_p", "min_p", "u"))
    off = got["off"].cpu().tolist() if case["ragged"] else None
    for i in range(case["m"]):
        z = (got["logits"][off[i]:off[i + 1]] if case["ragged"] else got["logits"][i]).double()
        kept = torch.argsort(-z, stable=True)  # descending logits, ascending places
        w = torch.softmax(z[kept] / (temperature[i] or 1.0), dim=0)
        count = 1 if temperature[i] == 0 else top_k[i] if top_k[i] > 0 else len(kept)
        kept, w = kept[:count], w[:count]
        mass = torch.cumsum(w, 0)
        count = 1 + int((mass[:-1] < top_p[i] * mass[-1]).sum())
        kept, w = kept[:count], w[:count]
        count = int((w >= min_p[i] * w[0]).sum())
        place, by_place = torch.sort(kept[:count])
        w = w[:count][by_place]
        mass = torch.cumsum(w, 0)
        at = min(int(torch.searchsorted(mass, u[i] * mass[-1], right=True)), count - 1)
        place = int(place[at])
        token.append(int(got["cand"][off[i] + place]) if case["ragged"] else place)
        logprob.append(torch.log(w[at]) - torch.log(mass[-1]))
    return dict(token=torch.tensor(token, dtype=torch.int32), logprob=torch.stack(logprob))
