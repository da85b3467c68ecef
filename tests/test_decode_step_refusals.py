"""Calls that the decode-step operators (RMS norm, adapter layer, sampling) refuse.  No device is needed: the
checks come before anything is launched.  The pointers are never followed."""

import ctypes as C

import pytest

P = 1 << 20  # stands for a device address


def at(k):
    return P + (k << 24)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg._lib.load()


def norm_args(**change):
    a = dict(x=at(0), ldx=96, r=at(1), ldr=96, scale=at(2), eps=1e-6, rows=4, dim=96, bf16=0, sum=at(3), out=at(4),
             q=at(5), a=at(6), err=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, why", [
    (dict(x=None), "missing"), (dict(scale=None), "missing"),
    (dict(rows=-1), "out of range"), (dict(rows=1 << 31), "out of range"),
    (dict(dim=0), "out of range"), (dict(dim=16385, ldx=1 << 15, ldr=1 << 15), "out of range"),
    (dict(ldx=95), "out of range"), (dict(ldr=95), "out of range"), (dict(ldx=1 << 30), "out of range"),
    (dict(ldr=1 << 61), "out of range"),
    (dict(eps=0.0), "out of range"), (dict(eps=-1e-6), "out of range"), (dict(eps=float("nan")), "out of range"),
    (dict(eps=float("inf")), "out of range"),
    (dict(out=None, q=None, a=None), "neither"),
    (dict(a=None), "together"), (dict(q=None), "together"),
    (dict(out=at(0) + 4), "overlaps an input"), (dict(sum=at(1) + 16), "overlaps an input"),
    (dict(q=at(0)), "overlaps an input"), (dict(a=at(2)), "overlaps an input"),
    (dict(out=at(0), bf16=1), "overlaps an input"), (dict(out=at(0), ldx=100), "overlaps an input"),
    (dict(sum=at(4)), "outputs overlap"), (dict(a=at(5)), "outputs overlap"),
])
def test_rms_norm_refuses(pkg, lib, change, why):
    assert lib.marian_hip_residual_rms_norm(*norm_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert why in pkg._lib.op_error()


def test_rms_norm_of_no_rows(pkg, lib):
    assert lib.marian_hip_residual_rms_norm(*norm_args(rows=0)) == pkg._lib.OK


def lora_args(**change):
    a = dict(x=at(0), xq=at(1), xa=at(2), M=4, K=128, w=at(3), mult=at(4), bias=at(5), N=96, relu=0, la=at(6), lb=at(7),
             ls=at(8), lr=at(9), slots=2, max_rank=16, slot=at(10), out=at(11), ws=at(12), ws_bytes=1 << 20, err=None,
             stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, why", [
    (dict(M=-1), "out of range"), (dict(M=1 << 31), "out of range"), (dict(K=0), "out of range"),
    (dict(K=100), "out of range"), (dict(K=(1 << 17) + 64), "out of range"), (dict(K=1 << 40), "out of range"), (dict(N=0), "out of range"), (dict(N=1 << 31), "out of range"),
    (dict(max_rank=0), "out of range"), (dict(max_rank=12), "out of range"), (dict(max_rank=136), "out of range"),
    (dict(slots=0), "out of range"), (dict(slots=(1 << 20) + 1), "out of range"), (dict(slots=1 << 31), "out of range"),
    (dict(x=None), "missing"), (dict(xq=None), "missing"), (dict(xa=None), "missing"), (dict(w=None), "missing"),
    (dict(mult=None), "missing"), (dict(bias=None), "missing"), (dict(la=None), "missing"), (dict(lb=None), "missing"),
    (dict(ls=None), "missing"), (dict(lr=None), "missing"), (dict(slot=None), "missing"), (dict(out=None), "missing"),
    (dict(x=at(0) + 4), "aligned"), (dict(la=at(6) + 2), "aligned"), (dict(lb=at(7) + 8), "aligned"),
    (dict(w=at(3) + 1), "aligned"), (dict(xq=at(1) + 8), "aligned"), (dict(ws=at(12) + 4), "aligned"),
    (dict(ws_bytes=16), "too small"), (dict(M=(1 << 26) + 1), "out of range"), (dict(N=1 << 20), "out of range"),
    (dict(out=at(1) + 16), "overlaps"), (dict(out=at(3)), "overlaps"), (dict(out=at(7) + 32), "overlaps"),
    (dict(out=at(10)), "overlaps"), (dict(out=at(12) + 64), "overlaps"), (dict(ws=at(0) + 256), "overlaps"),
    (dict(ws=at(1)), "overlaps"), (dict(ws=at(6) - 1024), "overlaps"), (dict(ws=at(10)), "overlaps"), (dict(ws=at(11)), "overlaps"),
])
def test_lora_refuses(pkg, lib, change, why):
    assert lib.marian_hip_q8_linear_lora(*lora_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert why in pkg._lib.op_error()


def test_lora_of_no_rows(pkg, lib):
    assert lib.marian_hip_q8_linear_lora(*lora_args(M=0)) == pkg._lib.OK


def test_lora_workspace_sizes(pkg, lib):
    n = C.c_size_t(0)

    def size(m, k, r, has):
        assert lib.marian_hip_q8_linear_lora_workspace(m, k, r, has, C.byref(n)) == pkg._lib.OK
        return n.value

    assert size(0, 64, 8, 1) == 0
    assert size(64, 512, 16, 0) >= size(64, 512, 16, 1) + 64 * 512 + 64 * 4
    assert size(64, 512, 16, 1) >= 64 * 16 * 4
    for bad in ((-1, 64, 8), (1, 65, 8), (1, 64, 4), (1, 64, 256)):
        assert lib.marian_hip_q8_linear_lora_workspace(*bad, 1, C.byref(n)) == pkg._lib.ERR_INVALID_INPUT
    assert lib.marian_hip_q8_linear_lora_workspace(1, 64, 8, 1, None) == pkg._lib.ERR_INVALID_INPUT


def sample_args(**change):
    a = dict(logits=at(0), ld=100, rows=4, V=96, bf16=0, t=None, k=None, p=None, mp=None, u=at(1), token=at(2), lp=None,
             err=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, why", [
    (dict(logits=None), "missing"), (dict(u=None), "missing"), (dict(token=None), "missing"),
    (dict(rows=-1), "out of range"), (dict(rows=(1 << 20) + 1), "out of range"), (dict(V=0), "out of range"),
    (dict(V=(1 << 19) + 1, ld=1 << 20), "out of range"), (dict(ld=95), "out of range"), (dict(ld=1 << 62), "out of range"),
    (dict(token=at(0) + 64), "overlaps"), (dict(token=at(0) + 4 * 395), "overlaps"), (dict(token=at(1)), "overlaps"),
    (dict(lp=at(2) + 12), "overlaps"), (dict(lp=at(3), t=at(3)), "overlaps"), (dict(k=at(2)), "overlaps"),
    (dict(p=at(2) + 4), "overlaps"), (dict(mp=at(2) - 4), "overlaps"),
])
def test_sample_logits_refuses(pkg, lib, change, why):
    assert lib.marian_hip_sample_logits(*sample_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert why in pkg._lib.op_error()


def candidate_args(**change):
    a = dict(logits=at(0), cand=at(1), off=at(2), rows=4, most=100, t=None, k=None, p=None, mp=None, u=at(3),
             token=at(4), lp=None, err=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, why", [
    (dict(logits=None), "missing"), (dict(cand=None), "missing"), (dict(off=None), "missing"), (dict(u=None), "missing"),
    (dict(token=None), "missing"), (dict(rows=-1), "out of range"), (dict(rows=(1 << 20) + 1), "out of range"),
    (dict(most=0), "out of range"), (dict(most=(1 << 19) + 1), "out of range"),
    (dict(token=at(2) + 16), "overlaps"), (dict(token=at(3) + 8), "overlaps"), (dict(lp=at(4)), "overlaps"),
    (dict(k=at(4) + 4), "overlaps"),
])
def test_sample_candidates_refuses(pkg, lib, change, why):
    assert lib.marian_hip_sample_candidates(*candidate_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert why in pkg._lib.op_error()


def test_sampling_of_no_rows(pkg, lib):
    assert lib.marian_hip_sample_logits(*sample_args(rows=0)) == pkg._lib.OK
    assert lib.marian_hip_sample_candidates(*candidate_args(rows=0)) == pkg._lib.OK
