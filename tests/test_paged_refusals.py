"""Calls that the operators over a paged cache refuse.  No device is needed: the checks come before anything is
launched.  The pointers are never followed."""

import ctypes as C

import pytest

P = 1 << 20  # stands for a device address


def at(k):
    return P + (k << 28)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg._lib.load()


def plan_args(**change):
    a = dict(lengths=at(0), new=at(1), held=at(2), requests=4, page=16, table=at(3), blocks=10, free=at(4), count=at(5), pages=50,
             lengths_out=at(0), held_out=at(2), count_out=at(5), cu=at(6), slot=at(7), request=at(8), position=at(9), cap=32,
             served=at(10), err=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, why", [
    *[({f: None}, "missing") for f in ("lengths", "new", "held", "table", "free", "count", "lengths_out", "held_out",
                                       "count_out", "cu", "served")],
    (dict(page=0), "power of two"), (dict(page=4), "power of two"), (dict(page=24), "power of two"),
    (dict(page=2048), "power of two"), (dict(page=-16), "power of two"),
    (dict(requests=0), "out of range"), (dict(requests=8193), "out of range"), (dict(blocks=0), "out of range"),
    (dict(blocks=(1 << 18) + 1), "out of range"), (dict(pages=0), "out of range"), (dict(pages=1 << 27), "out of range"),
    (dict(cap=-1), "out of range"), (dict(cap=(1 << 18) + 1), "out of range"),
    (dict(lengths_out=at(0) + 4), "overlaps"), (dict(held_out=at(0)), "overlaps"), (dict(count_out=at(4) + 8), "overlaps"),
    (dict(cu=at(1) + 12), "overlaps"), (dict(slot=at(8) + 64), "overlaps"), (dict(position=at(3) + 156), "overlaps"),
    (dict(served=at(2)), "overlaps"), (dict(table=at(4) + 196), "overlaps"), (dict(lengths_out=at(1)), "overlaps"),
])
def test_plan_refuses(pkg, lib, change, why):
    assert lib.marian_hip_paged_plan(*plan_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert why in pkg._lib.op_error()


def append_args(**change):
    a = dict(k=at(0), ldk=200, v=at(1), ldv=128, bf16=0, slot=at(2), rows=8, kv_heads=2, d=64, kc=at(3), vc=at(4), cache16=1,
             pages=30, page=16, err=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, why", [
    *[({f: None}, "missing") for f in ("k", "v", "slot", "kc", "vc")],
    (dict(rows=-1), "out of range"), (dict(rows=(1 << 18) + 1), "out of range"), (dict(ldk=127), "out of range"),
    (dict(ldv=127), "out of range"), (dict(ldv=1 << 30), "out of range"), (dict(ldk=1 << 62), "out of range"),
    (dict(kv_heads=0), "out of range"), (dict(kv_heads=129, ldk=9000, ldv=9000), "out of range"), (dict(pages=0), "out of range"),
    (dict(pages=1 << 27), "out of range"), (dict(d=32), "head_dim"), (dict(d=256, ldk=512, ldv=512), "head_dim"),
    (dict(page=12), "power of two"), (dict(page=4), "power of two"),
    (dict(kc=at(3) + 8), "16-byte"), (dict(vc=at(4) + 2), "16-byte"), (dict(k=at(0) + 2), "aligned to its values"),
    (dict(v=at(1) + 1, bf16=1), "aligned to its values"),
    (dict(kc=at(0) + 4096), "overlaps"), (dict(vc=at(1)), "overlaps"), (dict(vc=at(3) + 1024), "overlaps"),
    (dict(slot=at(4) + 64), "overlaps"),
])
def test_append_refuses(pkg, lib, change, why):
    assert lib.marian_hip_paged_append(*append_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert why in pkg._lib.op_error()


def attention_args(**change):
    a = dict(q=at(0), ldq=512, bf16=0, rows=8, kc=at(1), vc=at(2), cache16=1, pages=30, page=16, table=at(3), blocks=10,
             lengths=at(4), cu=at(5), requests=4, max_rows=3, max_keys=160, heads=8, kv_heads=2, d=64, scale=0.125, window=0,
             sinks=0, out=at(6), ldo=512, ws=at(7), ws_bytes=1 << 24, err=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, why", [
    *[({f: None}, "missing") for f in ("q", "kc", "vc", "table", "lengths", "cu", "out")],
    (dict(rows=-1), "out of range"), (dict(rows=(1 << 18) + 1), "out of range"), (dict(requests=-1), "out of range"),
    (dict(requests=8193), "out of range"), (dict(max_rows=0), "out of range"), (dict(max_rows=65), "out of range"),
    (dict(max_keys=0), "out of range"), (dict(max_keys=(1 << 27) + 1), "out of range"), (dict(window=-1), "out of range"),
    (dict(window=1 << 31), "out of range"), (dict(sinks=-1), "out of range"), (dict(sinks=1 << 40), "out of range"),
    (dict(heads=0), "multiple"), (dict(heads=9), "multiple"), (dict(heads=130, ldq=9000, ldo=9000), "multiple"),
    (dict(kv_heads=0), "multiple"), (dict(kv_heads=16), "multiple"), (dict(d=40), "head_dim"), (dict(d=512), "head_dim"),
    (dict(pages=0), "out of range"), (dict(pages=1 << 28), "out of range"), (dict(page=17), "power of two"),
    (dict(blocks=0), "out of range"), (dict(blocks=(1 << 18) + 1), "out of range"), (dict(ldq=504), "out of range"),
    (dict(ldo=508), "out of range"), (dict(ldq=516), "out of range"), (dict(ldo=514), "out of range"),
    (dict(ldq=1 << 30), "out of range"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=at(0) + 8), "16-byte"), (dict(out=at(6) + 4), "16-byte"), (dict(kc=at(1) + 8), "16-byte"), (dict(vc=at(2) + 2), "16-byte"),
    (dict(ws=at(7) + 8), "16-byte"),
    (dict(out=at(0)), "overlaps"), (dict(out=at(1) + 1024), "overlaps"), (dict(out=at(3)), "overlaps"), (dict(ws=at(2)), "overlaps"),
    (dict(ws=at(6) + 1024), "overlaps"), (dict(ws=at(4)), "overlaps"),
    (dict(max_keys=1 << 20, blocks=1 << 17, ws_bytes=16), "too small"),
])
def test_attention_refuses(pkg, lib, change, why):
    assert lib.marian_hip_paged_attention(*attention_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert why in pkg._lib.op_error()


def verify_args(**change):
    a = dict(logits=at(0), ld=128, rows=8, v=100, bf16=0, draft_logits=at(1), ld_draft=100, draft_rows=6, draft_row=at(2),
             drafts=at(3), cu=at(4), requests=3, max_rows=4, t=at(5), k=at(6), p=at(7), mp=at(8), u=at(9), u_draw=at(10),
             token=at(11), accepted=at(12), ws=at(13), ws_bytes=1 << 20, err=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, why", [
    *[({f: None}, "missing") for f in ("logits", "drafts", "cu", "u", "u_draw", "token", "accepted")],
    (dict(rows=-1), "out of range"), (dict(rows=(1 << 18) + 1), "out of range"), (dict(v=0), "out of range"),
    (dict(v=(1 << 19) + 1, ld=1 << 20, ld_draft=1 << 20), "out of range"), (dict(ld=99), "out of range"), (dict(ld=1 << 30), "out of range"),
    (dict(requests=-1), "out of range"), (dict(requests=8193), "out of range"), (dict(max_rows=0), "out of range"),
    (dict(ld_draft=99), "draft rows"), (dict(draft_rows=-1), "draft rows"), (dict(draft_rows=1 << 31), "draft rows"),
    (dict(draft_logits=None), "without draft_logits"), (dict(ws=at(13) + 4), "8-byte"),
    (dict(ws_bytes=64), "too small"),
    (dict(token=at(0) + 400), "overlaps"), (dict(token=at(3)), "overlaps"), (dict(accepted=at(11) + 16), "overlaps"),
    (dict(accepted=at(10)), "overlaps"), (dict(token=at(9) + 16), "overlaps"), (dict(ws=at(1)), "overlaps"),
    (dict(ws=at(2)), "overlaps"), (dict(accepted=at(4) + 12), "overlaps"), (dict(token=at(7)), "overlaps"),
])
def test_verify_refuses(pkg, lib, change, why):
    assert lib.marian_hip_verify_drafts(*verify_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert why in pkg._lib.op_error()


def test_calls_without_work(pkg, lib):
    assert lib.marian_hip_paged_append(*append_args(rows=0)) == pkg._lib.OK
    assert lib.marian_hip_paged_attention(*attention_args(rows=0)) == pkg._lib.OK
    assert lib.marian_hip_paged_attention(*attention_args(requests=0)) == pkg._lib.OK
    assert lib.marian_hip_verify_drafts(*verify_args(requests=0)) == pkg._lib.OK


def test_workspace_sizes(pkg, lib):
    n = C.c_size_t(0)
    size = lib.marian_hip_paged_attention_workspace
    assert size(1, 1, 64, 8, 8, 64, 1, 1, 0, 0, C.byref(n)) == pkg._lib.OK and n.value == 0  # one piece
    for q16, c16 in ((0, 0), (0, 1), (1, 1), (1, 0)):
        assert size(1, 1, 100000, 8, 8, 64, q16, c16, 0, 0, C.byref(n)) == pkg._lib.OK and n.value > 8 * 64 * 4
        assert size(1, 1, 100000, 8, 8, 64, q16, c16, 100, 4, C.byref(n)) == pkg._lib.OK and n.value == 0  # a short window
    assert size(1, 1, 100000, 8, 8, 64, 1, 1, 0, 0, None) == pkg._lib.ERR_INVALID_INPUT
    for bad in ((-1, 1, 64, 8, 8, 64, 1, 1, 0, 0), (1, 65, 64, 8, 8, 64, 1, 1, 0, 0), (1, 1, 64, 8, 3, 64, 1, 1, 0, 0),
                (1, 1, 64, 8, 8, 65, 1, 1, 0, 0), (1, 1, 64, 8, 8, 64, 1, 1, -1, 0)):
        assert size(*bad, C.byref(n)) == pkg._lib.ERR_INVALID_INPUT
    of_rows = lib.marian_hip_verify_drafts_workspace
    assert of_rows(10, 3, 1000, 0, C.byref(n)) == pkg._lib.OK
    one = n.value
    assert of_rows(10, 3, 1000, 1, C.byref(n)) == pkg._lib.OK and n.value > one > 0
    for bad in ((-1, 3, 1000, 1), (10, -1, 1000, 1), (10, 8193, 1000, 1), (10, 3, 0, 1), (10, 3, 1 << 20, 1)):
        assert of_rows(*bad, C.byref(n)) == pkg._lib.ERR_INVALID_INPUT
    assert of_rows(1, 1, 1, 1, None) == pkg._lib.ERR_INVALID_INPUT
