"""What the Python calls over a paged cache make of their buffers' sizes.  No device is needed: the library is a stand-in
that notes its arguments."""

from importlib import import_module

import pytest


class Buf:
    def __init__(self, *shape):
        self.shape, self.ptr, self.nbytes = shape, 1 << 20, 4


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def calls(pkg, monkeypatch):
    device, lib = import_module(pkg.__name__ + ".device"), Library()
    monkeypatch.setattr(device._lib, "load", lambda: lib)
    return device, lib.calls


@pytest.mark.parametrize("slot, request_, position, cap", [(128, 128, 128, 128), (128, 64, 128, 64), (64, 128, None, 64),
                                                           (None, 128, 96, 96), (None, None, 7, 7), (None, None, None, 0), (0, 5, 5, 0)])
def test_plan_writes_no_more_rows_than_the_shortest_map_has(calls, slot, request_, position, cap):
    device, made = calls
    maps = {f: Buf(n) for f, n in (("slot_of_row", slot), ("request_of_row", request_), ("position_of_row", position)) if n is not None}
    state = (Buf(4), Buf(4), 16, Buf(4, 10), Buf(4), Buf(50), Buf(1), Buf(4), Buf(4), Buf(1), Buf(5), Buf(1))
    device.paged_plan(*state, **maps)
    device.paged_plan(*state, row_cap=3, **maps)
    assert [a[17] for _, a in made] == [cap, 3]


@pytest.mark.parametrize("k, v, slots, refused", [(8, 8, 8, False), (9, 8, 8, False), (8, 9, 8, False), (7, 8, 8, True), (8, 7, 8, True),
                                                  (0, 0, 0, False), (0, 0, 1, True)])
def test_append_needs_a_row_for_every_slot(calls, k, v, slots, refused):
    """Rows are read before their slots are known."""
    device, made = calls
    call = lambda: device.paged_append(Buf(k, 128), Buf(v, 128), Buf(slots), Buf(30, 2, 16, 64), Buf(30, 2, 64, 16))  # noqa: E731
    if refused:
        with pytest.raises(ValueError, match="fewer rows"):
            call()
        assert not made
    else:
        call()
        assert made[0][1][6] == slots
