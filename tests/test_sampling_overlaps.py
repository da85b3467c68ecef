"""Sampling calls whose outputs begin where an input of unknown length does, or lie over the candidates' ids, are
refused.  No device is needed; the pointers are never followed."""

import pytest

from test_decode_step_refusals import at, candidate_args, lib  # noqa: F401 (lib: the fixture)


@pytest.mark.parametrize("change", [
    dict(token=at(0)), dict(lp=at(0)),          # the logits' first value
    dict(token=at(1)), dict(lp=at(1)),          # the ids
    dict(token=at(1) - 12), dict(lp=at(1) - 4), dict(token=at(0) - 4),
])
def test_outputs_over_a_list(pkg, lib, change):
    assert lib.marian_hip_sample_candidates(*candidate_args(**change)) == pkg._lib.ERR_INVALID_INPUT
    assert "overlaps" in pkg._lib.op_error()
