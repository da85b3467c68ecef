"""marian_hip_q8_linear_lora: a row's bits do not depend on which adapters the rows beside it use."""

import numpy as np
import pytest

from test_gpu_lora import check, dev, inputs, run  # noqa: F401 (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M, K, N, R", [
    (61, 512, 300, 16), (300, 512, 1100, 32),                    # a row at a time
    (1100, 192, 100, 16), (1100, 512, 300, 32), (1300, 320, 70, 48),  # tiles of 64 columns, the last block ragged
    (4100, 128, 1000, 16), (4101, 192, 900, 24), (4102, 128, 897, 72),  # tiles of 128
])
def test_bits_with_other_neighbours(dev, M, K, N, R):
    print(f"lora neighbours M={M} K={K} N={N} R={R}", flush=True)
    c = inputs(np.random.default_rng(M + R), M, K, N, R, 4)
    c["rank"][:] = [R, R - 3, 0, R]
    c["slot"][:] = 0
    alone, _ = run(dev, c)
    check(alone, c)
    for other in (1, 2, 3, -1):  # in one row of every 32
        c["slot"][:] = 0
        changed = np.arange(other + 1, M, 32)
        c["slot"][changed] = other
        got, _ = run(dev, c)
        check(got, c)
        same = c["slot"] == 0
        assert np.array_equal(got[same].view(np.uint32), alone[same].view(np.uint32)), other
