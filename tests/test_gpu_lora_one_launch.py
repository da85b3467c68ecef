"""marian_hip_q8_linear_lora on both sides of its one-launch sizes (M max_rank <= 64, M max_rank K <= 65536, K <= 2048)."""

import numpy as np
import pytest

from test_gpu_lora import check, dev, inputs, run  # noqa: F401 (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("N", [16, 1000, 1027])
@pytest.mark.parametrize("M, K, R", [(8, 512, 8), (9, 512, 8), (8, 1024, 8), (8, 1088, 8), (4, 1024, 16), (5, 512, 16),
                                     (1, 1024, 64), (1, 512, 72), (4, 2048, 8), (5, 2048, 8), (2, 2048, 16), (7, 64, 8),
                                     (1, 2112, 8), (3, 1344, 16)])
def test_sizes_around_it(dev, M, K, R, N, quantized):
    print(f"lora one launch M={M} K={K} N={N} R={R} quantized={quantized}", flush=True)
    c = inputs(np.random.default_rng(M + K + R), M, K, N, R, 3)
    c["slot"][0] = 0  # of full rank
    got, err = run(dev, c, bool(M % 2), quantized)
    assert err == 0
    check(got, c, bool(M % 2))
